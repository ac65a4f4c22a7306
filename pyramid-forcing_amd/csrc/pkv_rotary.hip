// Rotary positions at any distance: the rotation of q (and k) heads by
// angles that are computed where they are used, not read from a table of so
// many rows.  Pair j of a head turns by pos[axis(j)] * freq[j]:
//   (u, w) -> scale * (u cos a - w sin a, u sin a + w cos a)
// with (u, w) = (x[2j], x[2j + 1]) (interleaved) or (x[j], x[j + pairs])
// (halves); columns from 2 * pairs on are copied.  The inverse turns by -a:
// the gradient of the rotation, as the matrix is orthogonal up to scale.
//
// The angle's product, its reduction to a fraction of a turn (a position of a
// million times a frequency of 1 leaves an fp32 angle off by 0.06 radians), sine
// and cosine are taken in 64 bits and rounded once: the heads of a row share
// them, so that the timed cases below cost the same with sine and cosine in 32 bits
// (25.2 us against 25.1; one head of 256 pairs, the other end, 18.0 against 14.7 for
// 16,384 rows).
//
// Bound by memory: every element is read and written once.  A workgroup takes
// a few tokens, computes each (token, pair)'s sine and cosine once in LDS and
// applies them to all heads of q and k in 16-byte accesses.  4,680 rows of 12
// heads of 128 (bf16, 29 MB read and written) in 7.3 us, 4.0 TB/s; 8,191 rows of 20
// heads of 80 (fp32, 105 MB) in 18 us under the profiler and 25 a call, 4.2 TB/s (a
// copy of 1 GiB moves 4.8); 16 rows of 40 heads in 3.6, the launch and the chain of
// position, angle and store.  Reading q ahead of the angles was no faster.

#include "pkv_common.h"

namespace pkv {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 256;

// n / d and n % d for n < 2^31 by a multiplication (d fixed for the launch)
struct FastDiv {
  uint32_t d, mul, shift;
};

static FastDiv fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  while ((1ull << f.shift) < d) ++f.shift;
  f.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
  return f;
}

__device__ inline uint32_t div_by(uint32_t n, const FastDiv &f) { return (__umulhi(n, f.mul) + n) >> f.shift; }

struct RotParams {
  const void *q, *k;
  void *qo, *ko;
  const void *pos;
  const double *freqs;
  int64_t row0, rows;  // this launch's first row; the rows of all
  int64_t q_tok, q_head, k_tok, k_head, pos_row;
  int Hq, heads, D, pairs, n_axes, tokens;
  int axis_end[PKV_ROTARY_MAX_AXES];
  int pos64;
  float scale, sign;
  FastDiv by_items, by_heads, by_pairs;
};

template <typename T>
__device__ inline float rot_load(T x);
template <>
__device__ inline float rot_load<float>(float x) { return x; }
template <>
__device__ inline float rot_load<_Float16>(_Float16 x) { return static_cast<float>(x); }
template <>
__device__ inline float rot_load<__bf16>(__bf16 x) { return static_cast<float>(x); }

// N elements of T as one access: 16 bytes, or one or two elements that begin
// anywhere
template <typename T, int N>
struct RotVec {
  typedef T type __attribute__((ext_vector_type(N), aligned(N * sizeof(T) == 16 ? 16 : sizeof(T))));
};
template <typename T>
struct RotVec<T, 1> {
  typedef T type;
};

// V: pairs per item (HALF: two accesses of V elements, else one of 2 V; the
// copied columns go by the same number of elements).  V is 1 where pairs, strides
// or pointers do not fit 16 bytes, for all of a head: 8,191 rows of 20 heads of 80
// (bf16) with 13 pairs turned take 36 us by halves and 22 interleaved, with 16
// pairs 11.3.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(RotParams p) {
  extern __shared__ float2 cs[];  // [tokens][pairs]: cosine and sine, scaled
  const int64_t tok0 = p.row0 + static_cast<int64_t>(blockIdx.x) * p.tokens;
  const int left = p.rows - tok0 < p.tokens ? static_cast<int>(p.rows - tok0) : p.tokens;
  for (int e = threadIdx.x; e < left * p.pairs; e += kRotThreads) {
    const int t = div_by(e, p.by_pairs), j = e - t * p.pairs;
    int a = 0;
    while (j >= p.axis_end[a]) ++a;  // (the last axis ends at the last pair)
    const int64_t at = (tok0 + t) * p.pos_row + a;
    const double x = p.pos64 ? static_cast<double>(static_cast<const int64_t *>(p.pos)[at])
                             : static_cast<double>(static_cast<const int32_t *>(p.pos)[at]);
    const double turns = x * p.freqs[j] * 0.15915494309189535;  // 1 / 2 pi
    double s, c;
    sincospi(2.0 * (turns - rint(turns)), &s, &c);
    cs[e] = make_float2(static_cast<float>(c * p.scale), static_cast<float>(s * p.scale * p.sign));
  }
  __syncthreads();

  constexpr int E = HALF ? V : 2 * V;  // elements of an access
  typedef typename RotVec<T, E>::type vec;
  const int rot_items = p.pairs / V;
  const int items = rot_items + (p.D - 2 * p.pairs) / E;
  const uint32_t n = static_cast<uint32_t>(left) * p.heads * items;
  for (uint32_t i = threadIdx.x; i < n; i += kRotThreads) {
    const uint32_t th = div_by(i, p.by_items);
    const int c = i - th * items;
    const int t = div_by(th, p.by_heads);
    const int h = th - t * p.heads;
    const bool is_k = h >= p.Hq;
    const int64_t row = tok0 + t;
    const T *x = is_k ? static_cast<const T *>(p.k) + row * p.k_tok + (h - p.Hq) * p.k_head
                      : static_cast<const T *>(p.q) + row * p.q_tok + h * p.q_head;
    T *o = is_k ? static_cast<T *>(p.ko) + (row * (p.heads - p.Hq) + (h - p.Hq)) * p.D
                : static_cast<T *>(p.qo) + (row * p.Hq + h) * p.D;
    if (c >= rot_items) {
      const int d = 2 * p.pairs + (c - rot_items) * E;
      *reinterpret_cast<vec *>(o + d) = *reinterpret_cast<const vec *>(x + d);
      continue;
    }
    const float2 *turn = cs + t * p.pairs + c * V;
    T u[2 * V];
    if constexpr (HALF) {
      *reinterpret_cast<vec *>(u) = *reinterpret_cast<const vec *>(x + c * V);
      *reinterpret_cast<vec *>(u + V) = *reinterpret_cast<const vec *>(x + p.pairs + c * V);
    } else if constexpr (V == 1) {
      u[0] = x[2 * c];
      u[1] = x[2 * c + 1];
    } else {
      *reinterpret_cast<vec *>(u) = *reinterpret_cast<const vec *>(x + c * E);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int iu = HALF ? e : 2 * e, iw = HALF ? V + e : 2 * e + 1;
      const float a = rot_load<T>(u[iu]), b = rot_load<T>(u[iw]);
      const float2 r = turn[e];
      u[iu] = static_cast<T>(a * r.x - b * r.y);
      u[iw] = static_cast<T>(a * r.y + b * r.x);
    }
    if constexpr (HALF) {
      *reinterpret_cast<vec *>(o + c * V) = *reinterpret_cast<const vec *>(u);
      *reinterpret_cast<vec *>(o + p.pairs + c * V) = *reinterpret_cast<const vec *>(u + V);
    } else if constexpr (V == 1) {
      o[2 * c] = u[0];
      o[2 * c + 1] = u[1];
    } else {
      *reinterpret_cast<vec *>(o + c * E) = *reinterpret_cast<const vec *>(u);
    }
  }
}

template <typename T>
static int launch_rotary(const pkv_rotary_args *a, RotParams &p, hipStream_t st) {
  constexpr int W = 16 / sizeof(T);  // elements of 16 bytes
  auto aligned = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  bool vec = aligned(a->q) && aligned(a->q_out) && a->q_tok_stride % W == 0 && a->q_head_stride % W == 0 &&
             a->head_dim % W == 0;
  if (a->num_heads_k)
    vec = vec && aligned(a->k) && aligned(a->k_out) && a->k_tok_stride % W == 0 && a->k_head_stride % W == 0;
  vec = vec && (a->interleaved ? 2 * p.pairs : p.pairs) % W == 0;
  // items of one head: its pairs, then its copied columns
  const int V = !vec ? 1 : a->interleaved ? W / 2 : W;
  const int E = !vec ? (a->interleaved ? 2 : 1) : W;
  p.by_items = fast_div(p.pairs / V + (p.D - 2 * p.pairs) / E);
  void (*k)(RotParams) = nullptr;
  if (a->interleaved)
    k = vec ? rotary_kernel<T, W / 2, false> : rotary_kernel<T, 1, false>;
  else
    k = vec ? rotary_kernel<T, W, true> : rotary_kernel<T, 1, true>;
  // a launch counts its threads in 32 bits
  constexpr int64_t kMost = 0xffffffffll / kRotThreads;
  for (; p.row0 < p.rows; p.row0 += kMost * p.tokens) {
    const int64_t left = (p.rows - p.row0 + p.tokens - 1) / p.tokens;
    hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(left < kMost ? left : kMost)), dim3(kRotThreads),
                       sizeof(float2) * p.tokens * p.pairs, st, p);
    if (const int rc = check_launch("rotary_kernel")) return rc;
  }
  return PKV_OK;
}

}  // namespace pkv

using namespace pkv;

extern "C" int pkv_rotary(const pkv_rotary_args *a, pkv_stream_t stream) {
  if (!a) return fail(PKV_ERR_INVALID, "rotary: NULL argument");
  if (a->rows < 0 || a->num_heads_q < 0 || a->num_heads_k < 0 || a->head_dim <= 0)
    return fail(PKV_ERR_INVALID, "rotary: bad sizes");
  if (a->rows == 0 || a->num_heads_q + a->num_heads_k == 0) return PKV_OK;
  if ((a->num_heads_q && (!a->q || !a->q_out)) || (a->num_heads_k && (!a->k || !a->k_out)) || !a->pos || !a->freqs)
    return fail(PKV_ERR_INVALID, "rotary: NULL argument");
  if (a->num_axes < 1 || a->num_axes > PKV_ROTARY_MAX_AXES)
    return fail(PKV_ERR_INVALID, "rotary: %d axes (1 to %d)", a->num_axes, PKV_ROTARY_MAX_AXES);
  if (a->head_dim % 2) return fail(PKV_ERR_INVALID, "rotary: head_dim (%d) must be even", a->head_dim);
  RotParams p{};
  int pairs = 0;
  for (int i = 0; i < PKV_ROTARY_MAX_AXES; ++i) {
    if (i < a->num_axes) {
      if (a->axis_pairs[i] < 0 || a->axis_pairs[i] > kRotMaxPairs)
        return fail(PKV_ERR_INVALID, "rotary: bad pairs of axis %d", i);
      pairs += a->axis_pairs[i];
    }
    p.axis_end[i] = pairs;
  }
  if (pairs < 1 || 2 * pairs > a->head_dim || pairs > kRotMaxPairs)
    return fail(PKV_ERR_INVALID, "rotary: %d pairs in heads of %d (at most %d)", pairs, a->head_dim, kRotMaxPairs);
  if (a->head_dim > 0x10000 || a->num_heads_q > 0x8000 || a->num_heads_k > 0x8000)
    return fail(PKV_ERR_UNSUPPORTED, "rotary: heads too large");
  p.q = a->q; p.k = a->k; p.qo = a->q_out; p.ko = a->k_out;
  p.pos = a->pos; p.pos64 = a->pos_is_int64 ? 1 : 0; p.pos_row = a->num_axes;
  p.freqs = a->freqs;
  p.rows = a->rows;
  p.q_tok = a->q_tok_stride; p.q_head = a->q_head_stride;
  p.k_tok = a->k_tok_stride; p.k_head = a->k_head_stride;
  p.Hq = a->num_heads_q;
  p.heads = a->num_heads_q + a->num_heads_k;
  p.D = a->head_dim;
  p.pairs = pairs;
  p.n_axes = a->num_axes;
  p.scale = a->scale;
  p.sign = a->inverse ? -1.0f : 1.0f;
  // as many tokens as give every thread one angle, fewer where the launch would
  // leave compute units without a workgroup
  int64_t tokens = kRotThreads / pairs;
  if (tokens > a->rows / 1024) tokens = a->rows / 1024;
  p.tokens = static_cast<int>(tokens < 1 ? 1 : tokens);
  if (static_cast<int64_t>(p.tokens) * p.heads * p.D > 0x7fffffff)
    return fail(PKV_ERR_UNSUPPORTED, "rotary: heads too large");
  p.by_heads = fast_div(p.heads);
  p.by_pairs = fast_div(pairs);
  switch (a->dtype) {
    case PKV_DTYPE_BF16: return launch_rotary<__bf16>(a, p, as_stream(stream));
    case PKV_DTYPE_FP16: return launch_rotary<_Float16>(a, p, as_stream(stream));
    case PKV_DTYPE_FP32: return launch_rotary<float>(a, p, as_stream(stream));
    default: return fail(PKV_ERR_INVALID, "rotary: dtype %d", a->dtype);
  }
}
