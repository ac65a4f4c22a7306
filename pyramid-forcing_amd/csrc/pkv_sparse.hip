// Attention over chosen blocks of the cache: the mean key of every block, the
// blocks that each tile of queries scores highest, and the softmax attention
// of the tile over those blocks alone.  A tile is block_q tokens times the
// query heads that share a KV head: all of its rows read the same keys.
//
// Ragged sequences need no prefix sums: sequence s that begins at row c has
// its blocks at rows c / block + s and following, which leaves room for
// ceil(length / block) of them whatever the lengths (floor((c + n) / b) -
// floor(c / b) + 1 >= ceil(n / b)), and query sequences their tiles likewise.

#include <type_traits>

#include "pkv_common.h"

namespace pkv {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr int kMaxTopk = 1024;
constexpr int kMaxBlockK = 1024;
constexpr int kMaxRows = 256;  // query rows of a tile
constexpr int kSub = 64;       // keys: blocks are multiples of it

// Consecutive workgroups go round the 8 XCDs; renumbered, XCD x runs a
// contiguous range, so that the tiles of one KV head share its L2.
__device__ inline int xcd_order(int i, int n) {
  const int x = i & 7, base = n >> 3, rem = n & 7;
  return x * base + min(x, rem) + (i >> 3);
}

template <bool F16>
__device__ inline float elem_f32(uint16_t b) {
  if constexpr (F16) return static_cast<float>(__builtin_bit_cast(_Float16, b));
  else return bf16_to_f32(b);
}

// Rows [begin, begin + n) of sequence s, within a buffer of `total` rows
// whatever cu says.
struct Span {
  int begin, n;
};
__device__ inline Span seq_span(const int32_t *cu, int s, int total) {
  const int a = min(max(cu[s], 0), total);
  return {a, min(max(cu[s + 1], a), total) - a};
}
// of them, the keys that are in use
__device__ inline Span key_span(const int32_t *cu, const int32_t *used, int s, int total) {
  Span x = seq_span(cu, s, total);
  if (used) x.n = min(x.n, max(used[s], 0));
  return x;
}

// ---- block means -----------------------------------------------------------
// One wave per block and head: lane i takes 8 columns of every 64 / (D / 8)-th
// key in 16-byte reads, all in flight together, then the lanes of a column are
// added.  Sums in fp32, 16 keys a lane before the lanes are joined.
struct MeansParams {
  const uint16_t *k;
  float *means;
  const int32_t *cu, *used;
  int64_t total_rows;
  int64_t tok, head;
  int S, H, bk, last, total_k;
};

template <int D, bool F16>
__global__ void __launch_bounds__(256) block_means_kernel(MeansParams p) {
  constexpr int LPR = D / 8, RPI = 64 / LPR;  // lanes of a key row, rows of a read
  const int s = blockIdx.y;
  const Span keys = key_span(p.cu, p.used, s, p.total_k);
  const int begin = keys.begin, n = keys.n;
  const int64_t first = begin / p.bk + s;
  // the rows up to the next sequence's, the last sequence's up to the end
  const int64_t end = s + 1 < p.S ? seq_span(p.cu, s + 1, p.total_k).begin / p.bk + s + 1 : p.total_rows;
  const int from = p.last > 0 ? max(0, n - p.last) / p.bk : 0;
  const int64_t to = p.last > 0 ? (n + p.bk - 1) / p.bk : end - first;
  const int lane = threadIdx.x & 63, col = 8 * (lane % LPR), sub = lane / LPR;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 4;
  for (int64_t w = static_cast<int64_t>(from) * p.H + blockIdx.x * 4 + (threadIdx.x >> 6); w < to * p.H; w += stride) {
    const int64_t j = w / p.H;
    const int h = static_cast<int>(w - j * p.H);
    const int64_t left = n - j * p.bk;
    const int cnt = left >= p.bk ? p.bk : left > 0 ? static_cast<int>(left) : 0;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const uint16_t *base = p.k + (begin + j * p.bk) * p.tok + h * p.head + col;
    for (int r0 = 0; r0 < cnt; r0 += 64) {
      uint4 v[64 / RPI];
#pragma unroll
      for (int i = 0; i < 64 / RPI; ++i) {
        const int r = r0 + i * RPI + sub;
        v[i] = r < cnt ? *reinterpret_cast<const uint4 *>(base + r * p.tok) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 64 / RPI; ++i) {
        const uint32_t wd[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[2 * e] += elem_f32<F16>(static_cast<uint16_t>(wd[e] & 0xffff));
          acc[2 * e + 1] += elem_f32<F16>(static_cast<uint16_t>(wd[e] >> 16));
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int off = LPR; off < 64; off <<= 1) acc[e] += __shfl_xor(acc[e], off);
      acc[e] = cnt > 0 ? acc[e] / static_cast<float>(cnt) : 0.0f;
    }
    if (sub == 0) {
      float *o = p.means + ((first + j) * p.H + h) * D + col;
      *reinterpret_cast<float4 *>(o) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4 *>(o + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
  }
}

// ---- block selection ---------------------------------------------------------
// Scores and choice in two launches: a tile's scores go through the workspace
// as ordered 32-bit keys (larger score, larger key), so that the launch that
// reads the means splits over blocks and tiles as it likes.
//
// The score's sums are taken in fp64: the choice is then the one of the formula
// (two blocks change places only where their scores agree to 1e-15), whatever
// the order of the sums, and v_mfma_f64_16x16x4 makes them free: 16 tiles
// by 16 blocks a wave, 2 * 16 * 16 * D operations against the 64 * D bytes that
// a block's mean is read as.
struct SelectParams {
  const uint16_t *q;
  const float *means;
  int32_t *lists;
  const int32_t *cu_q, *cu_k, *used;
  int64_t tile_rows, mean_rows;
  int total_q, total_k;
  int64_t q_tok, q_head;
  int B, Hq, Hkv, G, per_head;
  int tiles;       // of the longest query sequence
  int most, nb;    // blocks of the longest key sequence; a row of keys: the next multiple of 64
  int bq, bk, topk, sink, recent, causal;
  int tile0, tile_n;  // the tiles of every sequence that this launch takes
  double *sums;    // [B, tile_n, Hkv, D] or NULL: summed by the score kernel itself
  uint32_t *keys;  // [B, tile_n, Hkv, nb]
};

struct TileKeys {
  int begin, limit, blocks;  // the key sequence's first row; keys that the tile may see; their blocks
  int64_t first;             // the first block's row in the means
};

template <typename P>
__device__ inline TileKeys tile_keys(const P &p, int b, int h, int Lq, int tile) {
  const int s = p.per_head ? b * p.Hkv + h : b;
  const Span x = key_span(p.cu_k, p.used, s, p.total_k);
  TileKeys t;
  t.begin = x.begin;
  t.limit = p.causal ? max(0, x.n - Lq + tile + 1) : x.n;
  t.blocks = (t.limit + p.bk - 1) / p.bk;
  t.first = x.begin / p.bk + s;
  return t;
}

// blocks that a tile chooses from: of its keys, within max_seqlen_k and the means
__device__ inline int chosen_from(const SelectParams &p, const TileKeys &t) {
  return static_cast<int>(min(static_cast<int64_t>(min(t.blocks, p.most)), max(p.mean_rows - t.first, static_cast<int64_t>(0))));
}

// 8 columns from d on of the tile's rows, added up in fp64
template <bool F16>
__device__ inline void sum_rows(const SelectParams &p, int b, int h, int tile, int q_begin, int Lq, int d, int from,
                                int step, double (&acc)[8]) {
  const int rows = min(p.bq, Lq - tile * p.bq) * p.G;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.0;
  for (int r = from; r < rows; r += step) {
    const int t = r / p.G, g = r - t * p.G;
    const uint4 v = *reinterpret_cast<const uint4 *>(p.q + (q_begin + static_cast<int64_t>(tile) * p.bq + t) * p.q_tok +
                                                     (h * p.G + g) * p.q_head + d);
    const uint32_t wd[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[2 * e] += static_cast<double>(elem_f32<F16>(static_cast<uint16_t>(wd[e] & 0xffff)));
      acc[2 * e + 1] += static_cast<double>(elem_f32<F16>(static_cast<uint16_t>(wd[e] >> 16)));
    }
  }
}

// the tile's summed query rows: one workgroup per (tile, KV head)
template <int D, bool F16>
__global__ void __launch_bounds__(256) tile_sums_kernel(SelectParams p) {
  constexpr int LPR = D / 8, ROWS = 256 / LPR;
  __shared__ double part[ROWS][D + 1];
  const int h = blockIdx.x % p.Hkv;
  const int rest = blockIdx.x / p.Hkv;
  const int b = rest / p.tile_n, tile = p.tile0 + rest % p.tile_n;
  const Span rows_q = seq_span(p.cu_q, b, p.total_q);
  const int q_begin = rows_q.begin, Lq = rows_q.n;
  if (tile * p.bq >= Lq) return;
  const int d = 8 * (threadIdx.x % LPR), sub = threadIdx.x / LPR;
  double acc[8];
  sum_rows<F16>(p, b, h, tile, q_begin, Lq, d, sub, ROWS, acc);
#pragma unroll
  for (int e = 0; e < 8; ++e) part[sub][d + e] = acc[e];
  __syncthreads();
  for (int c = threadIdx.x; c < D; c += 256) {
    double s = 0.0;
    for (int r = 0; r < ROWS; ++r) s += part[r][c];
    p.sums[static_cast<int64_t>(blockIdx.x) * D + c] = s;
  }
}

__device__ inline uint32_t score_key(float f) {
  if (!(f == f)) f = -INFINITY;
  const uint32_t b = __float_as_uint(f + 0.0f);  // (-0 counts as 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// grid: (block chunks, tile groups of 16, B * Hkv); 4 waves, each 16 blocks at
// a time.  A operand: lane l holds tile l % 16, columns (l / 16) * D / 4 and
// following; B operand: block l % 16, the same columns (the sum over the
// columns may run in any order); result: lane l holds block l % 16 of tiles
// l / 16 + 4 i.
template <int D, bool F16>
__global__ void __launch_bounds__(256) block_scores_kernel(SelectParams p) {
  constexpr int C = D / 4;  // columns of a lane
  const int b = blockIdx.z / p.Hkv, h = blockIdx.z % p.Hkv;
  const Span rows_q = seq_span(p.cu_q, b, p.total_q);
  const int q_begin = rows_q.begin, Lq = rows_q.n;
  const int t0 = p.tile0 + blockIdx.y * 16;
  const int last = min(min(t0 + 16, p.tile0 + p.tile_n), (Lq + p.bq - 1) / p.bq) - 1;  // the group's last tile
  if (last < t0) return;
  const TileKeys tk = tile_keys(p, b, h, Lq, last);
  const int blocks = chosen_from(p, tk);
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  int j = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16;
  if (j >= blocks) return;

  double qs[C];
  const int tile = min(t0 + i16, last);  // (lanes past the group's tiles repeat its last)
  if (p.sums) {
    const double *src =
        p.sums + ((static_cast<int64_t>(b) * p.tile_n + tile - p.tile0) * p.Hkv + h) * D + g * C;
#pragma unroll
    for (int c = 0; c < C; ++c) qs[c] = src[c];
  } else {
#pragma unroll
    for (int c = 0; c < C; c += 8) {
      double acc[8];
      sum_rows<F16>(p, b, h, tile, q_begin, Lq, g * C + c, 0, 1, acc);
#pragma unroll
      for (int e = 0; e < 8; ++e) qs[c + e] = acc[e];
    }
  }
  const int width = p.per_head ? 1 : p.Hkv;
  for (; j < blocks; j += gridDim.x * 64) {
    const int jj = min(j + i16, blocks - 1);
    const float *m = p.means + ((tk.first + jj) * width + (p.per_head ? 0 : h)) * D + g * C;
    float4 v[C / 4];
#pragma unroll
    for (int c = 0; c < C / 4; ++c) v[c] = *reinterpret_cast<const float4 *>(m + 4 * c);
    f64x4 s = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int c = 0; c < C / 4; ++c) {
      s = __builtin_amdgcn_mfma_f64_16x16x4f64(qs[4 * c], static_cast<double>(v[c].x), s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f64_16x16x4f64(qs[4 * c + 1], static_cast<double>(v[c].y), s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f64_16x16x4f64(qs[4 * c + 2], static_cast<double>(v[c].z), s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f64_16x16x4f64(qs[4 * c + 3], static_cast<double>(v[c].w), s, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = t0 + g + 4 * i;
      if (t <= last && j + i16 < blocks)
        p.keys[((static_cast<int64_t>(b) * p.tile_n + t - p.tile0) * p.Hkv + h) * p.nb + j + i16] =
            score_key(static_cast<float>(s[i]));
    }
  }
}

// The topk largest keys of a row of at most W * 64 * R, by W waves with R keys
// a lane: wave w holds keys [w * 64 * R, ...), lane l of it keys l, l + 64,
// ....  The topk-th largest is found bit by bit, counting with ballots; ties
// at it go to the lowest indices.  One row per workgroup (W > 1), or 4
// rows in 4 waves.
template <int W, int R>
__global__ void __launch_bounds__(W > 1 ? 64 * W : 256) block_choose_kernel(SelectParams p) {
  __shared__ int counts[2][W > 1 ? W : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = W > 1 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + wave;
  if (row >= static_cast<int64_t>(p.B) * p.tile_n * p.Hkv) return;
  const int h = static_cast<int>(row % p.Hkv);
  const int rest = static_cast<int>(row / p.Hkv);
  const int b = rest / p.tile_n, tile = p.tile0 + rest % p.tile_n;
  const Span rows_q = seq_span(p.cu_q, b, p.total_q);
  const int q_begin = rows_q.begin, Lq = rows_q.n;
  const int64_t first_row = q_begin / p.bq + b;
  const int have = min((Lq + p.bq - 1) / p.bq, p.tiles);
  if (tile == 0) {  // the rows behind the sequence's tiles
    const int64_t end = b + 1 < p.B ? seq_span(p.cu_q, b + 1, p.total_q).begin / p.bq + b + 1 : p.tile_rows;
    for (int64_t r = first_row + max(have, 0); r < end; ++r)
      for (int e = W > 1 ? static_cast<int>(threadIdx.x) : lane; e < p.topk; e += W > 1 ? 64 * W : 64)
        p.lists[(r * p.Hkv + h) * p.topk + e] = -1;
  }
  if (tile >= have) return;
  const TileKeys tk = tile_keys(p, b, h, Lq, tile);
  const int n = chosen_from(p, tk);
  const uint32_t *src = p.keys + row * p.nb;
  const int base = W > 1 ? wave * 64 * R : 0;
  uint32_t key[R];  // 0: no such block
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = base + r * 64 + lane;
    key[r] = j < n ? src[j] : 0u;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = base + r * 64 + lane;
    if (j < n && (j < p.sink || j >= n - p.recent)) key[r] = 0xffffffffu;
  }
  int which = 0;
  // over the row: how many keys are at least x
  auto count = [&](uint32_t x) {
    int c = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) c += __popcll(__builtin_amdgcn_ballot_w64(key[r] >= x));
    if constexpr (W > 1) {
      if (lane == 0) counts[which][wave] = c;
      __syncthreads();
      c = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) c += counts[which][w];
      which ^= 1;
    }
    return c;
  };
  const int want = min(p.topk, n);
  uint32_t at = 1;  // the want-th largest key
  int ties = W * 64 * R;  // how many of the keys equal to it are chosen
  if (n > p.topk) {
    at = 0;
    int reached = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t x = at | (1u << bit);
      const int c = count(x);
      if (c >= want) {
        at = x;
        reached = c;
        if (c == want) break;
      }
    }
    if (reached > want) ties = want - (at == 0xffffffffu ? 0 : count(at + 1));
  }
  int32_t *out = p.lists + ((first_row + tile) * p.Hkv + h) * p.topk;
  int pos = 0, tied = 0;
  if constexpr (W > 1) {  // those of the waves before
    int above = 0, equal = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      above += __popcll(__builtin_amdgcn_ballot_w64(key[r] > at));
      equal += __popcll(__builtin_amdgcn_ballot_w64(key[r] == at));
    }
    __syncthreads();
    if (lane == 0) {
      counts[0][wave] = above;
      counts[1][wave] = equal;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      pos += counts[0][w];
      tied += counts[1][w];
    }
    pos += min(tied, ties);
  }
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint64_t eq = __builtin_amdgcn_ballot_w64(key[r] == at);
    const bool take = key[r] > at || (key[r] == at && tied + __popcll(eq & below) < ties);
    const uint64_t taken = __builtin_amdgcn_ballot_w64(take);
    if (take) out[pos + __popcll(taken & below)] = base + r * 64 + lane;
    pos += __popcll(taken);
    tied += __popcll(eq);
  }
  for (int e = want + (W > 1 ? static_cast<int>(threadIdx.x) : lane); e < p.topk; e += W > 1 ? 64 * W : 64) out[e] = -1;
}

// ---- attention over the listed blocks -----------------------------------------
struct BlockAttnParams {
  const uint16_t *q, *k, *v;
  uint16_t *o;
  float *lse;
  const int32_t *lists, *cu_q, *cu_k, *used;
  int total_q, total_k;
  int64_t q_tok, q_head, kv_tok, kv_head, o_tok, o_head;
  int B, Hq, Hkv, G, per_head;
  int tiles, items;  // tiles of the longest sequence; B * Hkv * tiles
  int bq, bk, topk, causal;
  float scale_log2;
  int splits;        // workgroups of an item
  float *part;       // splits > 1: [items, splits, 32, D + 4]
};

template <int N>
__device__ inline void wait_copies() {  // vmcnt(N) alone
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
__device__ inline void wait_reads() {  // lgkmcnt(0) alone
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

template <bool F16>
__device__ inline f32x16 mfma16(uint4 a, uint4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

template <bool F16>
struct Elem8 {
  typedef std::conditional_t<F16, _Float16, __bf16> type;
  typedef type x4 __attribute__((ext_vector_type(4)));
  typedef type x8 __attribute__((ext_vector_type(8)));
};

__device__ inline i16x4 lds_read_tr(const char *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)((lds_char *)p));
}
__device__ inline float both_max(float x) {  // over lanes l and l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float both_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Where a K or V row's 16-byte chunk c lies in its LDS row: fragment reads
// of 32 rows (K) and transpose reads of 4 rows (V) then spread over the banks.
template <int D>
__device__ inline int k_chunk(int row, int c) { return c ^ (row & (D / 8 - 1)); }
template <int D>
__device__ inline int v_chunk(int row, int c) { return c ^ (D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1)); }

// One wave's copy of 64 / (D / 8) consecutive key rows into LDS at byte
// address lds (uniform), the chunks in the order that `voff` (this lane's
// source byte, relative to base) says; rows past `bytes` become zero.
__device__ inline void copy_rows(const uint16_t *base, int64_t bytes, uint32_t lds, int voff) {
  const uint64_t addr = reinterpret_cast<uint64_t>(base);
  i32x4 rsrc;
  // (uniform values, which the compiler may hold in vector registers)
  rsrc[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(addr & 0xffffffffu));
  rsrc[1] = __builtin_amdgcn_readfirstlane(static_cast<int>((addr >> 32) & 0xffffu));
  rsrc[2] = __builtin_amdgcn_readfirstlane(static_cast<int>(bytes));
  rsrc[3] = 0x00020000;
  // (the copies are inline assembly so that the compiler inserts no wait of its
  // own for them before LDS reads; every wait for them is explicit)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds), "v"(voff), "s"(rsrc) : "memory", "m0");
#pragma clang diagnostic pop
}

// The valid entries of a tile's list, each once, into LDS: list[0 .. return).
// Every thread of the workgroup calls it; scratch: 2 ints.
template <int THREADS>
__device__ int load_list(const int32_t *src, int topk, int blocks, int *list, int *scratch) {
  constexpr int PER = (kMaxTopk + THREADS - 1) / THREADS;
  const int tid = threadIdx.x;
  if (tid < 2) scratch[tid] = 0;
  for (int e = tid; e < topk; e += THREADS) list[e] = src[e];
  __syncthreads();
  auto valid = [&](int x) { return x >= 0 && x < blocks; };
  // ascending entries, then none: what a selection writes
  int n = 0, odd = 0;
  for (int e = tid; e < topk; e += THREADS) {
    const int x = list[e];
    if (valid(x)) {
      ++n;
      if (e > 0 && !(valid(list[e - 1]) && list[e - 1] < x)) odd = 1;
    }
  }
  if (n) atomicAdd(&scratch[0], n);
  if (odd) scratch[1] = 1;
  __syncthreads();
  n = scratch[0];
  if (!scratch[1]) return n;
  // otherwise an entry is kept where no earlier one equals it; its place is the
  // number of kept entries before it
  bool keep[PER];
  int x[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = tid + i * THREADS;
    keep[i] = e < topk && valid(list[e]);
    x[i] = keep[i] ? list[e] : -1;
    for (int j = 0; keep[i] && j < e; ++j) keep[i] = list[j] != x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (tid + i * THREADS < topk) list[tid + i * THREADS] = keep[i] ? 1 : 0;
  __syncthreads();
  int at[PER];
  int total = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    at[i] = 0;
    if (keep[i])
      for (int j = 0; j < tid + i * THREADS; ++j) at[i] += list[j];
  }
  for (int j = 0; j < topk; ++j) total += list[j];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (keep[i]) list[at[i]] = x[i];
  __syncthreads();
  return total;
}

// The softmax state of one wave's 32 query rows (lane l and l ^ 32: row l % 32)
// and their part of O^T: register i of o[db] is column 32 db + 8 (i / 4) + 4
// (l / 32) + i % 4.
template <int D>
struct RowState {
  f32x16 o[D / 32];
  float m, l;
};

// How far (log2) a row's scores may rise above its reference before O is
// rescaled: probabilities stay below 2^8, and the rescale, which most tiles
// do not need, is rare.
constexpr float kSlack = 8.0f;

// One wave's step over NK * 32 keys in LDS (K and V rows from kt / vt): S^T =
// K Q^T, the probabilities against the row's moving reference, O^T += V^T P^T.
// The first `keys` keys count.
template <int D, int NK, bool F16>
__device__ inline void attend_step(const char *kt, const char *vt, const uint4 (&qf)[D / 16], int keys, float c,
                                   RowState<D> &st) {
  constexpr int ROW = 2 * D;
  const int lane = threadIdx.x & 63, lq = lane & 31, hf = lane >> 5;
  f32x16 s[NK];
#pragma unroll
  for (int kb = 0; kb < NK; ++kb) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
      const int row = 32 * kb + lq;
      const uint4 a = *reinterpret_cast<const uint4 *>(kt + row * ROW + 16 * k_chunk<D>(row, 2 * x + hf));
      s[kb] = mfma16<F16>(a, qf[x], s[kb]);
    }
  }
  if (keys < 32 * NK) {
    asm volatile("");  // (kept a branch: whole tiles skip the compares)
#pragma unroll
    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (32 * kb + 8 * (i / 4) + 4 * hf + i % 4 >= keys) s[kb][i] = -INFINITY;
  }
  float t = s[0][0];
#pragma unroll
  for (int kb = 0; kb < NK; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) t = fmaxf(t, s[kb][i]);
  t = both_max(t) * c;
  // (the first keys that do not score -inf set the reference)
  const bool raise = t > st.m + kSlack || (st.m == -INFINITY && t > -INFINITY);
  if (__builtin_amdgcn_ballot_w64(raise) != 0) {
    const float m = raise ? t : st.m;
    const float f = raise ? __builtin_amdgcn_exp2f(st.m - m) : 1.0f;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[db][i] *= f;
    st.l *= f;
    st.m = m;
  }
  // P is rounded to the inputs' 16-bit type for the matrix product (half a unit
  // in the last place of each probability, as O's own rounding); the row sum
  // takes the unrounded ones.
  const float ref = st.m == -INFINITY ? 0.0f : st.m;
  typename Elem8<F16>::x8 pb[2 * NK];
#pragma unroll
  for (int kb = 0; kb < NK; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = __builtin_amdgcn_exp2f(fmaf(s[kb][i], c, -ref));
      st.l += e;
      pb[2 * kb + i / 8][i % 8] = static_cast<typename Elem8<F16>::type>(e);
    }
  // V^T fragment: lane j of each 16 addresses V[k0 + j / 4][d0 + 4 (j % 4)] and
  // receives one column of the four keys
  const int vr = 4 * hf + ((lane & 15) >> 2), vc = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
  for (int ks = 0; ks < 2 * NK; ++ks)
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      const int r0 = 16 * ks + vr;
      const char *p0 = vt + r0 * ROW + 16 * v_chunk<D>(r0, 4 * db + vc / 8) + 2 * (vc % 8);
      const i16x4 a8[2] = {lds_read_tr(p0), lds_read_tr(p0 + 8 * ROW)};  // (rows 8 apart lie alike)
      st.o[db] = mfma16<F16>(__builtin_bit_cast(uint4, a8), __builtin_bit_cast(uint4, pb[ks]), st.o[db]);
    }
}

struct AttnTile {
  int b, h, q_begin, Lq, tok0, rows, nsub;
  TileKeys tk;
};

// item -> its tile; false where the sequence has no such tile
__device__ inline bool attn_tile(const BlockAttnParams &p, int item, AttnTile &t) {
  const int seq = item / p.tiles, tile = item - seq * p.tiles;
  t.b = seq / p.Hkv;
  t.h = seq - t.b * p.Hkv;
  const Span q = seq_span(p.cu_q, t.b, p.total_q);
  t.q_begin = q.begin;
  t.Lq = q.n;
  t.tok0 = tile * p.bq;
  if (t.tok0 >= t.Lq) return false;
  t.rows = min(p.bq, t.Lq - t.tok0) * p.G;
  t.tk = tile_keys(p, t.b, t.h, t.Lq, tile);
  return true;
}

__device__ inline const int32_t *tile_list(const BlockAttnParams &p, const AttnTile &t) {
  const int64_t row = t.q_begin / p.bq + t.b + t.tok0 / p.bq;
  return p.lists + (row * p.Hkv + t.h) * p.topk;
}

template <int D>
__device__ inline void load_query(const BlockAttnParams &p, const AttnTile &t, int r, uint4 (&qf)[D / 16]) {
  const int hf = (threadIdx.x & 63) >> 5;
  const int tok = r / p.G, g = r - tok * p.G;
  const uint16_t *src =
      p.q + (t.q_begin + static_cast<int64_t>(t.tok0) + tok) * p.q_tok + (t.h * p.G + g) * p.q_head + 8 * hf;
#pragma unroll
  for (int x = 0; x < D / 16; ++x)
    qf[x] = r < t.rows ? *reinterpret_cast<const uint4 *>(src + 16 * x) : make_uint4(0, 0, 0, 0);
}

// 1 / the row sum, as the ragged attention has it: a row without keys is 0, one
// whose keys all score -inf NaN
__device__ inline float inv_sum(float l, bool keys) { return l > 0.0f || l != l ? 1.0f / l : (keys ? INFINITY : 0.0f); }

// O of row r (this lane's), from O^T / l
template <int D, bool F16>
__device__ inline void store_rows(const BlockAttnParams &p, const AttnTile &t, int r, const RowState<D> &st, float l,
                                  bool keys) {
  const int lane = threadIdx.x & 63, hf = lane >> 5;
  if (r >= t.rows) return;
  const int tok = r / p.G, g = r - tok * p.G, head = t.h * p.G + g;
  const int64_t row = t.q_begin + static_cast<int64_t>(t.tok0) + tok;
  uint16_t *o = p.o + row * p.o_tok + head * p.o_head;
  const float inv = inv_sum(l, keys);
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      typename Elem8<F16>::x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = static_cast<typename Elem8<F16>::type>(st.o[db][4 * i + e] * inv);
      *reinterpret_cast<typename Elem8<F16>::x4 *>(o + 32 * db + 8 * i + 4 * hf) = v;
    }
  if (p.lse && hf == 0)
    p.lse[static_cast<int64_t>(head) * p.total_q + row] = l > 0.0f || l != l ? (st.m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

// Tiles of up to 32 W rows: W waves of 32 rows, the keys in steps of 64 through
// two LDS buffers that all waves share.
template <int D, int W, bool F16>
__global__ void __launch_bounds__(64 * W, 2) block_attn_tile_kernel(BlockAttnParams p) {
  constexpr int ROW = 2 * D, TILE = kSub * ROW;  // bytes
  __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];  // K0 V0 K1 V1
  __shared__ int list[kMaxTopk];
  __shared__ int scratch[2];
  const int item = xcd_order(blockIdx.x, p.items);
  AttnTile t;
  if (!attn_tile(p, item, t)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = p.bk / kSub;
  const int n = __builtin_amdgcn_readfirstlane(load_list<64 * W>(tile_list(p, t), p.topk, t.tk.blocks, list, scratch)) * per;

  const int r = 32 * wave + (lane & 31);
  uint4 qf[D / 16];
  load_query<D>(p, t, r, qf);
  wait_copies<0>();  // (no load of the compiler's own is then pending among the copies)
  RowState<D> st;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) st.o[db][i] = 0.0f;
  st.m = -INFINITY;
  st.l = 0.0f;

  const int64_t head_off = p.per_head ? 0 : t.h * p.kv_head;
  const uint16_t *kp = p.k + t.tk.begin * p.kv_tok + head_off;
  const uint16_t *vp = p.v + t.tk.begin * p.kv_tok + head_off;
  constexpr int RPC = 64 / (D / 8);          // rows of a copy
  constexpr int COPIES = kSub / RPC / W;     // a wave's copies of K, and of V, per step
  const int crow = lane / (D / 8), cpos = lane % (D / 8);
  const int row_bytes = static_cast<int>(p.kv_tok) * 2;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char *)smem));
  auto first_key = [&](int s) {
    const int blk = __builtin_amdgcn_readfirstlane(list[s / per]);
    return blk * p.bk + (s % per) * kSub;
  };
  auto issue = [&](int s, int buf) {
    const int key = first_key(s);
    const int64_t left = max(0, min(kSub, t.tk.limit - key));
    const int64_t off = left > 0 ? key * p.kv_tok : 0;
    const uint32_t dst = lds0 + buf * 2 * TILE;
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int row = (wave * COPIES + i) * RPC + crow;
      const uint32_t at = dst + (wave * COPIES + i) * RPC * ROW;
      copy_rows(kp + off, left * row_bytes, at, row * row_bytes + 16 * k_chunk<D>(row, cpos));
      copy_rows(vp + off, left * row_bytes, at + TILE, row * row_bytes + 16 * v_chunk<D>(row, cpos));
    }
  };
  if (n > 0) issue(0, 0);
  for (int s = 0; s < n; ++s) {
    wait_copies<0>();
    wait_reads();
    __builtin_amdgcn_s_barrier();  // step s has arrived, and no wave reads the other buffer any more
    asm volatile("" ::: "memory");
    if (s + 1 < n) issue(s + 1, (s + 1) & 1);
    const char *kt = smem + (s & 1) * 2 * TILE;
    attend_step<D, 2, F16>(kt, kt + TILE, qf, max(0, t.tk.limit - first_key(s)), p.scale_log2, st);
  }
  store_rows<D, F16>(p, t, r, st, both_sum(st.l), n > 0);
}

// Tiles of up to 32 rows (single tokens of grouped heads): 4 waves that each
// take every fourth 32-key step of the list through a ring of their own, with
// no barrier in the loop, joined at the end.  splits > 1 divides the list over
// as many workgroups, whose parts block_attn_join_kernel adds up.
constexpr int kSmallWaves = 4;
constexpr int kRing = 2;

template <int D>
struct PartLayout {
  static constexpr int kRow = D + 4;  // O, reference, sum, whether any key was seen
  static constexpr int kFloats = 32 * kRow;
};

template <int D, bool F16>
__global__ void __launch_bounds__(64 * kSmallWaves, 1) block_attn_small_kernel(BlockAttnParams p) {
  constexpr int ROW = 2 * D, TILE = 32 * ROW;
  __shared__ __attribute__((aligned(1024))) char smem[kSmallWaves * kRing * 2 * TILE];
  __shared__ int list[kMaxTopk];
  __shared__ int scratch[2];
  __shared__ float2 ml[kSmallWaves][32];
  const int wg = xcd_order(blockIdx.x, p.items * p.splits);
  const int item = wg / p.splits, split = wg - item * p.splits;
  AttnTile t;
  if (!attn_tile(p, item, t)) return;
  const int lane = threadIdx.x & 63, lq = lane & 31, hf = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = p.bk / 32;
  const int n = __builtin_amdgcn_readfirstlane(
                    load_list<64 * kSmallWaves>(tile_list(p, t), p.topk, t.tk.blocks, list, scratch)) * per;

  uint4 qf[D / 16];
  load_query<D>(p, t, lq, qf);
  wait_copies<0>();
  RowState<D> st;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) st.o[db][i] = 0.0f;
  st.m = -INFINITY;
  st.l = 0.0f;

  const int64_t head_off = p.per_head ? 0 : t.h * p.kv_head;
  const uint16_t *kp = p.k + t.tk.begin * p.kv_tok + head_off;
  const uint16_t *vp = p.v + t.tk.begin * p.kv_tok + head_off;
  constexpr int RPC = 64 / (D / 8), COPIES = 32 / RPC;  // copies of K, and of V, per step
  const int crow = lane / (D / 8), cpos = lane % (D / 8);
  const int row_bytes = static_cast<int>(p.kv_tok) * 2;
  char *ring = smem + wave * kRing * 2 * TILE;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char *)ring));
  auto first_key = [&](int s) {
    const int blk = __builtin_amdgcn_readfirstlane(list[s / per]);
    return blk * p.bk + (s % per) * 32;
  };
  auto issue = [&](int s, int buf) {
    const int key = first_key(s);
    const int64_t left = max(0, min(32, t.tk.limit - key));
    const int64_t off = left > 0 ? key * p.kv_tok : 0;
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int row = i * RPC + crow;
      const uint32_t at = lds0 + buf * 2 * TILE + i * RPC * ROW;
      copy_rows(kp + off, left * row_bytes, at, row * row_bytes + 16 * k_chunk<D>(row, cpos));
      copy_rows(vp + off, left * row_bytes, at + TILE, row * row_bytes + 16 * v_chunk<D>(row, cpos));
    }
  };
  const int step = kSmallWaves * p.splits;
  int s = wave * p.splits + split;
  if (s < n) issue(s, 0);
  for (int it = 0; s < n; s += step, ++it) {
    wait_reads();  // the other buffer has been read
    if (s + step < n) {
      issue(s + step, (it + 1) & 1);
      wait_copies<2 * COPIES>();
    } else {
      wait_copies<0>();
    }
    asm volatile("" ::: "memory");
    const char *kt = ring + (it & 1) * 2 * TILE;
    attend_step<D, 1, F16>(kt, kt + TILE, qf, max(0, t.tk.limit - first_key(s)), p.scale_log2, st);
  }
  const float l = both_sum(st.l);

  // joined: the waves' O^T in LDS, scaled to the largest reference
  __syncthreads();
  if (hf == 0) ml[wave][lq] = make_float2(st.m, l);
  __syncthreads();
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < kSmallWaves; ++w) m = fmaxf(m, ml[w][lq].x);
  const float ref = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kSmallWaves; ++w) {
    const float2 x = ml[w][lq];
    sum += x.y == 0.0f ? 0.0f : x.y * __builtin_amdgcn_exp2f(x.x - ref);
  }
  const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(st.m - ref);
  float4 *buf = reinterpret_cast<float4 *>(smem);  // [wave][register quad][lane]
  constexpr int QUADS = D / 8;
#pragma unroll
  for (int i = 0; i < QUADS; ++i) {
    const f32x16 &o = st.o[i / 4];
    const int e = 4 * (i % 4);
    buf[(wave * QUADS + i) * 64 + lane] = make_float4(o[e] * f, o[e + 1] * f, o[e + 2] * f, o[e + 3] * f);
  }
  __syncthreads();
  const int tok = lq / p.G, g = lq - tok * p.G, head = t.h * p.G + g;
  const int64_t row = t.q_begin + static_cast<int64_t>(t.tok0) + tok;
  const bool here = lq < t.rows;
  const float inv = inv_sum(sum, n > 0);
  float *part = p.part + (static_cast<int64_t>(item) * p.splits + split) * PartLayout<D>::kFloats + lq * PartLayout<D>::kRow;
#pragma unroll
  for (int i = wave; i < QUADS; i += kSmallWaves) {
    float4 a = buf[i * 64 + lane];
#pragma unroll
    for (int w = 1; w < kSmallWaves; ++w) {
      const float4 x = buf[(w * QUADS + i) * 64 + lane];
      a = make_float4(a.x + x.x, a.y + x.y, a.z + x.z, a.w + x.w);
    }
    const int d = 8 * i + 4 * hf;
    if (!here) continue;
    if (p.splits > 1) {
      *reinterpret_cast<float4 *>(part + d) = a;
    } else {
      typename Elem8<F16>::x4 v;
      v[0] = static_cast<typename Elem8<F16>::type>(a.x * inv);
      v[1] = static_cast<typename Elem8<F16>::type>(a.y * inv);
      v[2] = static_cast<typename Elem8<F16>::type>(a.z * inv);
      v[3] = static_cast<typename Elem8<F16>::type>(a.w * inv);
      *reinterpret_cast<typename Elem8<F16>::x4 *>(p.o + row * p.o_tok + head * p.o_head + d) = v;
    }
  }
  if (!here || wave != 0 || hf != 0) return;
  if (p.splits > 1) {
    *reinterpret_cast<float4 *>(part + D) = make_float4(m, sum, n > 0 ? 1.0f : 0.0f, 0.0f);
  } else if (p.lse) {
    p.lse[static_cast<int64_t>(head) * p.total_q + row] =
        sum > 0.0f || sum != sum ? (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f : -INFINITY;
  }
}

// The parts of a tile's workgroups, added up in their order: one wave per
// query row, lane i columns i, i + 64.
template <int D, bool F16>
__global__ void __launch_bounds__(256) block_attn_join_kernel(BlockAttnParams p) {
  const int rows = p.bq * p.G;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int item = static_cast<int>(w / rows), r = static_cast<int>(w - static_cast<int64_t>(item) * rows);
  if (item >= p.items) return;
  AttnTile t;
  if (!attn_tile(p, item, t) || r >= t.rows) return;
  const int lane = threadIdx.x & 63;
  const float *part = p.part + static_cast<int64_t>(item) * p.splits * PartLayout<D>::kFloats + r * PartLayout<D>::kRow;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, part[s * PartLayout<D>::kFloats + D]);
  const float ref = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f, o[D / 64];
#pragma unroll
  for (int i = 0; i < D / 64; ++i) o[i] = 0.0f;
  bool keys = false;
  for (int s = 0; s < p.splits; ++s) {
    const float *x = part + s * PartLayout<D>::kFloats;
    const float l = x[D + 1], f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x[D] - ref);
    sum += l * f;
    keys = keys || x[D + 2] != 0.0f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] += x[64 * i + lane] * f;
  }
  const int tok = r / p.G, g = r - tok * p.G, head = t.h * p.G + g;
  const int64_t row = t.q_begin + static_cast<int64_t>(t.tok0) + tok;
  const float inv = inv_sum(sum, keys);
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    p.o[row * p.o_tok + head * p.o_head + 64 * i + lane] =
        __builtin_bit_cast(uint16_t, static_cast<typename Elem8<F16>::type>(o[i] * inv));
  if (p.lse && lane == 0)
    p.lse[static_cast<int64_t>(head) * p.total_q + row] =
        sum > 0.0f || sum != sum ? (m + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f : -INFINITY;
}

// ---- host ------------------------------------------------------------------------
// cu_seqlens are 32-bit: rows past them belong to no sequence
static int row_count(int64_t n) { return n < 0x7fffffff ? static_cast<int>(n) : 0x7fffffff; }

static bool is_16bit(int dtype) { return dtype == PKV_DTYPE_BF16 || dtype == PKV_DTYPE_FP16; }

static int check_block(int head_dim, int block_k, int dtype, const char *who) {
  if (head_dim != 64 && head_dim != 128)
    return fail(PKV_ERR_UNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", who, head_dim);
  if (block_k < kSub || block_k > kMaxBlockK || block_k % kSub)
    return fail(PKV_ERR_INVALID, "%s: block_k %d (a multiple of %d up to %d)", who, block_k, kSub, kMaxBlockK);
  if (!is_16bit(dtype)) return fail(PKV_ERR_INVALID, "%s: dtype %d (bf16 or fp16)", who, dtype);
  return PKV_OK;
}

static int check_tiles(int hq, int hkv, int block_q, int topk, int causal, const char *who) {
  if (hq <= 0 || hkv <= 0 || hq % hkv)
    return fail(PKV_ERR_INVALID, "%s: %d query heads over %d KV heads", who, hq, hkv);
  if (block_q < 1 || static_cast<int64_t>(block_q) * (hq / hkv) > kMaxRows)
    return fail(PKV_ERR_INVALID, "%s: tiles of %d tokens and %d heads (1 to %d rows)", who, block_q, hq / hkv, kMaxRows);
  if (topk < 1 || topk > kMaxTopk) return fail(PKV_ERR_INVALID, "%s: topk %d (1 to %d)", who, topk, kMaxTopk);
  if (causal && block_q != 1) return fail(PKV_ERR_UNSUPPORTED, "%s: causal needs tiles of one token (block_q 1)", who);
  return PKV_OK;
}

}  // namespace pkv

using namespace pkv;

extern "C" int pkv_block_means(const pkv_block_means_args *a, pkv_stream_t stream) {
  if (!a) return fail(PKV_ERR_INVALID, "block_means: NULL argument");
  if (a->num_seqs < 0 || a->num_heads <= 0 || a->total_k < 0 || a->last < 0 || a->max_seqlen_k < 0)
    return fail(PKV_ERR_INVALID, "block_means: bad sizes");
  if (const int rc = check_block(a->head_dim, a->block_k, a->dtype, "block_means")) return rc;
  if (a->num_seqs == 0) return PKV_OK;
  if (!a->means || !a->cu_seqlens_k || (!a->k && a->total_k > 0))
    return fail(PKV_ERR_INVALID, "block_means: NULL argument");
  if ((a->kv_tok_stride | a->kv_head_stride) & 7)
    return fail(PKV_ERR_INVALID, "block_means: strides must keep 16-byte rows aligned");
  if (a->num_seqs > 65535) return fail(PKV_ERR_UNSUPPORTED, "block_means: %d sequences (at most 65535)", a->num_seqs);
  MeansParams p{};
  p.k = a->k; p.means = a->means; p.cu = a->cu_seqlens_k; p.used = a->seqlens_k;
  p.total_rows = a->total_k / a->block_k + a->num_seqs;
  p.tok = a->kv_tok_stride; p.head = a->kv_head_stride;
  p.S = a->num_seqs; p.H = a->num_heads; p.bk = a->block_k; p.last = a->last;
  p.total_k = row_count(a->total_k);
  // a wave per block and head of a sequence of the bound's length (longer ones loop)
  const int64_t longest = a->max_seqlen_k > 0 ? a->max_seqlen_k : a->total_k;
  int64_t blocks = a->last > 0 ? a->last / a->block_k + 2 : longest / a->block_k + 1;
  if (blocks > longest / a->block_k + 1) blocks = longest / a->block_k + 1;
  int64_t grid = (blocks * a->num_heads + 3) / 4;
  if (grid > 65536) grid = 65536;
  const bool f16 = a->dtype == PKV_DTYPE_FP16;
  auto *k = a->head_dim == 128 ? (f16 ? block_means_kernel<128, true> : block_means_kernel<128, false>)
                               : (f16 ? block_means_kernel<64, true> : block_means_kernel<64, false>);
  hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(grid), a->num_seqs), dim3(256), 0, as_stream(stream), p);
  return check_launch("block_means_kernel");
}

namespace pkv {

// Tiles whose rows the score kernel adds up itself: every workgroup over the
// same tile repeats the sum, so only where it is short.
constexpr int kSumRowsInline = 16;
constexpr int64_t kSelectWorkspace = 64ll << 20;  // scores of more tiles go in several launches
constexpr int kMaxSelectBlocks = 32768;

struct SelectPlan {
  int64_t nb, tiles, tile_n, sums_bytes, bytes;
};

static int check_select(const pkv_block_select_args *a) {
  if (!a) return fail(PKV_ERR_INVALID, "block_select: NULL argument");
  if (a->num_batches < 0 || a->total_q < 0 || a->total_k < 0 || a->max_seqlen_q < 0 || a->max_seqlen_k < 0)
    return fail(PKV_ERR_INVALID, "block_select: bad sizes");
  if (const int rc = check_block(a->head_dim, a->block_k, a->dtype, "block_select")) return rc;
  if (const int rc = check_tiles(a->num_heads_q, a->num_heads_kv, a->block_q, a->topk, a->causal, "block_select"))
    return rc;
  if (a->sink_blocks < 0 || a->recent_blocks < 0 || static_cast<int64_t>(a->sink_blocks) + a->recent_blocks > a->topk)
    return fail(PKV_ERR_INVALID, "block_select: %d sink and %d recent blocks of %d", a->sink_blocks, a->recent_blocks,
                a->topk);
  if ((static_cast<int64_t>(a->max_seqlen_k) + a->block_k - 1) / a->block_k > kMaxSelectBlocks)
    return fail(PKV_ERR_UNSUPPORTED, "block_select: more than %d blocks", kMaxSelectBlocks);
  if (static_cast<int64_t>(a->num_batches) * a->num_heads_kv > 65535)
    return fail(PKV_ERR_UNSUPPORTED, "block_select: more than 65535 KV heads of all batches");
  if (a->total_q > 0x7fffffff) return fail(PKV_ERR_UNSUPPORTED, "block_select: too many query rows");
  return PKV_OK;
}

static SelectPlan select_plan(const pkv_block_select_args *a) {
  SelectPlan s{};
  s.tiles = (static_cast<int64_t>(a->max_seqlen_q) + a->block_q - 1) / a->block_q;
  s.nb = ((static_cast<int64_t>(a->max_seqlen_k) + a->block_k - 1) / a->block_k + 63) / 64 * 64;
  if (s.nb == 0) s.nb = 64;
  if (s.tiles == 0) s.tiles = 1;  // (the lists' rows are written all the same)
  const int64_t heads = static_cast<int64_t>(a->num_batches) * a->num_heads_kv;
  const bool sums = a->block_q * (a->num_heads_q / a->num_heads_kv) > kSumRowsInline;
  const int64_t per_tile = heads * (s.nb * 4 + (sums ? a->head_dim * 8 : 0));
  s.tile_n = kSelectWorkspace / (per_tile > 0 ? per_tile : 1) / 16 * 16;
  if (s.tile_n < 16) s.tile_n = 16;
  if (s.tile_n > s.tiles) s.tile_n = s.tiles;
  s.sums_bytes = sums ? heads * s.tile_n * a->head_dim * 8 : 0;
  s.bytes = s.sums_bytes + heads * s.tile_n * s.nb * 4;
  return s;
}

template <int D, bool F16>
static int launch_select(const SelectParams &p0, const SelectPlan &s, hipStream_t st) {
  const int64_t heads = static_cast<int64_t>(p0.B) * p0.Hkv;
  for (int64_t tile0 = 0; tile0 < s.tiles; tile0 += s.tile_n) {
    SelectParams p = p0;
    p.tile0 = static_cast<int>(tile0);
    p.tile_n = static_cast<int>(s.tiles - tile0 < s.tile_n ? s.tiles - tile0 : s.tile_n);
    const int64_t rows = heads * p.tile_n;
    if (p.sums) {
      hipLaunchKernelGGL((tile_sums_kernel<D, F16>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, st, p);
      if (const int rc = check_launch("tile_sums_kernel")) return rc;
    }
    const int64_t groups = (p.tile_n + 15) / 16;
    // enough workgroups for the chip, each with as many blocks as that leaves
    int64_t chunks = (s.nb + 63) / 64;
    const int64_t most = (2048 + groups * heads - 1) / (groups * heads);
    if (chunks > most) chunks = most;
    hipLaunchKernelGGL((block_scores_kernel<D, F16>),
                       dim3(static_cast<unsigned>(chunks), static_cast<unsigned>(groups), static_cast<unsigned>(heads)),
                       dim3(256), 0, st, p);
    if (const int rc = check_launch("block_scores_kernel")) return rc;
    // the fewest waves that hold a row's keys in registers
    if (s.nb <= 64 * 32) {
      auto *k = s.nb <= 64 * 2 ? block_choose_kernel<1, 2> : s.nb <= 64 * 8 ? block_choose_kernel<1, 8> : block_choose_kernel<1, 32>;
      hipLaunchKernelGGL(k, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, st, p);
    } else {
      auto *k = s.nb <= 1024 * 8 ? block_choose_kernel<16, 8> : block_choose_kernel<16, 32>;
      hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(rows)), dim3(1024), 0, st, p);
    }
    if (const int rc = check_launch("block_choose_kernel")) return rc;
  }
  return PKV_OK;
}

}  // namespace pkv

extern "C" int64_t pkv_block_select_workspace_size(const pkv_block_select_args *a) {
  if (!a || check_select(a) || a->num_batches == 0) return 0;
  return select_plan(a).bytes;
}

extern "C" int pkv_block_select(const pkv_block_select_args *a, void *workspace, int64_t workspace_bytes,
                                pkv_stream_t stream) {
  if (const int rc = check_select(a)) return rc;
  if (a->num_batches == 0) return PKV_OK;
  if (!a->lists || !a->cu_seqlens_q || !a->cu_seqlens_k || !a->means || (!a->q && a->total_q > 0))
    return fail(PKV_ERR_INVALID, "block_select: NULL argument");
  if ((a->q_tok_stride | a->q_head_stride) & 7)
    return fail(PKV_ERR_INVALID, "block_select: strides must keep 16-byte rows aligned");
  const SelectPlan s = select_plan(a);
  if (!workspace || workspace_bytes < s.bytes)
    return fail(PKV_ERR_CAPACITY, "block_select: workspace of %lld bytes, %lld needed",
                static_cast<long long>(workspace_bytes), static_cast<long long>(s.bytes));
  const int64_t heads = static_cast<int64_t>(a->num_batches) * a->num_heads_kv;
  if (heads * s.tile_n > 0x7fffffff || (s.tile_n + 15) / 16 > 65535)
    return fail(PKV_ERR_UNSUPPORTED, "block_select: grid too large");
  SelectParams p{};
  p.q = a->q; p.means = a->means; p.lists = a->lists;
  p.cu_q = a->cu_seqlens_q; p.cu_k = a->cu_seqlens_k; p.used = a->seqlens_k;
  p.tile_rows = a->total_q / a->block_q + a->num_batches;
  p.mean_rows = a->total_k / a->block_k + (a->kv_per_head ? heads : a->num_batches);
  p.total_q = row_count(a->total_q); p.total_k = row_count(a->total_k);
  p.q_tok = a->q_tok_stride; p.q_head = a->q_head_stride;
  p.B = a->num_batches; p.Hq = a->num_heads_q; p.Hkv = a->num_heads_kv;
  p.G = a->num_heads_q / a->num_heads_kv;
  p.per_head = a->kv_per_head ? 1 : 0;
  p.tiles = static_cast<int>((static_cast<int64_t>(a->max_seqlen_q) + a->block_q - 1) / a->block_q);
  p.most = static_cast<int>((static_cast<int64_t>(a->max_seqlen_k) + a->block_k - 1) / a->block_k);
  p.nb = static_cast<int>(s.nb);
  p.bq = a->block_q; p.bk = a->block_k; p.topk = a->topk; p.sink = a->sink_blocks; p.recent = a->recent_blocks;
  p.causal = a->causal ? 1 : 0;
  p.sums = s.sums_bytes ? static_cast<double *>(workspace) : nullptr;
  p.keys = reinterpret_cast<uint32_t *>(static_cast<char *>(workspace) + s.sums_bytes);
  hipStream_t st = as_stream(stream);
  const bool f16 = a->dtype == PKV_DTYPE_FP16;
  if (a->head_dim == 128) return f16 ? launch_select<128, true>(p, s, st) : launch_select<128, false>(p, s, st);
  return f16 ? launch_select<64, true>(p, s, st) : launch_select<64, false>(p, s, st);
}

namespace pkv {

static int check_attn(const pkv_block_attn_args *a) {
  if (!a) return fail(PKV_ERR_INVALID, "block_attn: NULL argument");
  if (a->num_batches < 0 || a->total_q < 0 || a->total_k < 0 || a->max_seqlen_q < 0)
    return fail(PKV_ERR_INVALID, "block_attn: bad sizes");
  if (const int rc = check_block(a->head_dim, a->block_k, a->dtype, "block_attn")) return rc;
  if (const int rc = check_tiles(a->num_heads_q, a->num_heads_kv, a->block_q, a->topk, a->causal, "block_attn")) return rc;
  if (!(a->softmax_scale > 0.0f) || a->softmax_scale > 3.0e38f)
    return fail(PKV_ERR_INVALID, "block_attn: softmax_scale must be above 0 and finite");
  const int64_t items = static_cast<int64_t>(a->num_batches) * a->num_heads_kv *
                        ((static_cast<int64_t>(a->max_seqlen_q) + a->block_q - 1) / a->block_q);
  if (items > 0x1fffffff || a->total_q > 0x7fffffff) return fail(PKV_ERR_UNSUPPORTED, "block_attn: grid too large");
  return PKV_OK;
}

static int64_t attn_items(const pkv_block_attn_args *a) {
  return static_cast<int64_t>(a->num_batches) * a->num_heads_kv *
         ((static_cast<int64_t>(a->max_seqlen_q) + a->block_q - 1) / a->block_q);
}

// Workgroups of a small tile: as many as give the chip one each, but at least
// four 32-key steps a wave.
static int attn_splits(const pkv_block_attn_args *a) {
  if (a->block_q * (a->num_heads_q / a->num_heads_kv) > 32) return 1;
  const int64_t items = attn_items(a);
  if (items == 0) return 1;
  int64_t s = 256 / items;
  const int64_t most = static_cast<int64_t>(a->topk) * (a->block_k / 32) / (4 * kSmallWaves);
  if (s > most) s = most;
  return static_cast<int>(s < 1 ? 1 : s);
}

template <int D, bool F16>
static int launch_block_attn(const BlockAttnParams &p, hipStream_t st) {
  const int rows = p.bq * p.G;
  if (rows <= 32) {
    hipLaunchKernelGGL((block_attn_small_kernel<D, F16>), dim3(p.items * p.splits), dim3(64 * kSmallWaves), 0, st, p);
    if (const int rc = check_launch("block_attn_small_kernel")) return rc;
    if (p.splits == 1) return PKV_OK;
    const int64_t waves = static_cast<int64_t>(p.items) * rows;
    hipLaunchKernelGGL((block_attn_join_kernel<D, F16>), dim3(static_cast<unsigned>((waves + 3) / 4)), dim3(256), 0, st, p);
    return check_launch("block_attn_join_kernel");
  }
  if (rows <= 64)
    hipLaunchKernelGGL((block_attn_tile_kernel<D, 2, F16>), dim3(p.items), dim3(128), 0, st, p);
  else if (rows <= 128)
    hipLaunchKernelGGL((block_attn_tile_kernel<D, 4, F16>), dim3(p.items), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((block_attn_tile_kernel<D, 8, F16>), dim3(p.items), dim3(512), 0, st, p);
  return check_launch("block_attn_tile_kernel");
}

}  // namespace pkv

extern "C" int64_t pkv_block_attn_workspace_size(const pkv_block_attn_args *a) {
  if (!a || check_attn(a)) return 0;
  const int s = attn_splits(a);
  return s > 1 ? attn_items(a) * s * 32 * (a->head_dim + 4) * 4 : 0;
}

extern "C" int pkv_block_attn(const pkv_block_attn_args *a, void *workspace, int64_t workspace_bytes,
                              pkv_stream_t stream) {
  if (const int rc = check_attn(a)) return rc;
  if (a->num_batches == 0 || a->max_seqlen_q == 0 || a->total_q == 0) return PKV_OK;
  if (!a->q || !a->o || !a->lists || !a->cu_seqlens_q || !a->cu_seqlens_k || ((!a->k || !a->v) && a->total_k > 0))
    return fail(PKV_ERR_INVALID, "block_attn: NULL argument");
  if (((a->q_tok_stride | a->q_head_stride | a->kv_tok_stride | a->kv_head_stride) & 7) ||
      ((a->o_tok_stride | a->o_head_stride) & 3))
    return fail(PKV_ERR_INVALID, "block_attn: strides must keep 16-byte rows aligned");
  // buffer offsets within one step of keys are 32-bit
  if (a->kv_tok_stride < 0 || a->kv_tok_stride * 2 * kSub > 0x7fffffff)
    return fail(PKV_ERR_UNSUPPORTED, "block_attn: kv token stride too large");
  const int64_t need = pkv_block_attn_workspace_size(a);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(PKV_ERR_CAPACITY, "block_attn: workspace of %lld bytes, %lld needed",
                static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  BlockAttnParams p{};
  p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o; p.lse = a->lse; p.lists = a->lists;
  p.cu_q = a->cu_seqlens_q; p.cu_k = a->cu_seqlens_k; p.used = a->seqlens_k;
  p.total_q = row_count(a->total_q);
  p.total_k = row_count(a->total_k);
  p.q_tok = a->q_tok_stride; p.q_head = a->q_head_stride;
  p.kv_tok = a->kv_tok_stride; p.kv_head = a->kv_head_stride;
  p.o_tok = a->o_tok_stride; p.o_head = a->o_head_stride;
  p.B = a->num_batches; p.Hq = a->num_heads_q; p.Hkv = a->num_heads_kv;
  p.G = a->num_heads_q / a->num_heads_kv;
  p.per_head = a->kv_per_head ? 1 : 0;
  p.tiles = static_cast<int>((static_cast<int64_t>(a->max_seqlen_q) + a->block_q - 1) / a->block_q);
  p.items = static_cast<int>(attn_items(a));
  p.bq = a->block_q; p.bk = a->block_k; p.topk = a->topk;
  p.causal = a->causal ? 1 : 0;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.splits = attn_splits(a);
  p.part = static_cast<float *>(workspace);
  hipStream_t st = as_stream(stream);
  const bool f16 = a->dtype == PKV_DTYPE_FP16;
  if (a->head_dim == 128) return f16 ? launch_block_attn<128, true>(p, st) : launch_block_attn<128, false>(p, st);
  return f16 ? launch_block_attn<64, true>(p, st) : launch_block_attn<64, false>(p, st);
}
