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
// key in 16-byte reads, 64 keys in flight together, then the lanes of a column
// are added.  Sums in fp32: a lane's keys in turn (16 of a block of 64 at head_dim
// 128), then the lanes' in a tree.
// Bound by memory, every key read once: 36 sequences of 6,240 to 32,760 keys
// (188 MB) in 34.7 us, 5.4 TB/s (a copy of 1 GiB moves 4.8); 3 sequences of 300
// keys in 4.2, most of it the launch.  Workgroups of a sequence lie together: with
// the sequences fastest the same call took 38.8.
struct MeansParams {
  const uint16_t *k;
  float *means;
  const int32_t *cu, *used;
  int64_t total_rows;
  int64_t tok, head;
  int S, H, bk, last, total_k;
  int chunks;  // workgroups of a sequence
};

template <int D, bool F16>
__global__ void __launch_bounds__(256) block_means_kernel(MeansParams p) {
  constexpr int LPR = D / 8, RPI = 64 / LPR;  // lanes of a key row, rows of a read
  const int s = blockIdx.x / p.chunks, chunk = blockIdx.x - s * p.chunks;
  const Span keys = key_span(p.cu, p.used, s, p.total_k);
  const int begin = keys.begin, n = keys.n;
  const int64_t first = begin / p.bk + s;
  // the rows up to the next sequence's, the last sequence's up to the end
  const int64_t end = s + 1 < p.S ? seq_span(p.cu, s + 1, p.total_k).begin / p.bk + s + 1 : p.total_rows;
  // (the first sequence's also zeroes the rows before it)
  const int64_t from = p.last > 0 ? max(0, n - p.last) / p.bk : s == 0 ? -first : 0;
  const int64_t to = p.last > 0 ? (n + p.bk - 1) / p.bk : end - first;
  const int lane = threadIdx.x & 63, col = 8 * (lane % LPR), sub = lane / LPR;
  const int64_t stride = static_cast<int64_t>(p.chunks) * 4;
  for (int64_t w = chunk * 4 + (threadIdx.x >> 6); w < (to - from) * p.H; w += stride) {
    const int64_t i = w / p.H, j = from + i;
    const int h = static_cast<int>(w - i * p.H);
    const int64_t left = j < 0 ? 0 : n - j * p.bk;
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
// Scores and choice in two launches, or three with the tiles' sums: a tile's
// scores go through the workspace as ordered 32-bit keys (larger score, larger
// key), so that the launch that reads the means splits over blocks and tiles as
// it likes; or all in one launch (block_select_kernel).
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
  int chunks;         // workgroups that share a tile group's blocks
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

// 8 columns from d on of the tile's rows `from`, from + step, ..., added up in
// fp64, kAhead rows read together (rows past the last repeat it and count 0)
template <bool F16>
__device__ inline void sum_rows(const SelectParams &p, int h, int tile, const Span &q, int d, int from, int step,
                                double (&acc)[8]) {
  constexpr int kAhead = 4;
  const int rows = min(p.bq, q.n - tile * p.bq) * p.G;
  const uint16_t *base = p.q + (q.begin + static_cast<int64_t>(tile) * p.bq) * p.q_tok + h * p.G * p.q_head + d;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.0;
  for (int r0 = from; r0 < rows; r0 += kAhead * step) {
    uint4 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int r = min(r0 + i * step, rows - 1), t = r / p.G;
      v[i] = *reinterpret_cast<const uint4 *>(base + t * p.q_tok + (r - t * p.G) * p.q_head);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const uint32_t keep = r0 + i * step < rows ? 0xffffffffu : 0u;
      const uint32_t wd[4] = {v[i].x & keep, v[i].y & keep, v[i].z & keep, v[i].w & keep};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[2 * e] += static_cast<double>(elem_f32<F16>(static_cast<uint16_t>(wd[e] & 0xffff)));
        acc[2 * e + 1] += static_cast<double>(elem_f32<F16>(static_cast<uint16_t>(wd[e] >> 16)));
      }
    }
  }
}

// x + its value 16 (32) lanes away, in both
__device__ inline double add_lane16(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const auto lo = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u), static_cast<uint32_t>(u), false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32), false, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]) +
         __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
}
__device__ inline double add_lane32(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const auto lo = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(u), static_cast<uint32_t>(u), false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32), false, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]) +
         __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
}

// The tile's summed query rows: grid (tiles, Hkv, B).  468 tiles of 120 rows of
// head_dim 128 (14.4 MB) in 5.3 us: the launch, two dependent reads and the tree.
template <int D, bool F16>
__global__ void __launch_bounds__(256) tile_sums_kernel(SelectParams p) {
  constexpr int LPR = D / 8, ROWS = 256 / LPR;
  __shared__ double part[ROWS][D + 1];
  const int b = blockIdx.z, h = blockIdx.y, tile = p.tile0 + blockIdx.x;
  const Span q = seq_span(p.cu_q, b, p.total_q);
  if (tile * p.bq >= q.n) return;
  const int d = 8 * (threadIdx.x % LPR), sub = threadIdx.x / LPR;
  double acc[8];
  sum_rows<F16>(p, h, tile, q, d, sub, ROWS, acc);
#pragma unroll
  for (int e = 0; e < 8; ++e) part[sub][d + e] = acc[e];
  __syncthreads();
  if (threadIdx.x < D) {
    double s = 0.0;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) s += part[r][threadIdx.x];
    p.sums[((static_cast<int64_t>(b) * p.tile_n + blockIdx.x) * p.Hkv + h) * D + threadIdx.x] = s;
  }
}

__device__ inline uint32_t score_key(float f) {
  if (!(f == f)) f = -INFINITY;
  const uint32_t b = __float_as_uint(f + 0.0f);  // (-0 counts as 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// grid: (tile groups of 16 * block chunks, Hkv, B); 4 waves, each 16 blocks at
// a time.  A operand: lane l holds tile l % 16, columns 16 c + 4 (l / 16) + e (e
// < 4, one matrix instruction each); B operand: block l % 16, the same columns,
// so that the 4 lanes of a block read 64 bytes together (a lane's quarter of the
// row in one piece had every read touch 64 cache lines, and again for each of
// its 8 parts); result: lane l holds block l % 16 of tiles l / 16 + 4 i.
// 36 groups of 13 tiles and 98 to 512 blocks each in 8.2 us: a chain of dependent
// reads (lengths, sums, means) and 32 matrix instructions.  Four chains of those
// and the means read before the sums: 8.6.
template <int D, bool F16>
__global__ void __launch_bounds__(256) block_scores_kernel(SelectParams p) {
  constexpr int C = D / 4;  // columns of a lane
  const int b = blockIdx.z, h = blockIdx.y;
  const int group = blockIdx.x / p.chunks, chunk = blockIdx.x - group * p.chunks;
  const Span q = seq_span(p.cu_q, b, p.total_q);
  const int t0 = p.tile0 + group * 16;
  const int last = min(min(t0 + 16, p.tile0 + p.tile_n), (q.n + p.bq - 1) / p.bq) - 1;  // the group's last tile
  const TileKeys tk = tile_keys(p, b, h, q.n, last);
  if (last < t0) return;
  const int blocks = chosen_from(p, tk);
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  int j = (chunk * 4 + (threadIdx.x >> 6)) * 16;
  if (chunk * 64 >= blocks) return;

  double qs[C];
  const int tile = min(t0 + i16, last);  // (lanes past the group's tiles repeat its last)
  if (p.sums) {
    const double *src =
        p.sums + ((static_cast<int64_t>(b) * p.tile_n + tile - p.tile0) * p.Hkv + h) * D + 4 * g;
#pragma unroll
    for (int c = 0; c < C; ++c) qs[c] = src[16 * (c / 4) + c % 4];
  } else {
    // thread i sums 8 columns of tile i / (D / 8)
    __shared__ double sums[16][D + 2];
    const int mine = threadIdx.x / (D / 8), d = 8 * (threadIdx.x % (D / 8));
    if (mine < 16) {
      double acc[8];
      sum_rows<F16>(p, h, min(t0 + mine, last), q, d, 0, 1, acc);
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[mine][d + e] = acc[e];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; ++c) qs[c] = sums[i16][16 * (c / 4) + 4 * g + c % 4];
  }
  const int width = p.per_head ? 1 : p.Hkv;
  for (; j < blocks; j += p.chunks * 64) {
    const int jj = min(j + i16, blocks - 1);
    const float *m = p.means + ((tk.first + jj) * width + (p.per_head ? 0 : h)) * D + 4 * g;
    float4 v[C / 4];
#pragma unroll
    for (int c = 0; c < C / 4; ++c) v[c] = *reinterpret_cast<const float4 *>(m + 16 * c);
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

// Writes the want = min(topk, n) largest of a row's keys, ascending by index and
// padded with -1, to out.  W waves of R keys a lane take part: wave w holds keys
// [w * 64 * R, ...), lane l of it keys l, l + 64, ...; 0 where there is none.
// The want-th largest is found bit by bit, counting with ballots (at most 32 rounds
// over keys in registers, whatever topk is); ties at it go to the lowest indices.
// counts: 2 * W ints of LDS (W > 1, where the whole workgroup calls it).
template <int W, int R>
__device__ inline void choose(const uint32_t (&key)[R], int n, int topk, int32_t *out, int *counts) {
  const int lane = threadIdx.x & 63, wave = W > 1 ? threadIdx.x >> 6 : 0;
  int which = 0;
  // over the row: how many keys are at least x
  auto count = [&](uint32_t x) {
    int c = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) c += __popcll(__builtin_amdgcn_ballot_w64(key[r] >= x));
    if constexpr (W > 1) {
      if (lane == 0) counts[which * W + wave] = c;
      __syncthreads();
      c = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) c += counts[which * W + w];
      which ^= 1;
    }
    return c;
  };
  const int want = min(topk, n);
  uint32_t at = 1;        // the want-th largest key
  int ties = W * 64 * R;  // how many of the keys equal to it are chosen
  if (n > topk) {
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
      counts[wave] = above;
      counts[W + wave] = equal;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      pos += counts[w];
      tied += counts[W + w];
    }
    pos += min(tied, ties);
  }
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint64_t eq = __builtin_amdgcn_ballot_w64(key[r] == at);
    const bool take = key[r] > at || (key[r] == at && tied + __popcll(eq & below) < ties);
    const uint64_t taken = __builtin_amdgcn_ballot_w64(take);
    if (take) out[pos + __popcll(taken & below)] = (wave * R + r) * 64 + lane;
    pos += __popcll(taken);
    tied += __popcll(eq);
  }
  for (int e = want + wave * 64 + lane; e < topk; e += 64 * W) out[e] = -1;
}

// The lists' rows behind sequence b's `have` tiles, of which `first` is the first
// row, and those before the first sequence's, for KV head h
__device__ inline void clear_rows(const SelectParams &p, int b, int h, int64_t first, int have, int thread, int threads) {
  const int64_t end = b + 1 < p.B ? seq_span(p.cu_q, b + 1, p.total_q).begin / p.bq + b + 1 : p.tile_rows;
  const int64_t before = b == 0 ? first : 0;
  for (int64_t i = 0; i < before + end - first - have; ++i) {
    const int64_t r = i < before ? i : first + have + (i - before);
    for (int e = thread; e < p.topk; e += threads) p.lists[(r * p.Hkv + h) * p.topk + e] = -1;
  }
}

// A row (tile, KV head) of the lists from block_scores_kernel's keys: one per
// workgroup of W waves, or, W 1, one per wave and 4 per workgroup.  Grid: (tiles,
// Hkv, B).  468 rows of 98 to 512 keys in 5.3 us, most of it the launch and the
// rounds of the search.
template <int W, int R>
__global__ void __launch_bounds__(W > 1 ? 64 * W : 256) block_choose_kernel(SelectParams p) {
  __shared__ int counts[2 * W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.z, h = blockIdx.y, nth = W > 1 ? blockIdx.x : blockIdx.x * 4 + wave, tile = p.tile0 + nth;
  const Span q = seq_span(p.cu_q, b, p.total_q);
  const TileKeys tk = tile_keys(p, b, h, q.n, tile);
  const int64_t first_row = q.begin / p.bq + b;
  const int have = min((q.n + p.bq - 1) / p.bq, p.tiles);
  if (tile == 0)
    clear_rows(p, b, h, first_row, have, W > 1 ? static_cast<int>(threadIdx.x) : lane, W > 1 ? 64 * W : 64);
  if (tile >= have || nth >= p.tile_n) return;
  const int n = chosen_from(p, tk);
  const int64_t row = (static_cast<int64_t>(b) * p.tile_n + nth) * p.Hkv + h;
  const uint32_t *src = p.keys + row * p.nb;
  const int base = W > 1 ? wave * 64 * R : 0;
  uint32_t key[R];
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
  choose<W, R>(key, n, p.topk, p.lists + ((first_row + tile) * p.Hkv + h) * p.topk, counts);
}

// Scores and choice in one launch, where a row's blocks are few: W waves a row
// (W 1: 4 rows a workgroup, each wave by itself), grid (tiles, Hkv, B).  The row's summed queries and
// its keys lie in LDS; 4 lanes take a block's mean, 16 blocks a wave at a time,
// in vector fp64.  A row of the lists costs nb * 4 D bytes of means, which the
// rows of a sequence do not share as block_scores_kernel's 16 do: bound by what a
// compute unit reads (16 tokens of 8 KV heads, 63 to 512 blocks, in 12.5 us: the
// longest row's 262 KB at about 20 bytes a clock, and the search; 2,047 tokens of 2
// KV heads, up to 32 blocks, in 11.8).
template <int D, bool F16, int W, int R>
__global__ void __launch_bounds__(W > 1 ? 64 * W : 256) block_select_kernel(SelectParams p) {
  constexpr int ROWS = W > 1 ? 1 : 4, NB = W * 64 * R;  // rows of a workgroup, keys of a row
  constexpr int LPR = D / 8, SUB = 64 / LPR, C = D / 4;
  __shared__ double sums[ROWS][W][D];
  __shared__ uint32_t keys[ROWS][NB];
  __shared__ int counts[2 * W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slot = W > 1 ? 0 : wave, part = W > 1 ? wave : 0;
  const int b = blockIdx.z, h = blockIdx.y, tile = W > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  const Span q = seq_span(p.cu_q, b, p.total_q);
  const TileKeys tk = tile_keys(p, b, h, q.n, tile);
  const int64_t first_row = q.begin / p.bq + b;
  const int have = min((q.n + p.bq - 1) / p.bq, p.tiles);
  if (tile == 0)
    clear_rows(p, b, h, first_row, have, W > 1 ? static_cast<int>(threadIdx.x) : lane, W > 1 ? 64 * W : 64);
  if (tile >= have) return;
  const int n = chosen_from(p, tk);
  const int i16 = lane & 15, g = lane >> 4;
  const int width = p.per_head ? 1 : p.Hkv;
  const float *means = p.means + (tk.first * width + (p.per_head ? 0 : h)) * D + 4 * g;
  auto fetch = [&](int j, float4 (&v)[C / 4]) {  // (blocks past the last repeat it)
    const float *m = means + static_cast<int64_t>(min(j + i16, n - 1)) * width * D;
#pragma unroll
    for (int c = 0; c < C / 4; ++c) v[c] = *reinterpret_cast<const float4 *>(m + 16 * c);
  };
  constexpr int kAhead = 2;  // reads of 16 blocks in flight
  float4 v[kAhead][C / 4];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)  // on their way while the queries are summed
    if ((part + i * W) * 16 < n) fetch((part + i * W) * 16, v[i]);

  const int sub = part * SUB + lane / LPR;
  double acc[8];
  sum_rows<F16>(p, h, tile, q, 8 * (lane % LPR), sub, W * SUB, acc);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (LPR == 8) acc[e] += __shfl_xor(acc[e], 8);
    acc[e] = add_lane32(add_lane16(acc[e]));
  }
  if (lane < LPR)
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[slot][part][8 * lane + e] = acc[e];
  if constexpr (W > 1) {
    __syncthreads();
    if (threadIdx.x < D) {
      double x = sums[0][0][threadIdx.x];
#pragma unroll
      for (int w = 1; w < W; ++w) x += sums[0][w][threadIdx.x];
      sums[0][0][threadIdx.x] = x;
    }
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  double qs[C];
#pragma unroll
  for (int c = 0; c < C; ++c) qs[c] = sums[slot][0][16 * (c / 4) + 4 * g + c % 4];
  for (int j0 = part * 16; j0 < n; j0 += kAhead * 16 * W)
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int j = j0 + i * 16 * W;
      if (j >= n) break;
      double s0 = 0.0, s1 = 0.0;
#pragma unroll
      for (int c = 0; c < C / 4; ++c) {
        s0 = fma(qs[4 * c], static_cast<double>(v[i][c].x), s0);
        s1 = fma(qs[4 * c + 1], static_cast<double>(v[i][c].y), s1);
        s0 = fma(qs[4 * c + 2], static_cast<double>(v[i][c].z), s0);
        s1 = fma(qs[4 * c + 3], static_cast<double>(v[i][c].w), s1);
      }
      if (j + kAhead * 16 * W < n) fetch(j + kAhead * 16 * W, v[i]);
      const double s = add_lane32(add_lane16(s0 + s1));
      const int at = j + i16;
      if (g == 0 && at < n)
        keys[slot][at] = at < p.sink || at >= n - p.recent ? 0xffffffffu : score_key(static_cast<float>(s));
    }
  if constexpr (W > 1) __syncthreads();
  else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  int32_t *out = p.lists + ((first_row + tile) * p.Hkv + h) * p.topk;
  // one wave where it holds the keys: no barriers in the search (128 rows of 512
  // blocks 14.5 us, 15.4 by all eight)
  if (W == 1 || n <= 512) {
    if (W > 1 && wave > 0) return;
    constexpr int R1 = W == 1 ? R : 8;
    uint32_t key[R1];
#pragma unroll
    for (int r = 0; r < R1; ++r) key[r] = r * 64 + lane < n ? keys[slot][r * 64 + lane] : 0u;
    choose<1, R1>(key, n, p.topk, out, counts);
  } else {
    uint32_t key[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int at = (wave * R + r) * 64 + lane;
      key[r] = at < n ? keys[slot][at] : 0u;
    }
    choose<W, R>(key, n, p.topk, out, counts);
  }
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
  int tiles, items;  // tiles (groups of tiles) of the longest sequence; B * Hkv * tiles
  int group;         // tiles that a workgroup takes together
  int max_q;         // tokens of the longest sequence: later ones are left alone
  int bq, bk, topk, causal;
  float scale_log2;
  int splits;        // workgroups of an item
  int part_rows;     // rows of a part: those of the workgroup's waves
  float *part;       // splits > 1: [items, splits, part_rows, D + 4]
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
// source byte, relative to base) says; rows past `bytes` become zero.  FIRST: the
// first copy with this base and these bytes.
template <bool FIRST>
__device__ inline void copy_rows(const uint16_t *base, int64_t bytes, uint32_t lds, int voff) {
  const uint64_t addr = reinterpret_cast<uint64_t>(base);
  i32x4 rsrc;
  // (uniform values, which the compiler may hold in vector registers)
  rsrc[0] = __builtin_amdgcn_readfirstlane(static_cast<int>(addr & 0xffffffffu));
  rsrc[1] = __builtin_amdgcn_readfirstlane(static_cast<int>((addr >> 32) & 0xffffu));
  rsrc[2] = __builtin_amdgcn_readfirstlane(static_cast<int>(bytes));
  rsrc[3] = 0x00020000;
  // The copies are inline assembly so that the compiler inserts no wait of its
  // own for them before LDS reads; every wait for them is explicit.  Nor does it
  // add wait states: one is due between the write of m0 and a load into LDS, five
  // between a vector instruction's write of a scalar register (v_readfirstlane
  // above) and a memory instruction that reads it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\ts_nop %3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(voff), "s"(rsrc), "n"(FIRST ? 3 : 0)
               : "memory", "m0");
#pragma clang diagnostic pop
}
// copy(i, whether it is the first) for i < COPIES
template <int COPIES, typename F>
__device__ inline void copy_each(F copy) {
  copy(0, std::true_type());
#pragma unroll
  for (int i = 1; i < COPIES; ++i) copy(i, std::false_type());
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
  __device__ void reset() {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    m = -INFINITY;
    l = 0.0f;
  }
};

// whether the sum and all of O are numbers
template <int D>
__device__ inline bool finite(const RowState<D> &st) {
  float check = st.l;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) check = fmaf(st.o[db][i], 0.0f, check);
  return check - check == 0.0f;
}

// How far (log2) a row's scores may rise above its reference before O is
// rescaled: probabilities stay below 2^8, and the rescale, which most tiles
// do not need, is rare.
constexpr float kSlack = 8.0f;

// One wave's step over NK * 32 keys in LDS (K and V rows from kt / vt): S^T =
// K Q^T, the probabilities against the row's moving reference, O^T += V^T P^T.
// The first `keys` keys count (LANES: of each lane's row its own; a row of none
// takes no part: its probabilities are 2^(0 S - inf), which is 0 unless S is not
// finite).
template <int D, int NK, bool F16, bool LANES, bool FINE>
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
  if (LANES ? __builtin_amdgcn_ballot_w64(keys < 32 * NK && keys > 0) != 0 : keys < 32 * NK) {
    asm volatile("");  // (kept a branch: whole tiles skip the compares)
    const int some = LANES && keys <= 0 ? 32 * NK : keys;
#pragma unroll
    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (32 * kb + 8 * (i / 4) + 4 * hf + i % 4 >= some) s[kb][i] = -INFINITY;
  }
  float t = s[0][0];
#pragma unroll
  for (int kb = 0; kb < NK; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) t = fmaxf(t, s[kb][i]);
  t = both_max(t) * c;
  const bool none = LANES && keys <= 0;
  if (none) t = -INFINITY;
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
  // in the last place of each probability, as O's own rounding: the error against
  // 64 bits is 1.3 to 1.4 times that of O's rounding alone), FINE: in two such parts, a
  // second product that takes the rest; the row sum takes the unrounded ones.
  // FINE where the kernel waits for memory; where it waits for the matrix units the
  // second product costs 228 -> 297 us (tiles of 120 rows) and 55.6 -> 68 (groups of
  // single tokens), which the ragged attention does not pay either.
  const float ref = none ? INFINITY : st.m == -INFINITY ? 0.0f : st.m;
  const float cl = none ? 0.0f : c;
  typename Elem8<F16>::x8 pb[2 * NK], pl[FINE ? 2 * NK : 1];
#pragma unroll
  for (int kb = 0; kb < NK; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = __builtin_amdgcn_exp2f(fmaf(s[kb][i], cl, -ref));
      st.l += e;
      const typename Elem8<F16>::type h = static_cast<typename Elem8<F16>::type>(e);
      pb[2 * kb + i / 8][i % 8] = h;
      if constexpr (FINE) pl[2 * kb + i / 8][i % 8] = static_cast<typename Elem8<F16>::type>(e - static_cast<float>(h));
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
      if constexpr (FINE)
        st.o[db] = mfma16<F16>(__builtin_bit_cast(uint4, a8), __builtin_bit_cast(uint4, pl[ks]), st.o[db]);
    }
}

struct AttnTile {
  int b, h, q_begin, Lq, tok0, rows;
  TileKeys tk;  // of the last tile
};

// The item of workgroup i of a causal launch: the tiles with the most keys first,
// KV heads next to each other (2,047 tokens of 2 KV heads, 16 blocks each: 55.6 us,
// 68.6 in xcd_order's).
__device__ inline int causal_order(const BlockAttnParams &p, int i) {
  const int seqs = p.items / p.tiles, tile = i / seqs;
  return (i - tile * seqs) * p.tiles + (p.tiles - 1 - tile);
}

// item -> its tile; false where the sequence has no such tile
__device__ inline bool attn_tile(const BlockAttnParams &p, int item, AttnTile &t) {
  const int seq = item / p.tiles, tile = item - seq * p.tiles;
  t.b = seq / p.Hkv;
  t.h = seq - t.b * p.Hkv;
  const Span q = seq_span(p.cu_q, t.b, p.total_q);
  t.q_begin = q.begin;
  t.Lq = q.n;
  t.tok0 = tile * p.group * p.bq;
  const int left = min(t.Lq, p.max_q) - t.tok0;
  if (left <= 0) return false;
  const int tokens = min(p.group * p.bq, left);
  t.rows = tokens * p.G;
  t.tk = tile_keys(p, t.b, t.h, t.Lq, (t.tok0 + tokens - 1) / p.bq);
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

// the natural logarithm of a row's softmax sum l against the reference m (log2)
__device__ inline float log_sum(float m, float l) {
  return l > 0.0f || l != l ? (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

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
  if (p.lse && hf == 0) p.lse[static_cast<int64_t>(head) * p.total_q + row] = log_sum(st.m, l);
}

// Row r of a split item's part: O, the reference, the sum, whether any key was
// seen
template <int D>
__device__ inline float *part_row(const BlockAttnParams &p, int item, int split, int r) {
  return p.part + ((static_cast<int64_t>(item) * p.splits + split) * p.part_rows + r) * (D + 4);
}

// The copies of a step's K and V rows (STEP keys) into one of two buffers, by W
// waves together
template <int D, int W, int STEP>
struct TileCopies {
  static constexpr int ROW = 2 * D, TILE = STEP * ROW;
  static constexpr int RPC = 64 / (D / 8);       // rows of a copy
  static constexpr int COPIES = STEP / RPC / W;  // a wave's copies of K, and of V
  const uint16_t *k, *v;
  int row_bytes;
  uint32_t lds;
  int kvoff[COPIES], vvoff[COPIES];  // this lane's source bytes
  __device__ TileCopies(const BlockAttnParams &p, const AttnTile &t, char *smem, int wave) {
    const int64_t off = t.tk.begin * p.kv_tok + (p.per_head ? 0 : t.h * p.kv_head);
    k = p.k + off;
    v = p.v + off;
    row_bytes = static_cast<int>(p.kv_tok) * 2;
    lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char *)smem)) + wave * COPIES * RPC * ROW;
    const int lane = threadIdx.x & 63, pos = lane % (D / 8);
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int row = (wave * COPIES + i) * RPC + lane / (D / 8);
      kvoff[i] = row * row_bytes + 16 * k_chunk<D>(row, pos);
      vvoff[i] = row * row_bytes + 16 * v_chunk<D>(row, pos);
    }
  }
  // keys [key, key + STEP) below `limit`
  __device__ void issue(const BlockAttnParams &p, int key, int buf, int limit) const {
    const int left = max(0, min(STEP, limit - key));
    const int64_t off = left > 0 ? key * p.kv_tok : 0;
    const uint32_t dst = lds + buf * 2 * TILE;
    copy_each<COPIES>([&](int i, auto first) {
      copy_rows<decltype(first)::value>(k + off, static_cast<int64_t>(left) * row_bytes, dst + i * RPC * ROW, kvoff[i]);
      copy_rows<decltype(first)::value>(v + off, static_cast<int64_t>(left) * row_bytes, dst + i * RPC * ROW + TILE, vvoff[i]);
    });
  }
};

// Tiles of up to 32 W rows: W waves of 32 rows, the keys in steps of 64 through
// two LDS buffers that all waves share; two workgroups on a compute unit, so that
// one's matrix instructions run beside the other's exponentials.  Two waves (up to
// 64 rows) leave half of the unit's room for waves empty so, and take steps of 32
// where there are workgroups for four on a unit: 1,024 tiles of 64 rows and 32
// blocks 88 us (107 in steps of 64), but 400 of 48 rows 69 (55).  splits > 1
// divides the list over as many workgroups, whose parts block_attn_join_kernel
// adds up.
//
// 468 tiles of 120 rows over 6,400 keys each (bf16, head_dim 128; 184 GFLOP) take 220
// to 237 us, 775 to 835 TFLOP/s, where a large library product of such values reaches
// 1,200 to 1,281 on the same cards.  Matrix units are busy 56% of the time of the
// units that have work; without the copies it takes 178 us, without LDS reads too 145,
// without exponentials too 121: copies, fragment reads and exponentials each take time
// that the matrix instructions of two waves a SIMD do not cover.  A copy serves one
// tile; what a head's tiles list in common (here 24 sink and recent blocks of 100) is
// copied for each of them.  Not faster: steps of 32 keys in a ring of four; the scores
// of the next step beside the exponentials of this one (219 to 240 in all orders
// tried); 64 rows a wave (260); raised wave priority; touching the next blocks ahead
// (235 to 268).
template <int D, int W, int STEP, bool F16>
__global__ void __launch_bounds__(64 * W, 2) block_attn_tile_kernel(BlockAttnParams p) {
  constexpr int ROW = 2 * D, TILE = STEP * ROW;  // bytes
  __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];  // K0 V0 K1 V1
  __shared__ int list[kMaxTopk + 2];
  __shared__ int scratch[2];
  AttnTile t;
  const int wg = xcd_order(blockIdx.x, p.items * p.splits);
  const int item = wg / p.splits, split = wg - item * p.splits;
  if (!attn_tile(p, item, t)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = __builtin_amdgcn_readfirstlane(load_list<64 * W>(tile_list(p, t), p.topk, t.tk.blocks, list, scratch));
  const int r = 32 * wave + (threadIdx.x & 31);
  uint4 qf[D / 16];
  load_query<D>(p, t, r, qf);
  wait_copies<0>();  // (no load of the compiler's own is then pending among the copies)
  RowState<D> st;
  st.reset();

  const TileCopies<D, W, STEP> copies(p, t, smem, wave);
  // this workgroup's steps of the list's, from a block and an offset in it on
  const int per = p.bk / STEP, steps = n * per;
  const int first = static_cast<int>(static_cast<int64_t>(steps) * split / p.splits);
  const int last = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits);
  int e = first / per, off = (first - e * per) * STEP, buf = 0;
  int blk = __builtin_amdgcn_readfirstlane(list[e]);
  int nxt = list[e + 1];  // (past the last block it may be anything)
  if (first < last) copies.issue(p, blk * p.bk + off, 0, t.tk.limit);
  for (int step = first; step < last;) {
    const int key = blk * p.bk + off;
    ++step;
    off += STEP;
    if (off == p.bk) {
      off = 0;
      ++e;
      blk = __builtin_amdgcn_readfirstlane(nxt);
      nxt = list[e + 1];
    }
    wait_copies<0>();
    wait_reads();
    __builtin_amdgcn_s_barrier();  // the step has arrived, and no wave reads the other buffer any more
    asm volatile("" ::: "memory");
    if (step < last) copies.issue(p, blk * p.bk + off, buf ^ 1, t.tk.limit);
    const char *kt = smem + buf * 2 * TILE;
    attend_step<D, STEP / 32, F16, false, false>(kt, kt + TILE, qf, max(0, t.tk.limit - key), p.scale_log2, st);
    buf ^= 1;
  }
  const float l = both_sum(st.l);
  if (p.splits == 1) {
    store_rows<D, F16>(p, t, r, st, l, n > 0);
    return;
  }
  if (r >= t.rows) return;
  const int hf = (threadIdx.x & 63) >> 5;
  float *part = part_row<D>(p, item, split, r);
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<float4 *>(part + 32 * db + 8 * i + 4 * hf) =
          make_float4(st.o[db][4 * i], st.o[db][4 * i + 1], st.o[db][4 * i + 2], st.o[db][4 * i + 3]);
  if (hf == 0) *reinterpret_cast<float4 *>(part + D) = make_float4(st.m, l, n > 0 ? 1.0f : 0.0f, 0.0f);
}

// Several consecutive small tiles at once (a prompt in which every token has a
// list of its own): a workgroup walks the union of their lists in steps of 64
// keys through two buffers; a step counts for the rows whose tile lists its
// block, and a wave none of whose rows do only copies.  Neighbouring tokens
// share most of their blocks, so that the keys are copied for all of them at
// once, and a wave of 32 rows, which a single small tile would not fill, does
// no more matrix work than the tiles one by one.  A row gets 0 * V from
// blocks that only its neighbours list: where that is not 0 (V holds an
// infinity or NaN) the results say so, and the workgroup takes its tiles one by
// one instead.
//
// 2,047 tokens of 2 KV heads and 16 query heads each, 16 blocks a token (fp16,
// head_dim 128) in 55 to 57 us; the small kernel, one token a workgroup, 208.
// 512 workgroups in one round of the chip, two on a unit; each walks the 16 to 32
// blocks of its tokens' lists, a step's copies, reads and exponentials one after
// the other as in the tile kernel.
constexpr int kWindow = 1024;    // blocks whose lists are joined at a time
constexpr int kMaxGroup = 32;    // tiles: a bit each
constexpr int kPlaces = 512;     // workgroups that the chip takes in one round, two a unit

template <int D, int W, bool F16>
__global__ void __launch_bounds__(64 * W, 2) block_attn_group_kernel(BlockAttnParams p) {
  constexpr int ROW = 2 * D, TILE = kSub * ROW;  // bytes
  __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];  // K0 V0 K1 V1
  __shared__ int list[kWindow + 2];      // the window's blocks that any tile lists, in order
  __shared__ uint32_t members[kWindow];  // of every block of the window, the tiles that list it
  __shared__ int scratch[W > 2 ? W : 2];
  static_assert(kWindow % (64 * W) == 0, "window");
  AttnTile t;
  if (!attn_tile(p, p.causal ? causal_order(p, blockIdx.x) : xcd_order(blockIdx.x, p.items), t)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = 32 * wave + (lane & 31);
  uint4 qf[D / 16];
  load_query<D>(p, t, r, qf);
  wait_copies<0>();  // (no load of the compiler's own is then pending among the copies)

  const TileCopies<D, W, kSub> copies(p, t, smem, wave);
  const int32_t *src = tile_list(p, t);
  const int64_t row = static_cast<int64_t>(p.Hkv) * p.topk;
  const int last = (t.rows / p.G - 1) / p.bq;  // the group's last tile, whose limit t.tk has
  // keys that a tile may see (causal tiles are one token each)
  auto limit_of = [&](int tile) { return p.causal ? max(0, t.tk.limit - (last - tile)) : t.tk.limit; };
  const int my_tile = min(r, t.rows - 1) / p.G / p.bq;
  const int my_limit = limit_of(my_tile);
  uint32_t wave_tiles = 0;  // those that this wave has rows of
  if (32 * wave < t.rows) {
    const int lo = 32 * wave / p.G / p.bq, hi = min(32 * wave + 31, t.rows - 1) / p.G / p.bq;
    wave_tiles = (0xffffffffu >> (31 - (hi - lo))) << lo;
  }
  wave_tiles = __builtin_amdgcn_readfirstlane(wave_tiles);

  // the union of the lists (only < 0), and only if that will not do each tile's
  for (int only = -1; only <= last; ++only) {
    RowState<D> st;
    st.reset();
    bool seen = false;  // whether this lane's row had a key
    const int limit = only < 0 ? t.tk.limit : limit_of(only);
    const uint32_t take = only < 0 ? 0xffffffffu : 1u << only;
    for (int w0 = 0; w0 < t.tk.blocks; w0 += kWindow) {
      __syncthreads();
      for (int e = threadIdx.x; e < kWindow; e += 64 * W) members[e] = 0;
      __syncthreads();
      for (int e = threadIdx.x; e < (last + 1) * p.topk; e += 64 * W) {
        const int tile = e / p.topk;
        const int x = src[tile * row + (e - tile * p.topk)];
        if (x >= w0 && x < w0 + kWindow && x < (limit_of(tile) + p.bk - 1) / p.bk)
          atomicOr(&members[x - w0], (1u << tile) & take);
      }
      __syncthreads();
      // each thread a run of the window
      constexpr int RUN = kWindow / (64 * W);
      int mine = 0;
#pragma unroll
      for (int i = 0; i < RUN; ++i) mine += members[threadIdx.x * RUN + i] != 0;
      const int upto = wave_incl_sum(mine);
      if (lane == 63) scratch[wave] = upto;
      __syncthreads();
      int at = upto - mine, n = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        at += w < wave ? scratch[w] : 0;
        n += scratch[w];
      }
#pragma unroll
      for (int i = 0; i < RUN; ++i)
        if (members[threadIdx.x * RUN + i] != 0) list[at++] = w0 + threadIdx.x * RUN + i;
      __syncthreads();
      n = __builtin_amdgcn_readfirstlane(n);
      if (n == 0) continue;

      int blk = __builtin_amdgcn_readfirstlane(list[0]), off = 0, buf = 0;
      int nxt = list[1];  // (past the last block it may be anything)
      copies.issue(p, blk * p.bk, 0, limit);
      for (int e = 0; e < n;) {
        const int key = blk * p.bk + off;
        const uint32_t who_v = members[blk - w0];
        off += kSub;
        if (off == p.bk) {
          off = 0;
          ++e;
          blk = __builtin_amdgcn_readfirstlane(nxt);
          nxt = list[e + 1];
        }
        wait_copies<0>();
        wait_reads();
        __builtin_amdgcn_s_barrier();  // the step has arrived, and no wave reads the other buffer any more
        asm volatile("" ::: "memory");
        if (e < n) copies.issue(p, blk * p.bk + off, buf ^ 1, limit);
        const uint32_t who = __builtin_amdgcn_readfirstlane(who_v);
        if ((who & wave_tiles) != 0) {
          const char *kt = smem + buf * 2 * TILE;
          const int keys = (who >> my_tile) & 1 ? max(0, my_limit - key) : 0;
          seen = seen || keys > 0;
          attend_step<D, 2, F16, true, false>(kt, kt + TILE, qf, keys, p.scale_log2, st);
        }
        buf ^= 1;
      }
    }
    if (only >= 0) {
      store_rows<D, F16>(p, t, my_tile == only ? r : t.rows, st, both_sum(st.l), seen);
      continue;
    }
    const bool odd = __builtin_amdgcn_ballot_w64(r < t.rows && !finite(st)) != 0;
    if (!__syncthreads_or(odd)) {
      store_rows<D, F16>(p, t, r, st, both_sum(st.l), seen);
      return;
    }
  }
}

// Tiles of up to 32 rows (single tokens of grouped heads): 4 waves that each
// take every fourth 32-key step of the list through a ring of their own, with
// no barrier in the loop, joined at the end.  splits > 1 divides the list over
// as many workgroups, whose parts block_attn_join_kernel adds up.
//
// Bound by memory: 16 tokens of 8 KV heads over 32 blocks each (134 MB of K and V)
// take 25 us here, 5.3 TB/s, and 4 in the join; one token of 2 KV heads over 8 blocks
// 7.2, a chain of dependent reads (lengths, list, keys) and the launch.
constexpr int kSmallWaves = 4;
constexpr int kRing = 2;

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
  const int32_t *src = tile_list(p, t);
  uint4 qf[D / 16];
  load_query<D>(p, t, lq, qf);
  // a list that fits the lanes, ascending and then none, stays in them
  const int x = lane < p.topk ? src[lane] : -1;
  const bool valid = x >= 0 && x < t.tk.blocks;
  const uint64_t valids = __builtin_amdgcn_ballot_w64(valid);
  const int before = __shfl_up(x, 1);  // (by every lane: one that did not take part has nothing to read from)
  const bool odd = valid && lane > 0 && !((valids >> (lane - 1) & 1) && before < x);
  const bool in_lanes = p.topk <= 64 && __builtin_amdgcn_ballot_w64(odd) == 0;
  const int n = in_lanes ? __popcll(valids)
                         : __builtin_amdgcn_readfirstlane(
                               load_list<64 * kSmallWaves>(src, p.topk, t.tk.blocks, list, scratch));
  auto block = [&](int e) {
    return in_lanes ? __builtin_amdgcn_readlane(x, e) : __builtin_amdgcn_readfirstlane(list[e]);
  };
  wait_copies<0>();  // (no load of the compiler's own is then pending among the copies)
  RowState<D> st;
  st.reset();

  const int64_t head_off = t.tk.begin * p.kv_tok + (p.per_head ? 0 : t.h * p.kv_head);
  const uint16_t *kp = p.k + head_off, *vp = p.v + head_off;
  constexpr int RPC = 64 / (D / 8), COPIES = 32 / RPC;  // copies of K, and of V, per step
  const int row_bytes = static_cast<int>(p.kv_tok) * 2;
  char *ring = smem + wave * kRing * 2 * TILE;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char *)ring));
  int kvoff[COPIES], vvoff[COPIES];
#pragma unroll
  for (int i = 0; i < COPIES; ++i) {
    const int row = i * RPC + lane / (D / 8), pos = lane % (D / 8);
    kvoff[i] = row * row_bytes + 16 * k_chunk<D>(row, pos);
    vvoff[i] = row * row_bytes + 16 * v_chunk<D>(row, pos);
  }
  auto issue = [&](int key, int buf) {
    const int left = max(0, min(32, t.tk.limit - key));
    const int64_t off = left > 0 ? key * p.kv_tok : 0;
    copy_each<COPIES>([&](int i, auto first) {
      const uint32_t at = lds0 + buf * 2 * TILE + i * RPC * ROW;
      copy_rows<decltype(first)::value>(kp + off, static_cast<int64_t>(left) * row_bytes, at, kvoff[i]);
      copy_rows<decltype(first)::value>(vp + off, static_cast<int64_t>(left) * row_bytes, at + TILE, vvoff[i]);
    });
  };
  // this wave's steps: every (4 * splits)-th 32 keys of the list, as an entry and an
  // offset in its block
  const int stride = 32 * kSmallWaves * p.splits, blocks_on = stride / p.bk, keys_on = stride - blocks_on * p.bk;
  const int start = 32 * (wave * p.splits + split);
  auto walk = [&](auto fine) {
    int e = start / p.bk, off = start - e * p.bk;
    int key = e < n ? block(e) * p.bk + off : 0;
    wait_reads();  // (of the walk before)
    if (e < n) issue(key, 0);
    for (int buf = 0; e < n; buf ^= 1) {
      const int now = key;
      e += blocks_on;
      off += keys_on;
      if (off >= p.bk) {
        off -= p.bk;
        ++e;
      }
      wait_reads();  // the other buffer has been read
      if (e < n) {
        key = block(e) * p.bk + off;
        issue(key, buf ^ 1);
        wait_copies<2 * COPIES>();
      } else {
        wait_copies<0>();
      }
      asm volatile("" ::: "memory");
      const char *kt = ring + buf * 2 * TILE;
      attend_step<D, 1, F16, false, decltype(fine)::value>(kt, kt + TILE, qf, max(0, t.tk.limit - now), p.scale_log2, st);
    }
  };
  walk(std::true_type());
  // an infinity in V is one of O, but the second part of P may be 0 or negative
  // there, and the two parts' products NaN: such a wave takes its keys again, P in
  // one part
  if (__builtin_amdgcn_ballot_w64(!finite(st)) != 0) {
    st.reset();
    walk(std::false_type());
  }
  const float l = both_sum(st.l);

  // joined: the waves' O^T in LDS, scaled to the largest reference
  const bool here = lq < t.rows;
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
    const float2 y = ml[w][lq];
    sum += y.y == 0.0f ? 0.0f : y.y * __builtin_amdgcn_exp2f(y.x - ref);
  }
  const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(st.m - ref);
  float4 *buf = reinterpret_cast<float4 *>(smem);  // [wave][register quad][lane]
  constexpr int QUADS = D / 8;
  if (here)
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      const f32x16 &o = st.o[i / 4];
      const int q = 4 * (i % 4);
      buf[(wave * QUADS + i) * 64 + lane] = make_float4(o[q] * f, o[q + 1] * f, o[q + 2] * f, o[q + 3] * f);
    }
  __syncthreads();
  if (!here) return;
  const int tok = lq / p.G, g = lq - tok * p.G, head = t.h * p.G + g;
  const int64_t row = t.q_begin + static_cast<int64_t>(t.tok0) + tok;
  const float inv = inv_sum(sum, n > 0);
  float *part = part_row<D>(p, item, split, lq);
#pragma unroll
  for (int i = wave; i < QUADS; i += kSmallWaves) {
    float4 a = buf[i * 64 + lane];
#pragma unroll
    for (int w = 1; w < kSmallWaves; ++w) {
      const float4 y = buf[(w * QUADS + i) * 64 + lane];
      a = make_float4(a.x + y.x, a.y + y.y, a.z + y.z, a.w + y.w);
    }
    const int d = 8 * i + 4 * hf;
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
  if (wave != 0 || hf != 0) return;
  if (p.splits > 1) {
    *reinterpret_cast<float4 *>(part + D) = make_float4(m, sum, n > 0 ? 1.0f : 0.0f, 0.0f);
  } else if (p.lse) {
    p.lse[static_cast<int64_t>(head) * p.total_q + row] = log_sum(m, sum);
  }
}

// The parts of a tile's workgroups, added up in their order: one wave per query
// row.  Lane i first holds part i's reference and sum (64 parts at a time), then
// columns i and i + 64; parts are read eight together.
template <int D, bool F16>
__global__ void __launch_bounds__(256) block_attn_join_kernel(BlockAttnParams p) {
  constexpr int C = D / 64, kAhead = 8;
  const int64_t part_floats = static_cast<int64_t>(p.part_rows) * (D + 4);  // from part to part
  const int rows = p.bq * p.G;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int item = static_cast<int>(w / rows), r = static_cast<int>(w - static_cast<int64_t>(item) * rows);
  if (item >= p.items) return;
  AttnTile t;
  if (!attn_tile(p, item, t) || r >= t.rows) return;
  const int lane = threadIdx.x & 63;
  const float *part = part_row<D>(p, item, 0, r);
  float m = -INFINITY, sum = 0.0f, o[C];
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = 0.0f;
  bool keys = false;
  for (int s0 = 0; s0 < p.splits; s0 += 64) {
    const int cnt = min(64, p.splits - s0);
    const float *x = part + s0 * part_floats;
    const float4 mine = lane < cnt ? *reinterpret_cast<const float4 *>(x + lane * part_floats + D)
                                   : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    float top = mine.x, add;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    top = fmaxf(top, m);
    const float ref = top == -INFINITY ? 0.0f : top;
    const float f = mine.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mine.x - ref);
    const float old = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - ref);
    add = mine.y * f;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) add += __shfl_xor(add, off);
    sum = sum * old + add;
    keys = keys || __builtin_amdgcn_ballot_w64(mine.z != 0.0f) != 0;
    m = top;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] *= old;
    for (int s = 0; s < cnt; s += kAhead) {
      float v[kAhead][C];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) v[i][c] = x[min(s + i, cnt - 1) * part_floats + 64 * c + lane];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float fi = __shfl(f, s + i);
        if (s + i < cnt)
#pragma unroll
          for (int c = 0; c < C; ++c) o[c] = fmaf(v[i][c], fi, o[c]);
      }
    }
  }
  const int tok = r / p.G, g = r - tok * p.G, head = t.h * p.G + g;
  const int64_t row = t.q_begin + static_cast<int64_t>(t.tok0) + tok;
  const float inv = inv_sum(sum, keys);
#pragma unroll
  for (int c = 0; c < C; ++c)
    p.o[row * p.o_tok + head * p.o_head + 64 * c + lane] =
        __builtin_bit_cast(uint16_t, static_cast<typename Elem8<F16>::type>(o[c] * inv));
  if (p.lse && lane == 0) p.lse[static_cast<int64_t>(head) * p.total_q + row] = log_sum(m, sum);
}

// ---- host ------------------------------------------------------------------------
// threads that a launch has at most in a dimension: the dispatch counts them in
// 32 bits
constexpr int64_t kMaxThreads = 0xffffffffll;

// rows of q or k at most: cu_seqlens are 32-bit, and lengths are rounded up to
// whole tiles and blocks (32 * 128 rows, 1,024 keys) in 32 bits
constexpr int64_t kMaxTokens = 0x7fffffff - 4096;

// what the kernels read and write in pieces of `bytes`
static bool aligned(const void *p, uintptr_t bytes = 16) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

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
  if (a->total_k > kMaxTokens) return fail(PKV_ERR_UNSUPPORTED, "block_means: too many rows");
  if (const int rc = check_block(a->head_dim, a->block_k, a->dtype, "block_means")) return rc;
  if (a->num_seqs == 0) return PKV_OK;
  if (!a->means || !a->cu_seqlens_k || (!a->k && a->total_k > 0))
    return fail(PKV_ERR_INVALID, "block_means: NULL argument");
  if ((a->kv_tok_stride | a->kv_head_stride) & 7)
    return fail(PKV_ERR_INVALID, "block_means: strides must keep 16-byte rows aligned");
  if (!aligned(a->k) || !aligned(a->means)) return fail(PKV_ERR_INVALID, "block_means: k and means must begin at 16 bytes");
  if (a->num_seqs > kMaxThreads / 256) return fail(PKV_ERR_UNSUPPORTED, "block_means: too many sequences");
  MeansParams p{};
  p.k = a->k; p.means = a->means; p.cu = a->cu_seqlens_k; p.used = a->seqlens_k;
  p.total_rows = a->total_k / a->block_k + a->num_seqs;
  p.tok = a->kv_tok_stride; p.head = a->kv_head_stride;
  p.S = a->num_seqs; p.H = a->num_heads; p.bk = a->block_k; p.last = a->last;
  p.total_k = static_cast<int>(a->total_k);
  // a wave per block and head of a sequence of the bound's length, as long as
  // those make no more workgroups than fill the chip many times (the others loop)
  const int64_t longest = a->max_seqlen_k > 0 ? a->max_seqlen_k : a->total_k;
  int64_t blocks = a->last > 0 ? a->last / a->block_k + 2 : longest / a->block_k + 1;
  if (blocks > longest / a->block_k + 1) blocks = longest / a->block_k + 1;
  int64_t chunks = (blocks * a->num_heads + 3) / 4;
  const int64_t most = 65536 / a->num_seqs;
  if (chunks > most) chunks = most > 1 ? most : 1;
  p.chunks = static_cast<int>(chunks);
  const bool f16 = a->dtype == PKV_DTYPE_FP16;
  auto *k = a->head_dim == 128 ? (f16 ? block_means_kernel<128, true> : block_means_kernel<128, false>)
                               : (f16 ? block_means_kernel<64, true> : block_means_kernel<64, false>);
  hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(a->num_seqs * chunks)), dim3(256), 0, as_stream(stream), p);
  return check_launch("block_means_kernel");
}

namespace pkv {

// Tiles whose rows the score kernel adds up itself: every workgroup over the
// same tile repeats the sum, so only where it is short.  1,024 tiles of 512 blocks
// (512 tokens of 8 KV heads) with 4 rows take 13.3 us so and 20.1 with a launch for
// the sums, 4,096 with 16 rows 40.4 and 46.5; but with 32 rows 512 tiles take 16.8
// and 15.1, with 120 rows 468 tiles 46.5 and 18.6.
constexpr int kSumRowsInline = 16;
constexpr int64_t kSelectWorkspace = 64ll << 20;  // scores of more tiles go in several launches
constexpr int kMaxSelectBlocks = 32768;

struct SelectPlan {
  int64_t nb, tiles, tile_n, sums_bytes, bytes;
  bool fused;
};

// Scores and choice in one launch where that reads few means more than once,
// measured against three launches (two without the sums'), microseconds each:
// * up to 128 blocks (a wave a row) where no other tile of the sequence reads the
//   same means and the sum is short: 32 single tokens of 64 blocks and head_dim 128
//   7.2 against 10.4, 4,096 26.5 against 46.6, of 128 blocks 47.8 against 70.6;
// * up to kFusedRow columns of means a row and kFusedBytes in all (causal rows
//   counted by the blocks that they see on average): 2,048 rows of 32 blocks and
//   head_dim 128 (32 MB) 8.4 against 10.7, 4,000 causal ones of 32 to 63 and head_dim
//   64 (46 MB) 10.5 against 11.4, 2,048 of 64 and 128 (64 MB) 11.0 alike, 4,094 of
//   32 and 128 (64 MB) 14.6 against 12.1, 4,094 of 64 (128 MB) 20.3 against 12.4,
//   16,384 71 against 29; and 156 rows of 128 blocks and head_dim 128 (10 MB) 15.6
//   against 13.1, of 64 blocks 11.2 against 13.2;
// * more, where no other tile of the sequence reads the same means (single
//   tokens) and the rows fill the chip: 128 rows of 512 blocks 14.4 against
//   18.1, 512 of 2,048 106 against 124, but 8 of 2,048 37 against 19, and
//   468 rows of 13 tiles a sequence and 320 blocks 21.7 against 16.8.
constexpr int64_t kFusedBytes = 48ll << 20, kFusedRow = 64 * 128;
constexpr int64_t kFusedMost = 4096, kFusedRows = 64;

static int check_select(const pkv_block_select_args *a) {
  if (!a) return fail(PKV_ERR_INVALID, "block_select: NULL argument");
  if (a->num_batches < 0 || a->total_q < 0 || a->total_k < 0 || a->max_seqlen_q < 0 || a->max_seqlen_k < 0)
    return fail(PKV_ERR_INVALID, "block_select: bad sizes");
  if (const int rc = check_block(a->head_dim, a->block_k, a->dtype, "block_select")) return rc;
  if (const int rc = check_tiles(a->num_heads_q, a->num_heads_kv, a->block_q, a->topk, a->causal, "block_select"))
    return rc;
  if (a->causal < PKV_NOT_CAUSAL || a->causal > PKV_CAUSAL_RANKED)
    return fail(PKV_ERR_INVALID, "block_select: causal %d", a->causal);
  if (a->sink_blocks < 0 || a->recent_blocks < 0 || static_cast<int64_t>(a->sink_blocks) + a->recent_blocks > a->topk)
    return fail(PKV_ERR_INVALID, "block_select: %d sink and %d recent blocks of %d", a->sink_blocks, a->recent_blocks,
                a->topk);
  if ((static_cast<int64_t>(a->max_seqlen_k) + a->block_k - 1) / a->block_k > kMaxSelectBlocks)
    return fail(PKV_ERR_UNSUPPORTED, "block_select: more than %d blocks", kMaxSelectBlocks);
  if (a->num_batches > 65535 || a->num_heads_kv > 65535)
    return fail(PKV_ERR_UNSUPPORTED, "block_select: more than 65535 batches or KV heads");
  if (a->total_q > kMaxTokens || a->max_seqlen_q > kMaxTokens || a->total_k > kMaxTokens)
    return fail(PKV_ERR_UNSUPPORTED, "block_select: too many rows");
  return PKV_OK;
}

static SelectPlan select_plan(const pkv_block_select_args *a) {
  SelectPlan s{};
  s.tiles = (static_cast<int64_t>(a->max_seqlen_q) + a->block_q - 1) / a->block_q;
  s.nb = ((static_cast<int64_t>(a->max_seqlen_k) + a->block_k - 1) / a->block_k + 63) / 64 * 64;
  if (s.nb == 0) s.nb = 64;
  if (s.tiles == 0) s.tiles = 1;  // (the lists' rows are written all the same)
  const int64_t heads = static_cast<int64_t>(a->num_batches) * a->num_heads_kv;
  const int64_t rows = heads * s.tiles;
  const bool sums = a->block_q * (a->num_heads_q / a->num_heads_kv) > kSumRowsInline;
  int64_t keys = a->max_seqlen_k;  // that a row sees on average
  if (a->causal) keys -= (a->max_seqlen_q < keys ? a->max_seqlen_q : keys) / 2;
  const int64_t means = rows * (keys / a->block_k + 1) * a->head_dim * 4;
  if (s.nb <= 128)
    s.fused = (s.tiles == 1 && !sums) || (s.nb * a->head_dim <= kFusedRow && means <= kFusedBytes);
  else
    s.fused = s.tiles == 1 && rows >= kFusedRows && s.nb <= kFusedMost;
  if (s.fused) return s;
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
  if (s.fused) {
    SelectParams p = p0;
    p.tile0 = 0;
    p.tile_n = static_cast<int>(s.tiles);
    if (s.nb <= 128) {
      auto *k = s.nb <= 64 ? block_select_kernel<D, F16, 1, 1> : block_select_kernel<D, F16, 1, 2>;
      hipLaunchKernelGGL(k, dim3((p.tile_n + 3) / 4, p.Hkv, p.B), dim3(256), 0, st, p);
    } else {
      auto *k = s.nb <= 512 ? block_select_kernel<D, F16, 8, 1> : block_select_kernel<D, F16, 8, 8>;
      hipLaunchKernelGGL(k, dim3(p.tile_n, p.Hkv, p.B), dim3(512), 0, st, p);
    }
    return check_launch("block_select_kernel");
  }
  for (int64_t tile0 = 0; tile0 < s.tiles; tile0 += s.tile_n) {
    SelectParams p = p0;
    p.tile0 = static_cast<int>(tile0);
    p.tile_n = static_cast<int>(s.tiles - tile0 < s.tile_n ? s.tiles - tile0 : s.tile_n);
    if (p.sums) {
      hipLaunchKernelGGL((tile_sums_kernel<D, F16>), dim3(p.tile_n, p.Hkv, p.B), dim3(256), 0, st, p);
      if (const int rc = check_launch("tile_sums_kernel")) return rc;
    }
    const int64_t groups = (p.tile_n + 15) / 16;
    // enough workgroups for the chip, each with as many blocks as that leaves
    int64_t chunks = (s.nb + 63) / 64;
    const int64_t most = (2048 + groups * heads - 1) / (groups * heads);
    if (chunks > most) chunks = most;
    p.chunks = static_cast<int>(chunks);
    hipLaunchKernelGGL((block_scores_kernel<D, F16>), dim3(static_cast<unsigned>(groups * chunks), p.Hkv, p.B), dim3(256),
                       0, st, p);
    if (const int rc = check_launch("block_scores_kernel")) return rc;
    // one wave up to 8 keys a lane (no barriers in the search: 1,024 rows of 512 keys
    // in 13.3 us with the scores, 18.4 by four waves a row), then the fewest that
    // hold them
    if (s.nb <= 64 * 8) {
      auto *k = s.nb <= 64 * 2 ? block_choose_kernel<1, 2> : block_choose_kernel<1, 8>;
      hipLaunchKernelGGL(k, dim3((p.tile_n + 3) / 4, p.Hkv, p.B), dim3(256), 0, st, p);
    } else if (s.nb <= 256 * 8) {
      hipLaunchKernelGGL((block_choose_kernel<4, 8>), dim3(p.tile_n, p.Hkv, p.B), dim3(256), 0, st, p);
    } else {
      auto *k = s.nb <= 1024 * 8 ? block_choose_kernel<16, 8> : block_choose_kernel<16, 32>;
      hipLaunchKernelGGL(k, dim3(p.tile_n, p.Hkv, p.B), dim3(1024), 0, st, p);
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
  if (!aligned(a->q) || !aligned(a->means) || !aligned(workspace))
    return fail(PKV_ERR_INVALID, "block_select: q, means and the workspace must begin at 16 bytes");
  const SelectPlan s = select_plan(a);
  if (s.bytes > 0 && (!workspace || workspace_bytes < s.bytes))
    return fail(PKV_ERR_CAPACITY, "block_select: workspace of %lld bytes, %lld needed",
                static_cast<long long>(workspace_bytes), static_cast<long long>(s.bytes));
  const int64_t heads = static_cast<int64_t>(a->num_batches) * a->num_heads_kv;
  SelectParams p{};
  p.q = a->q; p.means = a->means; p.lists = a->lists;
  p.cu_q = a->cu_seqlens_q; p.cu_k = a->cu_seqlens_k; p.used = a->seqlens_k;
  p.tile_rows = a->total_q / a->block_q + a->num_batches;
  p.mean_rows = a->total_k / a->block_k + (a->kv_per_head ? heads : a->num_batches);
  p.total_q = static_cast<int>(a->total_q); p.total_k = static_cast<int>(a->total_k);
  p.q_tok = a->q_tok_stride; p.q_head = a->q_head_stride;
  p.B = a->num_batches; p.Hq = a->num_heads_q; p.Hkv = a->num_heads_kv;
  p.G = a->num_heads_q / a->num_heads_kv;
  p.per_head = a->kv_per_head ? 1 : 0;
  p.tiles = static_cast<int>((static_cast<int64_t>(a->max_seqlen_q) + a->block_q - 1) / a->block_q);
  p.most = static_cast<int>((static_cast<int64_t>(a->max_seqlen_k) + a->block_k - 1) / a->block_k);
  p.nb = static_cast<int>(s.nb);
  p.bq = a->block_q; p.bk = a->block_k; p.topk = a->topk; p.sink = a->sink_blocks; p.recent = a->recent_blocks;
  p.causal = a->causal ? 1 : 0;
  // a token's own block, the last that it chooses from, is taken, not scored: its
  // mean covers later keys
  if (a->causal == PKV_CAUSAL && p.recent < 1) p.recent = 1;
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
  if (a->total_q > kMaxTokens || a->max_seqlen_q > kMaxTokens || a->total_k > kMaxTokens)
    return fail(PKV_ERR_UNSUPPORTED, "block_attn: too many rows");
  if (items > kMaxThreads / 512) return fail(PKV_ERR_UNSUPPORTED, "block_attn: grid too large");
  return PKV_OK;
}

// How a launch is cut: tiles that a workgroup takes together, workgroups that
// share a tile.
struct AttnPlan {
  int64_t tiles, items;  // groups of a sequence, of all
  int group, splits, part_rows;
};

static AttnPlan attn_plan(const pkv_block_attn_args *a) {
  AttnPlan s{};
  const int rows = a->block_q * (a->num_heads_q / a->num_heads_kv);
  const int64_t heads = static_cast<int64_t>(a->num_batches) * a->num_heads_kv;
  const int64_t tiles = (static_cast<int64_t>(a->max_seqlen_q) + a->block_q - 1) / a->block_q;
  s.group = s.splits = 1;
  if (rows <= 32) {
    // as few tiles a workgroup as the chip takes in one round, up to 128 rows.  Tokens of
    // 2 KV heads of 16 query heads, 16 blocks each of the same 512 / of lists of their
    // own: 256 tokens one by one 33 / 36 us, by fours 47 / 98; 512 by twos 42 / 58, one
    // by one 59 / 67, by eights 41 / 134; 1,500 by eights 60 / 152, by fours (two
    // rounds) 95 / 190, one by one 163 / 181
    const int64_t most = 128 / rows < kMaxGroup ? 128 / rows : kMaxGroup;
    int64_t g = 1;
    while (g < most && heads * ((tiles + g - 1) / g) > kPlaces) g = 2 * g < most ? 2 * g : most;
    s.group = static_cast<int>(g);
  }
  s.tiles = (tiles + s.group - 1) / s.group;
  s.items = heads * s.tiles;
  if (rows <= 32 && s.group == 1 && s.items > 0) {
    // as many workgroups as give the chip one each, at least one 32-key step a
    // wave, where a workgroup alone would take eight: joining the parts costs
    // what four steps do (8 tiles of 32 blocks 13.0 us in 16 parts, 15.0 in 4; 2
    // tiles of 8 blocks 10.1 alone, 12.6 in 4)
    int64_t n = 256 / s.items;
    const int64_t steps = static_cast<int64_t>(a->topk) * (a->block_k / 32) / kSmallWaves;
    if (n > steps) n = steps;
    if (steps >= 8 && n > 1) s.splits = static_cast<int>(n);
  }
  s.part_rows = rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
  if (rows > 32 && s.items > 0) {
    // one round of the chip (two workgroups on a unit, one of 8 waves) where it takes
    // three a tile, each at least four steps of 64 keys: 12 tiles of 120 rows and 64
    // blocks 24.5 us (83.7 alone; 25.3 in pieces of 8 steps, 32.8 of 16), a token of 2
    // KV heads of 48 query heads and 15 blocks 16.3 (25.8; 26.5 in pieces of 8), 156
    // tiles of 128 rows and 64 blocks 72 in threes (91), but 200 of 32 blocks 61 in
    // twos (51)
    int64_t places = (rows <= 128 ? kPlaces : kPlaces / 2) / s.items;
    const int64_t pieces = static_cast<int64_t>(a->topk) * (a->block_k / kSub) / 4;
    // (four a unit in steps of 32 keys: 300 tiles of 64 rows and 64 blocks 87 us in
    // threes, 104 alone, but 256 of 8 blocks 31 in twos, 18 alone)
    if (rows <= 64 && places < 3 && pieces >= 3) places = 2 * kPlaces / s.items;
    const int64_t n = places < pieces ? places : pieces;
    if (places >= 3 && n > 1) s.splits = static_cast<int>(n);
  }
  return s;
}

template <int D, bool F16>
static int launch_block_attn(const BlockAttnParams &p, hipStream_t st) {
  const int rows = p.bq * p.G;
  if (p.group > 1) {
    const bool two = p.group * rows <= 64;
    hipLaunchKernelGGL((two ? block_attn_group_kernel<D, 2, F16> : block_attn_group_kernel<D, 4, F16>), dim3(p.items),
                       dim3(two ? 128 : 256), 0, st, p);
    return check_launch("block_attn_group_kernel");
  }
  if (rows > 32) {
    const int w = rows <= 64 ? 2 : rows <= 128 ? 4 : 8;
    auto *k = w == 4 ? block_attn_tile_kernel<D, 4, 64, F16> : block_attn_tile_kernel<D, 8, 64, F16>;
    if (w == 2)
      k = p.items * p.splits > kPlaces ? block_attn_tile_kernel<D, 2, 32, F16> : block_attn_tile_kernel<D, 2, 64, F16>;
    hipLaunchKernelGGL(k, dim3(p.items * p.splits), dim3(64 * w), 0, st, p);
    if (const int rc = check_launch("block_attn_tile_kernel")) return rc;
  } else {
    hipLaunchKernelGGL((block_attn_small_kernel<D, F16>), dim3(p.items * p.splits), dim3(64 * kSmallWaves), 0, st, p);
    if (const int rc = check_launch("block_attn_small_kernel")) return rc;
  }
  if (p.splits == 1) return PKV_OK;
  const int64_t waves = static_cast<int64_t>(p.items) * rows;
  hipLaunchKernelGGL((block_attn_join_kernel<D, F16>), dim3(static_cast<unsigned>((waves + 3) / 4)), dim3(256), 0, st, p);
  return check_launch("block_attn_join_kernel");
}

}  // namespace pkv

extern "C" int64_t pkv_block_attn_workspace_size(const pkv_block_attn_args *a) {
  if (!a || check_attn(a)) return 0;
  const AttnPlan s = attn_plan(a);
  return s.splits > 1 ? s.items * s.splits * s.part_rows * (a->head_dim + 4) * 4 : 0;
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
  if (!aligned(a->q) || !aligned(a->k) || !aligned(a->v) || !aligned(a->o, 8) || !aligned(workspace))
    return fail(PKV_ERR_INVALID, "block_attn: q, k, v and the workspace must begin at 16 bytes, o at 8");
  // buffer offsets within one step of keys are 32-bit; a step's bound is its keys
  // times the stride, which must hold a whole row
  if (a->kv_tok_stride < a->head_dim || a->kv_tok_stride * 2 * kSub > 0x7fffffff)
    return fail(PKV_ERR_UNSUPPORTED, "block_attn: kv token stride %lld (%d to %d)",
                static_cast<long long>(a->kv_tok_stride), a->head_dim, 0x7fffffff / 2 / kSub);
  const int64_t need = pkv_block_attn_workspace_size(a);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(PKV_ERR_CAPACITY, "block_attn: workspace of %lld bytes, %lld needed",
                static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  BlockAttnParams p{};
  p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o; p.lse = a->lse; p.lists = a->lists;
  p.cu_q = a->cu_seqlens_q; p.cu_k = a->cu_seqlens_k; p.used = a->seqlens_k;
  p.total_q = static_cast<int>(a->total_q);
  p.total_k = static_cast<int>(a->total_k);
  p.q_tok = a->q_tok_stride; p.q_head = a->q_head_stride;
  p.kv_tok = a->kv_tok_stride; p.kv_head = a->kv_head_stride;
  p.o_tok = a->o_tok_stride; p.o_head = a->o_head_stride;
  p.B = a->num_batches; p.Hq = a->num_heads_q; p.Hkv = a->num_heads_kv;
  p.G = a->num_heads_q / a->num_heads_kv;
  p.per_head = a->kv_per_head ? 1 : 0;
  const AttnPlan s = attn_plan(a);
  p.tiles = static_cast<int>(s.tiles);
  p.items = static_cast<int>(s.items);
  p.group = s.group;
  p.max_q = a->max_seqlen_q;
  p.bq = a->block_q; p.bk = a->block_k; p.topk = a->topk;
  p.causal = a->causal ? 1 : 0;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.splits = s.splits;
  p.part_rows = s.part_rows;
  p.part = static_cast<float *>(workspace);
  hipStream_t st = as_stream(stream);
  const bool f16 = a->dtype == PKV_DTYPE_FP16;
  if (a->head_dim == 128) return f16 ? launch_block_attn<128, true>(p, st) : launch_block_attn<128, false>(p, st);
  return f16 ? launch_block_attn<64, true>(p, st) : launch_block_attn<64, false>(p, st);
}
