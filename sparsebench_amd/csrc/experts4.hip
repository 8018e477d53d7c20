// The gated layer with 4-bit weights, for the few tokens of a decode step.
//
// A weight is a code of one sign, two exponent and one mantissa bits (0, 0.5, 1,
// 1.5, 2, 3, 4, 6) times 2^(s - 127), a byte s for each 32 along the reduction.
// Of w [E, K, N] the codes are [E, N/32, K/32, 32, 16] bytes, 32 consecutive k of
// a column in 16 (the even ones in the low halves), the scales [E, N/32, K/32, 32].
// gfx950 turns two codes and a scale into two bf16 values in one instruction
// (the product is exact in bf16), which then feed the matrix units as they are.
//
//   up4    h[c] = a(x W1g) (x W1u), a row per copy, bf16
//   down4  part[s][c] = h W2 over the s-th part of F, fp32
//   out4   out[t] = sum_j gates[t, j] sum_s part[s][t k + j]
//
// A workgroup of up4 / down4 has 4 waves for one expert and the rows of its
// copies, 32 at a time. A wave owns 32 columns (in up4, of both halves) and 1 / WK
// of the reduction, in steps of 128 k; with few columns in all, WK waves share
// them and add up through LDS in a fixed order. A lane's 16 bytes of codes are 32 k
// of a column: one load and one scale feed four 16 x 16 x 32 products whose k are
// taken in that order on both sides. Codes are loaded two (up4) or four steps ahead.
//
// Bound by the weights' bytes, 17 / 32 of one each: one token, D = 4096, F = 14336, top 2
// 22.6 us (5.5 TB/s), 14.1 (4.4) and 4.0; 24 tokens, D = 1024, F = 4096, 64 experts 31.9
// (4.7), 20.9 (3.6) and 4.5. Where experts have many rows the rates are lower: 250 tokens,
// D = 2048, F = 768, 128 experts, top 4 49 (3.6), 27 (3.3), 4.8, and 5.8 for the sort. There
// waves wait for loads 44% of their cycles and to issue 45%, as with few rows; vector
// instructions, the conversions among them, take 6% (counters). One token of a small layer is two launches, 9.6.

#include "gated_act.hpp"
#include "gated.hpp"
#include "workspace.hpp"

namespace sb {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kCols = 32, kRows = 32, kStepK = 128;
constexpr int kMaxCopies = 2048, kMaxSplits = 8, kMaxExperts = 1024;
constexpr int kFew = 64;  // copies that a wave looks through by itself
constexpr int kTileBytes = kCols * kStepK / 2, kScaleBytes = kCols * kStepK / 32;  // of a step
constexpr int kBlockBytes = 16 * kStepK * 2;  // of a step of 16 packed rows

struct Few4Args {
  const uint16_t* x;
  const void *expert_idx, *gates;
  const uint8_t *w1, *s1, *w2, *s2;
  const int32_t* valid_tokens;
  uint16_t *h, *out;
  float* part;
  const int32_t* rows;  // rows4_kernel's; null for few copies
  int32_t idx_is_i64, num_tokens, k, num_experts, d_model, ffn_dim, splits, gate_dtype, units, blocks;
};

__device__ __forceinline__ int32_t copy_limit(const Few4Args& a) {
  const int32_t tokens = a.valid_tokens ? min(a.num_tokens, max(0, *a.valid_tokens)) : a.num_tokens;
  return tokens * a.k;
}

__device__ __forceinline__ int32_t expert_of(const Few4Args& a, int32_t c) {
  const int64_t e = a.idx_is_i64 ? static_cast<const int64_t*>(a.expert_idx)[c]
                                 : static_cast<const int32_t*>(a.expert_idx)[c];
  return e >= 0 && e < a.num_experts ? static_cast<int32_t>(e) : -1;
}

// ---- the copies by expert ----
//
// Up to kFew copies: a unit is a copy; the one that is the first of its expert
// does the rows of all of them, which each wave finds with a ballot. More: one
// workgroup sorts the copies by expert (stable, so in order) and cuts each
// expert's into tiles of 32 rows; a unit is a tile. In int32:
//   rows[0] tiles; rows[4 + 4 i ..] expert, first, count of tile i, and its first
//   block of 16 rows; then the copies.
// up4 then writes h as down4's products take it, in blocks of 16 rows: a step's
// 128 k of a block are 4 KB, 1 KB for each of its four products, 16 bytes a lane.
// Read row by row, 16 bytes from each of 16 rows, they cost the CU's address unit
// more than the weights (down4, 250 tokens, D = 2048, F = 768, E = 128, top 4: 40 us
// against 28). Packing x as well takes its own kernel as long as it saves.

int64_t max_row_tiles(int64_t copies, int64_t num_experts) { return copies / kRows + std::min(copies, num_experts); }
int64_t max_row_blocks(int64_t copies, int64_t num_experts) { return copies / 16 + std::min(copies, num_experts); }
__host__ __device__ inline int64_t row_words(int64_t tiles, int64_t copies) { return 4 + 4 * tiles + copies; }

constexpr int kSortThreads = 1024, kSortChunks = kMaxCopies / 64;

__global__ void __launch_bounds__(kSortThreads) rows4_kernel(Few4Args a, int32_t* __restrict__ rows, int32_t max_tiles) {
  __shared__ uint16_t counts[kSortChunks][kMaxExperts];  // of a chunk of 64 copies; then of those before it
  __shared__ int32_t starts[kMaxExperts], waves[3][kSortThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int32_t limit = copy_limit(a);
  const int chunks = (limit + 63) / 64;
  for (int i = threadIdx.x; i < chunks * (kMaxExperts / 2); i += kSortThreads) reinterpret_cast<uint32_t*>(counts)[i] = 0;
  __syncthreads();
  int expert[kSortChunks / 16], rank[kSortChunks / 16];
#pragma unroll
  for (int i = 0; i < kSortChunks / 16; ++i) {
    const int chunk = wave + 16 * i, c = chunk * 64 + lane;
    const int e = c < limit ? expert_of(a, c) : -1;
    uint64_t peers = __ballot(e >= 0);
#pragma unroll
    for (int bit = 0; bit < 10; ++bit) {
      const uint64_t set = __ballot(e >> bit & 1);
      peers &= e >> bit & 1 ? set : ~set;
    }
    expert[i] = e;
    rank[i] = __builtin_popcountll(peers & ((uint64_t{1} << lane) - 1));
    if (e >= 0 && rank[i] == 0) counts[chunk][e] = static_cast<uint16_t>(__builtin_popcountll(peers));
  }
  __syncthreads();
  // A lane per expert: its copies, and where they and their tiles start.
  const int e = threadIdx.x;
  int total = 0;
  for (int c = 0; c < chunks; ++c) {
    const int n = counts[c][e];
    counts[c][e] = static_cast<uint16_t>(total);
    total += n;
  }
  const int tiles = (total + kRows - 1) / kRows, blocks = (total + 15) / 16;
  int to[3] = {total, tiles, blocks};  // inclusive sums over the lanes up to this one
  for (int s = 1; s < 64; s <<= 1)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int x = __shfl_up(to[i], s);
      if (lane >= s) to[i] += x;
    }
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < 3; ++i) waves[i][wave] = to[i];
  __syncthreads();
  for (int w = 0; w < wave; ++w)
#pragma unroll
    for (int i = 0; i < 3; ++i) to[i] += waves[i][w];
  starts[e] = to[0] - total;
  if (e == kSortThreads - 1) rows[0] = to[1];
  for (int i = 0; i < tiles; ++i) {
    int32_t* t = rows + 4 + 4 * (to[1] - tiles + i);
    t[0] = e;
    t[1] = to[0] - total + i * kRows;
    t[2] = min(kRows, total - i * kRows);
    t[3] = to[2] - blocks + i * (kRows / 16);
  }
  __syncthreads();
  int32_t* sorted = rows + 4 + 4 * max_tiles;
#pragma unroll
  for (int i = 0; i < kSortChunks / 16; ++i) {
    const int chunk = wave + 16 * i;
    if (expert[i] >= 0) sorted[starts[expert[i]] + counts[chunk][expert[i]] + rank[i]] = chunk * 64 + lane;
  }
}

// A workgroup's rows: those of `expert`'s copies at list[0 .. count).
struct Few4Rows {
  int expert, count, block;  // block: its first of 16 packed rows
};

// Of a unit; list: LDS of kFew copies, written by each wave alike.
template <bool FEW>
__device__ __forceinline__ Few4Rows unit_rows(const Few4Args& a, int unit, int32_t* list) {
  const int lane = threadIdx.x & 63;
  if constexpr (FEW) {
    const int32_t limit = copy_limit(a);
    const int mine = lane < limit ? expert_of(a, lane) : -1;
    const int e = uniform(__builtin_amdgcn_readlane(mine, unit));
    const uint64_t all = __ballot(mine == e);
    if (e < 0 || __builtin_ctzll(all) != unit) return {-1, 0, 0};
    if (mine == e) list[__builtin_popcountll(all & ((uint64_t{1} << lane) - 1))] = lane;
    return {e, uniform(__builtin_popcountll(all)), 0};
  } else {
    if (unit >= scalar_load(a.rows)) return {-1, 0, 0};
    const int32_t* t = a.rows + 4 + 4 * unit;
    const int count = scalar_load(t + 2);
    const int32_t* sorted = a.rows + 4 + 4 * static_cast<int64_t>(a.units) + scalar_load(t + 1);
    if (lane < count) list[lane] = sorted[lane];
    return {scalar_load(t), count, scalar_load(t + 3)};
  }
}

// Eight codes of a dword as bf16 values.
__device__ __forceinline__ bf16x8_t dequantize(uint32_t codes, float scale) {
  const bf16x2_pack_t v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2_pack_t v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2_pack_t v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2_pack_t v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8_t{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

__device__ __forceinline__ float scale_of(uint8_t s) { return __uint_as_float(static_cast<uint32_t>(s) << 23); }

// P column tiles' codes and scales of one expert (uniform addresses); steps
// first, first + WK, ... < last of them are this wave's. A ring of kAhead steps in
// registers: a slot is loaded again as soon as it has been used, past the end with
// the last step, so that every wait is for a fixed number of loads. A lane has
// columns lane % 16 and 16 + lane % 16, and k = 32 (lane / 16) .. + 31 of a step.
// NT: past the caches, where each weight is read once (41.8 us a call against 46 for
// one token, D = 4096, F = 14336); an expert of several row tiles meets them there.
template <int P, int WK, bool NT>
struct Weights {
  static constexpr int kAhead = P == 1 ? 4 : 2;
  __amdgpu_buffer_rsrc_t codes[P], scales[P];
  int first, last;
  struct Ring {
    u32x4_t w[kAhead][P][2];
    uint8_t s[kAhead][P][2];
  };
  __device__ __forceinline__ void set(int p, const uint8_t* c, const uint8_t* s, int steps) {
    codes[p] = make_rsrc(c, static_cast<uint32_t>(steps) * kTileBytes);
    scales[p] = make_rsrc(s, static_cast<uint32_t>(steps) * kScaleBytes);
  }
  template <int I>
  __device__ __forceinline__ void load(int t, Ring& r) const {
    const uint32_t at = (threadIdx.x & 63) / 16 * kCols + threadIdx.x % 16;  // of [4][32]
    const int step = min(t, last - 1);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        r.w[I][p][c] = __builtin_amdgcn_raw_buffer_load_b128(codes[p], (at + 16u * c) * 16u, step * kTileBytes, NT ? 2 : 0);
        r.s[I][p][c] = __builtin_amdgcn_raw_buffer_load_b8(scales[p], at + 16u * c, step * kScaleBytes, 0);
      }
  }
  __device__ __forceinline__ void start(Ring& r) const {
    static_for<0, kAhead>([&](auto i) { load<decltype(i)::value>(first + decltype(i)::value * WK, r); });
  }
};

// acc[i][p][c] += rows 16 i .. 16 i + 15 . columns 16 c .. of column tile p. row[i]:
// where the lane's row of A (16 i + lane % 16) starts, at k = 32 (lane / 16), out of
// range for none (zeros, without a read); the ring holds the first steps (start).
template <int RT, int P>
using Sums4 = f32x4_t[RT][P][2];

// PACKED: rows in blocks of 16, as up4 writes h; row[i] is the lane's place in block i.
template <bool PACKED, int RT, int P, int WK, bool NT>
__device__ __forceinline__ void multiply(Sums4<RT, P>& acc, __amdgpu_buffer_rsrc_t rows, const uint32_t (&row)[RT],
                                         const Weights<P, WK, NT>& w, typename Weights<P, WK, NT>::Ring& ring) {
  constexpr int kAhead = Weights<P, WK, NT>::kAhead;
  u32x4_t x[RT][4];
  auto load_row = [&](int t, int q) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
      x[i][q] = __builtin_amdgcn_raw_buffer_load_b128(rows, row[i] + (PACKED ? 1024u : 16u) * q,
                                                     min(t, w.last - 1) * (PACKED ? kBlockBytes : kStepK * 2), 0);
  };
#pragma unroll
  for (int q = 0; q < 4; ++q) load_row(w.first, q);
  for (int t = w.first; t < w.last; t += kAhead * WK) {
    static_for<0, kAhead>([&](auto ic) {
      constexpr int I = decltype(ic)::value;
      const int at = t + I * WK;
      if (at >= w.last) return;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const bf16x8_t b = dequantize(ring.w[I][p][c][q], scale_of(ring.s[I][p][c]));
#pragma unroll
            for (int i = 0; i < RT; ++i)
              acc[i][p][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x[i][q]), b,
                                                                     acc[i][p][c], 0, 0, 0);
          }
        load_row(at + WK, q);
      }
      w.template load<I>(at + kAhead * WK, ring);
    });
  }
}

// The row of acc[i][.][.][v], and the column of acc[.][.][c][.], in a tile.
__device__ __forceinline__ int acc_row(int i, int v, int lane) { return 16 * i + 4 * (lane / 16) + v; }
__device__ __forceinline__ int acc_col(int c, int lane) { return 16 * c + lane % 16; }

// The sums over the WK waves of a column tile: fn(i, c, v, sums of each p), each
// in one of those waves. No LDS where WK = 1.
template <int P, int WK>
struct Joint {
  float sums[kWaves][8][P][64];
};
template <int P>
struct Joint<P, 1> {};

template <int RT, int P, int WK, class Fn>
__device__ __forceinline__ void join(Joint<P, WK>& lds, const Sums4<RT, P>& acc, Fn fn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    if constexpr (WK == 1) {
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        float s[P];
#pragma unroll
        for (int p = 0; p < P; ++p) s[p] = acc[i][p][n / 4][n % 4];
        fn(i, n / 4, n % 4, s);
      }
    } else {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int p = 0; p < P; ++p) lds.sums[wave][n][p][lane] = acc[i][p][n / 4][n % 4];
      __syncthreads();
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if (wave % WK != n % WK) continue;
        float s[P] = {};
        const int from = wave / WK * WK;
#pragma unroll
        for (int w = 0; w < WK; ++w)
#pragma unroll
          for (int p = 0; p < P; ++p) s[p] += lds.sums[from + w][n][p][lane];
        fn(i, n / 4, n % 4, s);
      }
      __syncthreads();
    }
  }
}

// f(RT as an integral constant) for each 32 rows of `own`: rows r0 .., one or two
// blocks of 16.
template <class F>
__device__ __forceinline__ void for_rows(const Few4Rows& own, F&& f) {
  for (int r0 = 0; r0 < own.count; r0 += kRows) {
    if (own.count - r0 > 16) f(std::integral_constant<int, 2>{}, r0);
    else f(std::integral_constant<int, 1>{}, r0);
  }
}

// Where the lane's rows r0 .. of A start in bytes, for `of` values a row.
template <bool PACKED, int RT, class RowOf>
__device__ __forceinline__ void row_starts(const Few4Rows& own, int r0, int of, RowOf row_of, uint32_t (&row)[RT]) {
  const uint32_t lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int m = r0 + 16 * i + static_cast<int>(lane % 16);
    row[i] = kOutOfRange;
    if (m < own.count)
      row[i] = PACKED ? static_cast<uint32_t>(own.block + i) * static_cast<uint32_t>(of / kStepK) * kBlockBytes + lane * 16u
                      : (static_cast<uint32_t>(row_of(m)) * static_cast<uint32_t>(of) + 32u * (lane / 16)) * 2u;
  }
}

template <int ACT, int WK, bool FEW>
__global__ void __launch_bounds__(kThreads, FEW ? 4 : 3) up4_kernel(Few4Args a) {
  __shared__ int32_t list[kFew];
  __shared__ Joint<2, WK> joint;
  constexpr int kTiles = kWaves / WK;  // of a workgroup
  const int tiles = a.ffn_dim / kCols, groups = (tiles + kTiles - 1) / kTiles;
  const int unit = uniform(static_cast<int>(blockIdx.x) / groups), group = uniform(static_cast<int>(blockIdx.x) % groups);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int tile = group * kTiles + wave / WK;
  const int steps = a.d_model / kStepK;
  const Few4Rows own = unit_rows<FEW>(a, unit, list);
  if (own.expert < 0) return;
  Weights<2, WK, FEW> w;
  w.first = wave % WK;
  w.last = tile < tiles ? steps : 0;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int64_t at = (static_cast<int64_t>(own.expert) * 2 * tiles + p * tiles + tile) * steps;
    w.set(p, a.w1 + at * kTileBytes, a.s1 + at * kScaleBytes, steps);
  }
  const bool works = w.first < w.last;
  const __amdgpu_buffer_rsrc_t x = make_rsrc(a.x, static_cast<uint32_t>(a.num_tokens) * static_cast<uint32_t>(a.d_model) * 2u);
  for_rows(own, [&](auto rt, int r0) {
    constexpr int RT = decltype(rt)::value;
    Sums4<RT, 2> acc = {};
    if (works) {
      typename Weights<2, WK, FEW>::Ring ring;
      w.start(ring);
      uint32_t row[RT];
      row_starts<false, RT>(own, r0, a.d_model, [&](int m) { return list[m] / a.k; }, row);
      multiply<false, RT, 2, WK>(acc, x, row, w, ring);
    }
    join<RT, 2, WK>(joint, acc, [&](int i, int c, int v, const float (&s)[2]) {
      const int r = r0 + acc_row(i, v, lane), col = acc_col(c, lane);
      if (r >= own.count || tile >= tiles) return;
      const int64_t to = FEW ? static_cast<int64_t>(list[r]) * a.ffn_dim + tile * kCols + col
                             : ((static_cast<int64_t>(own.block + i) * (a.ffn_dim / kStepK) + tile / 4) * kBlockBytes +
                                col / 8 * 1024 + (tile % 4 * 16 + r % 16) * 16) / 2 + col % 8;
      a.h[to] = f32_to_bf16(gated_act<ACT>(s[0]) * s[1]);
    });
  });
}

template <int WK, bool FEW>
__global__ void __launch_bounds__(kThreads, 4) down4_kernel(Few4Args a) {
  __shared__ int32_t list[kFew];
  __shared__ Joint<1, WK> joint;
  constexpr int kTiles = kWaves / WK;
  const int tiles = a.d_model / kCols, groups = (tiles + kTiles - 1) / kTiles;
  int at = static_cast<int>(blockIdx.x);
  const int group = uniform(at % groups);
  at /= groups;
  const int split = uniform(at % a.splits), unit = uniform(at / a.splits);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int tile = group * kTiles + wave / WK;
  const int steps = a.ffn_dim / kStepK;
  const Few4Rows own = unit_rows<FEW>(a, unit, list);
  if (own.expert < 0) return;
  Weights<1, WK, FEW> w;
  w.first = static_cast<int>(static_cast<int64_t>(steps) * split / a.splits) + wave % WK;
  w.last = tile < tiles ? static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / a.splits) : 0;
  const int64_t from = (static_cast<int64_t>(own.expert) * tiles + tile) * steps;
  w.set(0, a.w2 + from * kTileBytes, a.s2 + from * kScaleBytes, steps);
  const bool works = w.first < w.last;
  const int64_t num_copies = static_cast<int64_t>(a.num_tokens) * a.k;
  const __amdgpu_buffer_rsrc_t h =
      make_rsrc(a.h, static_cast<uint32_t>(FEW ? num_copies : a.blocks * 16) * static_cast<uint32_t>(a.ffn_dim) * 2u);
  for_rows(own, [&](auto rt, int r0) {
    constexpr int RT = decltype(rt)::value;
    Sums4<RT, 1> acc = {};
    if (works) {
      typename Weights<1, WK, FEW>::Ring ring;
      w.start(ring);
      uint32_t row[RT];
      row_starts<!FEW, RT>(own, r0, a.ffn_dim, [&](int m) { return list[m]; }, row);
      multiply<!FEW, RT, 1, WK>(acc, h, row, w, ring);
    }
    join<RT, 1, WK>(joint, acc, [&](int i, int c, int v, const float (&s)[1]) {
      const int r = r0 + acc_row(i, v, lane);
      if (r < own.count && tile < tiles)
        a.part[(split * num_copies + list[r]) * a.d_model + tile * kCols + acc_col(c, lane)] = s[0];
    });
  });
}

__device__ __forceinline__ float gate_of(const Few4Args& a, int64_t i) {
  if (a.gate_dtype == SB_DTYPE_F32) return static_cast<const float*>(a.gates)[i];
  const uint16_t bits = static_cast<const uint16_t*>(a.gates)[i];
  return a.gate_dtype == SB_DTYPE_BF16 ? bf16_to_f32(bits) : static_cast<float>(__builtin_bit_cast(_Float16, bits));
}

// The second product and the sum together, for few copies: a workgroup of 16
// waves has 32 columns of out and all copies. Its waves are 16 / WK groups that
// take the experts in turn, of WK waves that share the reduction; each copy's WK
// sums wait in LDS until all are there. One CU then reads all that its columns
// need, so that this pays where the columns make enough workgroups or the
// weights of all copies are few (few4_form).
constexpr int kFusedWaves = 16, kFusedMost = 256;  // copies x WK

template <int WK>
__global__ void __launch_bounds__(64 * kFusedWaves) down_out4_kernel(Few4Args a) {
  __shared__ int32_t lists[kFusedWaves][kFew];
  __shared__ float sums[kFusedMost][kCols];  // [copy][wk]
  const int tiles = a.d_model / kCols, tile = static_cast<int>(blockIdx.x);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int steps = a.ffn_dim / kStepK;
  const __amdgpu_buffer_rsrc_t h =
      make_rsrc(a.h, static_cast<uint32_t>(a.num_tokens * a.k) * static_cast<uint32_t>(a.ffn_dim) * 2u);
  const int share = wave % WK;
  int turn = 0;
  for (int unit = 0; unit < a.units; ++unit) {
    const Few4Rows own = unit_rows<true>(a, unit, lists[wave]);
    if (own.expert < 0) continue;
    if (turn++ % (kFusedWaves / WK) != wave / WK) continue;
    Weights<1, WK, true> w;
    w.first = share;
    w.last = steps;
    const int64_t from = (static_cast<int64_t>(own.expert) * tiles + tile) * steps;
    w.set(0, a.w2 + from * kTileBytes, a.s2 + from * kScaleBytes, steps);
    for_rows(own, [&](auto rt, int r0) {
      constexpr int RT = decltype(rt)::value;
      Sums4<RT, 1> acc = {};
      if (w.first < w.last) {
        typename Weights<1, WK, true>::Ring ring;
        w.start(ring);
        uint32_t row[RT];
        row_starts<false, RT>(own, r0, a.ffn_dim, [&](int m) { return lists[wave][m]; }, row);
        multiply<false, RT, 1, WK>(acc, h, row, w, ring);
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int r = r0 + acc_row(i, v, lane);
            if (r < own.count) sums[lists[wave][r] * WK + share][acc_col(c, lane)] = acc[i][0][c][v];
          }
    });
  }
  __syncthreads();
  const int tokens = copy_limit(a) / a.k;
  for (int item = threadIdx.x; item < tokens * kCols; item += 64 * kFusedWaves) {
    const int t = item / kCols, col = item % kCols;
    float out = 0.0f;
    for (int j = 0; j < a.k; ++j) {
      const int c = t * a.k + j;
      if (expert_of(a, c) < 0) continue;
      float y = 0.0f;
#pragma unroll
      for (int q = 0; q < WK; ++q) y += sums[c * WK + q][col];
      out += gate_of(a, c) * y;
    }
    a.out[static_cast<int64_t>(t) * a.d_model + tile * kCols + col] = f32_to_bf16(out);
  }
}

// A lane owns four columns of a token.
__global__ void __launch_bounds__(256) out4_kernel(Few4Args a) {
  const int quads = a.d_model / 4;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int32_t t = static_cast<int32_t>(item / quads), q = static_cast<int32_t>(item % quads);
  if (t >= copy_limit(a) / a.k) return;
  const int64_t num_copies = static_cast<int64_t>(a.num_tokens) * a.k;
  f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j = 0; j < a.k; ++j) {
    const int64_t c = static_cast<int64_t>(t) * a.k + j;
    if (expert_of(a, static_cast<int32_t>(c)) < 0) continue;
    f32x4_t y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s)
      y += *reinterpret_cast<const f32x4_t*>(a.part + (s * num_copies + c) * a.d_model + 4 * q);
    sum += gate_of(a, c) * y;
  }
  *reinterpret_cast<u32x2_t*>(a.out + static_cast<int64_t>(t) * a.d_model + 4 * q) =
      u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
}

// How many waves share a column tile's reduction (wk): few tiles need it for
// waves enough to keep the memory busy, while many tiles' waves read the same rows
// of x at the same time. More rows a tile (not few) make that count more. The
// second product's tiles are half as many and their reductions longer; where even
// four waves each leave CUs with few, workgroups share it too (splits), through
// memory. us a call, with up4's wk, down4's wk and the splits:
//   T = 1, D = 4096, F = 14336, E = 8   2,4,2 41.8   2,4,1 45.8   4,4,4 45.8   1,1,1 90
//   T = 24, D = 1024, F = 4096, E = 64  1,2,1 56.7   1,4,1 57.1   2,4,1 59.8   4,4,4 73
//   T = 16, D = 4096, F = 14336, E = 8  1,4,1 144    2,2,1 163    2,1,1 180
//   T = 250, D = 2048, F = 768, E = 128 2,1,1 95     2,2,1 97     1,2,1 102    4,4,4 165
//   T = 1, D = 1024, F = 4096, E = 64   4,4,4 12.0   2,4,4 13.1   2,2,1 19
struct Few4Form {
  int units, blocks, up_wk, down_wk, splits, fused_wk;  // fused_wk 0: down4 and out4
};
// Copies x F up to which one workgroup's share of the second product's weights is
// read in about the time that a launch takes. us a call of the GPU, fused and not, top 2
// of 8 experts: T = 1, D = 1024 F = 512 9.1 10.4, F = 1024 10.4 10.7, F = 2048 11.0 11.3, F = 4096
// 12.4 11.0; D = 4096, F = 14336 57 48. More copies take their experts in turn in a wave: T = 4,
// F = 512 11.4 10.6, T = 8, F = 256 12.8 10.6. But a launch takes 3.4 us of the host, whose 12
// us a call without it are the longer of the two unless the call is captured.
constexpr int64_t kFusedMostRead = 4096;

Few4Form few4_form(int64_t copies, int64_t num_experts, int64_t d_model, int64_t ffn_dim, int cus) {
  Few4Form f;
  const bool few = copies <= kFew;
  f.units = static_cast<int>(few ? copies : max_row_tiles(copies, num_experts));
  f.blocks = static_cast<int>(max_row_blocks(copies, num_experts));
  const int64_t up = f.units * (ffn_dim / kCols), down = f.units * (d_model / kCols);  // column tiles
  const int64_t up_steps = d_model / kStepK, down_steps = ffn_dim / kStepK;
  f.up_wk = up >= int64_t{24} * cus || up_steps < 2 ? 1 : !few || up * 2 >= int64_t{6} * cus || up_steps < 4 ? 2 : 4;
  f.down_wk = 1;
  while (f.down_wk < (few ? kWaves : 2) && down * f.down_wk < int64_t{few ? 64 : 24} * cus && down_steps >= 2 * f.down_wk)
    f.down_wk *= 2;
  f.splits = 1;
  while (f.splits < kMaxSplits && down * f.down_wk * f.splits < int64_t{8} * cus &&
         down_steps >= int64_t{4} * f.down_wk * f.splits)
    f.splits *= 2;
  f.fused_wk = 0;
  if (few && copies * ffn_dim <= kFusedMostRead) {
    f.fused_wk = kFusedWaves;
    while (f.fused_wk > 1 && f.fused_wk * copies > kFusedWaves) f.fused_wk /= 2;
  }
  return f;
}

// f(WK as an integral constant).
template <class F>
void with_wk(int wk, F&& f) {
  if (wk == 1) f(std::integral_constant<int, 1>{});
  else if (wk == 2) f(std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 4>{});
}

struct Few4Buffers {
  uint16_t* h;
  float* part;
  int32_t* rows;
  int64_t used;
};

Few4Buffers carve_few4(void* workspace, int64_t copies, int64_t d_model, int64_t ffn_dim, const Few4Form& f) {
  const bool few = copies <= kFew;
  Carver ws{static_cast<uint8_t*>(workspace)};
  Few4Buffers b;
  b.h = ws.take<uint16_t>((few ? copies : f.blocks * int64_t{16}) * ffn_dim);
  b.part = ws.take<float>(f.splits * copies * d_model);
  b.rows = ws.take<int32_t>(few ? 0 : row_words(f.units, copies));
  b.used = ws.used;
  return b;
}

int check_few4(int64_t num_tokens, int32_t k, int32_t num_experts, int64_t d_model, int64_t ffn_dim) {
  if (num_tokens <= 0 || k <= 0 || num_tokens > kMaxCopies / k)
    return fail(SB_ERR_INVALID, "4-bit experts: T, k > 0 and at most %d copies, got %lld x %d", kMaxCopies,
                static_cast<long long>(num_tokens), k);
  if (num_experts <= 0 || num_experts > kMaxExperts)
    return fail(SB_ERR_INVALID, "4-bit experts: num_experts must be in [1, 1024], got %d", num_experts);
  if (d_model <= 0 || d_model % 128 != 0 || ffn_dim <= 0 || ffn_dim % 128 != 0 || d_model > (1 << 20) ||
      ffn_dim > (1 << 20))
    return fail(SB_ERR_INVALID, "4-bit experts: D (%lld) and F (%lld) must be multiples of 128, up to 2^20",
                static_cast<long long>(d_model), static_cast<long long>(ffn_dim));
  // Rows are read with 32-bit buffer offsets.
  if (max_row_blocks(num_tokens * k, num_experts) * 16 * std::max(d_model, ffn_dim) * 2 >= kI32Limit)
    return fail(SB_ERR_INVALID, "4-bit experts: too many copies of too long rows for 32-bit buffer offsets");
  return SB_OK;
}

// ---- codes from weights and back ----

// A lane takes a column's group of 32; lanes of a half wave are neighbouring columns.
__global__ void __launch_bounds__(256)
    quantize4_kernel(const void* __restrict__ w, int32_t dtype, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                     int64_t groups, int32_t k_groups, int64_t n, int64_t k) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;  // [E, N/32, K/32, 32]
  if (item >= groups) return;
  const int col = static_cast<int>(item % kCols);
  const int64_t tile = item / kCols;
  const int64_t kg = tile % k_groups, nt = tile / k_groups % (n / kCols), e = tile / k_groups / (n / kCols);
  const int64_t at = (e * k + kg * 32) * n + nt * kCols + col;
  float v[32];
  float most = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int64_t p = at + i * n;
    if (dtype == SB_DTYPE_F32) {
      v[i] = static_cast<const float*>(w)[p];
    } else {
      const uint16_t bits = static_cast<const uint16_t*>(w)[p];
      v[i] = dtype == SB_DTYPE_BF16 ? bf16_to_f32(bits) : static_cast<float>(__builtin_bit_cast(_Float16, bits));
    }
    most = fmaxf(most, fabsf(v[i]));
    finite = finite && (__float_as_uint(v[i]) & 0x7f800000u) != 0x7f800000u;
  }
  // The largest value lies in [4, 8) steps of the scale (from 6 on it is taken as 6).
  int s = 127;
  if (!finite) s = 255;
  else if (most > 0.0f) s = min(254, max(1, static_cast<int>(__float_as_uint(most) >> 23) - 2));
  scales[item] = static_cast<uint8_t>(s);
  u32x4_t packed = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float a = ldexpf(fabsf(v[i]), 127 - s);
    // To nearest, halves to the even code.
    const uint32_t code = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
    packed[i / 8] |= (finite ? code | (__float_as_uint(v[i]) >> 31) << 3 : 0u) << (4 * (i % 8));
  }
  *reinterpret_cast<u32x4_t*>(codes + item * 16) = packed;
}

__global__ void __launch_bounds__(256)
    dequantize4_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint16_t* __restrict__ w,
                       int64_t groups, int32_t k_groups, int64_t n, int64_t k) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (item >= groups) return;
  const int col = static_cast<int>(item % kCols);
  const int64_t tile = item / kCols;
  const int64_t kg = tile % k_groups, nt = tile / k_groups % (n / kCols), e = tile / k_groups / (n / kCols);
  const int64_t at = (e * k + kg * 32) * n + nt * kCols + col;
  const u32x4_t packed = *reinterpret_cast<const u32x4_t*>(codes + item * 16);
  const float scale = scale_of(scales[item]);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const u32x4_t v = __builtin_bit_cast(u32x4_t, dequantize(packed[q], scale));
#pragma unroll
    for (int i = 0; i < 8; ++i) w[at + (8 * q + i) * n] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
  }
}

int check_codes(const char* what, int64_t num_experts, int64_t k, int64_t n) {
  if (num_experts <= 0 || k <= 0 || n <= 0 || k % 32 != 0 || n % 32 != 0 || k > (1 << 24) || n > (1 << 24) ||
      num_experts > (int64_t{1} << 38) / 4 / (k / 32 * n))
    return fail(SB_ERR_INVALID, "%s: w must be [E, K, N], K and N multiples of 32, got [%lld, %lld, %lld]", what,
                static_cast<long long>(num_experts), static_cast<long long>(k), static_cast<long long>(n));
  return SB_OK;
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_experts4_sizes(int64_t num_tokens, int32_t k, int32_t num_experts, int64_t d_model, int64_t ffn_dim,
                                 int64_t* workspace_bytes) {
  if (const int rc = check_few4(num_tokens, k, num_experts, d_model, ffn_dim)) return rc;
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  const int64_t copies = num_tokens * k;
  const Few4Form f = few4_form(copies, num_experts, d_model, ffn_dim, cus);
  if (workspace_bytes) *workspace_bytes = carve_few4(nullptr, copies, d_model, ffn_dim, f).used;
  return clear_ok();
}

extern "C" int sb_experts4_layer(const void* x, const void* expert_idx, int32_t idx_is_i64, const void* gates,
                                 int32_t gate_dtype, const void* w1_codes, const void* w1_scales, const void* w2_codes,
                                 const void* w2_scales, void* out, int32_t act, void* workspace,
                                 int64_t workspace_bytes, int64_t num_tokens, int32_t k, int32_t num_experts,
                                 int64_t d_model, int64_t ffn_dim, const int32_t* valid_tokens, void* stream) {
  if (const int rc = check_few4(num_tokens, k, num_experts, d_model, ffn_dim)) return rc;
  if (!x || !expert_idx || !gates || !w1_codes || !w1_scales || !w2_codes || !w2_scales || !out)
    return fail(SB_ERR_INVALID, "4-bit experts: null buffer");
  if (!aligned16(x) || !aligned16(w1_codes) || !aligned16(w2_codes) || !aligned16(out))
    return fail(SB_ERR_INVALID, "4-bit experts: x, the codes and out must be 16-byte aligned");
  if (gate_dtype != SB_DTYPE_BF16 && gate_dtype != SB_DTYPE_F16 && gate_dtype != SB_DTYPE_F32)
    return fail(SB_ERR_INVALID, "4-bit experts: unsupported gate dtype code %d", gate_dtype);
  if (act != SB_ACT_SILU && act != SB_ACT_GELU)
    return fail(SB_ERR_INVALID, "4-bit experts: unknown activation code %d", act);
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  const int64_t copies = num_tokens * k;
  const Few4Form f = few4_form(copies, num_experts, d_model, ffn_dim, cus);
  const Few4Buffers b = carve_few4(workspace, copies, d_model, ffn_dim, f);
  if (const int rc = check_workspace(workspace, workspace_bytes, b.used)) return rc;
  Few4Args a{};
  a.x = static_cast<const uint16_t*>(x);
  a.expert_idx = expert_idx;
  a.gates = gates;
  a.w1 = static_cast<const uint8_t*>(w1_codes);
  a.s1 = static_cast<const uint8_t*>(w1_scales);
  a.w2 = static_cast<const uint8_t*>(w2_codes);
  a.s2 = static_cast<const uint8_t*>(w2_scales);
  a.valid_tokens = valid_tokens;
  a.h = b.h;
  a.out = static_cast<uint16_t*>(out);
  a.part = b.part;
  a.idx_is_i64 = idx_is_i64;
  a.num_tokens = static_cast<int32_t>(num_tokens);
  a.k = k;
  a.num_experts = num_experts;
  a.d_model = static_cast<int32_t>(d_model);
  a.ffn_dim = static_cast<int32_t>(ffn_dim);
  a.splits = f.splits;
  a.gate_dtype = gate_dtype;
  a.units = f.units;
  const hipStream_t s = as_stream(stream);
  auto grid = [&](int64_t parts, int64_t columns, int wk) {
    const int64_t tiles = kWaves / wk;
    return dim3(static_cast<uint32_t>(parts * ((columns / kCols + tiles - 1) / tiles)));
  };
  auto launch = [&](auto kernel, dim3 blocks) { kernel<<<blocks, kThreads, 0, s>>>(a); };
  const bool few = copies <= kFew;
  if (!few) {
    rows4_kernel<<<1, kSortThreads, 0, s>>>(a, b.rows, f.units);
    if (const int rc = check_launch("4-bit experts: rows")) return rc;
    a.rows = b.rows;
    a.blocks = f.blocks;
  }
  with_wk(f.up_wk, [&](auto wk) {
    constexpr int WK = decltype(wk)::value;
    const dim3 blocks = grid(f.units, ffn_dim, WK);
    if (act == SB_ACT_SILU) few ? launch(up4_kernel<SB_ACT_SILU, WK, true>, blocks) : launch(up4_kernel<SB_ACT_SILU, WK, false>, blocks);
    else few ? launch(up4_kernel<SB_ACT_GELU, WK, true>, blocks) : launch(up4_kernel<SB_ACT_GELU, WK, false>, blocks);
  });
  if (const int rc = check_launch("4-bit experts")) return rc;
  if (f.fused_wk) {
    const uint32_t blocks = static_cast<uint32_t>(d_model / kCols);
    auto fused = [&](auto kernel) { kernel<<<blocks, 64 * kFusedWaves, 0, s>>>(a); };
    switch (f.fused_wk) {
      case 1: fused(down_out4_kernel<1>); break;
      case 2: fused(down_out4_kernel<2>); break;
      case 4: fused(down_out4_kernel<4>); break;
      case 8: fused(down_out4_kernel<8>); break;
      default: fused(down_out4_kernel<16>); break;
    }
    if (const int rc = check_launch("4-bit experts")) return rc;
    return clear_ok();
  }
  with_wk(f.down_wk, [&](auto wk) {
    constexpr int WK = decltype(wk)::value;
    const dim3 blocks = grid(int64_t{f.units} * f.splits, d_model, WK);
    few ? launch(down4_kernel<WK, true>, blocks) : launch(down4_kernel<WK, false>, blocks);
  });
  if (const int rc = check_launch("4-bit experts")) return rc;
  out4_kernel<<<static_cast<uint32_t>((num_tokens * (d_model / 4) + 255) / 256), 256, 0, s>>>(a);
  if (const int rc = check_launch("4-bit experts")) return rc;
  return clear_ok();
}

extern "C" int sb_quantize4(const void* w, int32_t dtype, void* codes, void* scales, int64_t num_experts, int64_t k,
                            int64_t n, void* stream) {
  if (const int rc = check_codes("quantize4", num_experts, k, n)) return rc;
  if (dtype != SB_DTYPE_BF16 && dtype != SB_DTYPE_F16 && dtype != SB_DTYPE_F32)
    return fail(SB_ERR_INVALID, "quantize4: unsupported dtype code %d", dtype);
  if (!w || !codes || !scales) return fail(SB_ERR_INVALID, "quantize4: null buffer");
  if (!aligned16(codes)) return fail(SB_ERR_INVALID, "quantize4: the codes must be 16-byte aligned");
  const int64_t groups = num_experts * (k / 32) * n;
  quantize4_kernel<<<static_cast<uint32_t>((groups + 255) / 256), 256, 0, as_stream(stream)>>>(
      w, dtype, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), groups, static_cast<int32_t>(k / 32), n, k);
  if (const int rc = check_launch("quantize4")) return rc;
  return clear_ok();
}

extern "C" int sb_dequantize4(const void* codes, const void* scales, void* w, int64_t num_experts, int64_t k, int64_t n,
                              void* stream) {
  if (const int rc = check_codes("dequantize4", num_experts, k, n)) return rc;
  if (!w || !codes || !scales) return fail(SB_ERR_INVALID, "dequantize4: null buffer");
  if (!aligned16(codes)) return fail(SB_ERR_INVALID, "dequantize4: the codes must be 16-byte aligned");
  const int64_t groups = num_experts * (k / 32) * n;
  dequantize4_kernel<<<static_cast<uint32_t>((groups + 255) / 256), 256, 0, as_stream(stream)>>>(
      static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<uint16_t*>(w), groups,
      static_cast<int32_t>(k / 32), n, k);
  if (const int rc = check_launch("dequantize4")) return rc;
  return clear_ok();
}
