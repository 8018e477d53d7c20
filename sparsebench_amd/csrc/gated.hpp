// What the gated experts' kernels share: their launches (one entry point each
// for gated_layer.hip to call), the tile's place in the routing layout and
// the epilogues' staging.
//
// Operands on a routing layout (block size 128), P = padded rows:
//   w1   [E, D, 2F]  gate columns, then up columns
//   w2   [E, F, D]
//   gu   [P, 2F]     G | U, the pre-activations of each row
//   h    BSR blocks [P/128 * F/128, 128, 128]: a(G) U
//   y    [P, D]      H W2
// Rows past an expert's real rows are neither written nor read.
#pragma once

#include <algorithm>
#include <limits>

#include "common.hpp"
#include "expert_chunks.hpp"
#include "gemm_dma.hpp"

namespace sb {

// A routing layout as the kernels read it.
struct GatedLayout {
  const int32_t *row_token, *row_block_expert, *tokens_per_expert, *padded_offsets;
  int32_t num_experts, max_row_blocks;
};

// G | U = x[row_token] W1[e] and H = a(G) U; gu may be null.
int launch_gated_up(const void* x, const void* w1, const GatedLayout& layout, void* h, void* gu, int64_t num_tokens,
                    int64_t num_copies, int64_t d_model, int64_t ffn_dim, int32_t act, hipStream_t stream);

// The whole forward pass for one or two tokens (few_copies; gated_few.hip),
// without a routing layout. workspace: few_workspace_floats of it.
bool few_copies(int64_t num_tokens, int32_t k);
int64_t few_workspace_floats(int64_t num_copies, int64_t d_model, int64_t ffn_dim);
int launch_few(const void* x, const void* expert_idx, int32_t idx_is_i64, const void* gates, int32_t gate_dtype,
               const void* w1, const void* w2, void* out, float* workspace, int64_t num_tokens, int32_t k,
               int64_t num_experts, int64_t d_model, int64_t ffn_dim, int32_t act, const int32_t* valid_tokens,
               hipStream_t stream);

// Per copy c = t k + j in row r: grad_gates[c] = <grad_out[t], y[r]>; per row:
// row_gate[r] = gates[c], xg[r] = x[t], gog[r] = grad_out[t]. expert_order [E]:
// the experts, those with most rows first.
int launch_grad_rows(const void* x, const void* grad_out, const void* y, const GatedLayout& layout,
                     const int32_t* copy_row, const void* gates, int32_t gate_dtype, void* grad_gates, float* row_gate,
                     void* xg, void* gog, int64_t num_tokens, int32_t k, int64_t d_model, int32_t* expert_order,
                     const int32_t* valid_tokens, hipStream_t stream);

// dH = row_gate gog W2[e]^T; grad_gu = dH U a'(G) | dH a(G); wh [P, F] = row_gate a(G) U.
int launch_gated_slope(const void* gog, const void* w2, const void* gu, const float* row_gate,
                       const GatedLayout& layout, void* grad_gu, void* wh, int64_t num_copies, int64_t d_model,
                       int64_t ffn_dim, int32_t act, hipStream_t stream);

// y[P, D] = H W2[e] (gated_down.hip). partial: gated_form's parts (1: unused) of [P, D].
int launch_gated_down(const void* h, const void* w2, const GatedLayout& layout, void* out, float* partial,
                      int64_t num_copies, int64_t d_model, int64_t ffn_dim, hipStream_t stream);

// out[P, N] = a[P, K] b[e]^T, b [E, N, K]. partial: gated_form's parts (1: unused) of [P, N].
int launch_rows_bt(const void* a, const void* b, const GatedLayout& layout, void* out, float* partial,
                   int64_t num_copies, int64_t n, int64_t k, hipStream_t stream);

// out[r] = sum over parts of partial[s][r], for rows with a token.
int launch_join_parts(const float* partial, const GatedLayout& layout, void* out, int32_t parts, int64_t columns,
                      hipStream_t stream);

// out1[e] [M, N] = sum over e's rows of a1[r]^T b1[r], a1 [P, M], b1 [P, N],
// and out2 likewise, in one launch; zeros for an expert with no rows.
int launch_expert_outers(const void* a1, const void* b1, void* out1, int64_t m1, int64_t n1, const void* a2,
                         const void* b2, void* out2, int64_t m2, int64_t n2, const GatedLayout& layout,
                         const int32_t* expert_order, hipStream_t stream);

// out[t] = sum_j y[copy_row[t k + j]], fp32 sums (combine.hip).
int launch_sum_copies(const void* y, const int32_t* copy_row, void* out, int64_t num_tokens, int32_t k,
                      int64_t d_model, int64_t y_rows, const int32_t* valid_tokens, hipStream_t stream);

// ------------------------------------------------------------- in tiles ---

// *p for a uniform p that this kernel does not write: a scalar load. (Of a
// pointer inside a struct the compiler cannot tell, and takes a vector load,
// whose wait is then one for every load before it.)
__device__ __forceinline__ int32_t scalar_load(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)(reinterpret_cast<uintptr_t>(p));
}

// A tile's rows are a Chunk (expert_chunks.hpp): real rows of one expert from
// a padded row that is a multiple of 128.
//
// Two forms, with the same results: row blocks (up to 128 rows, narrow tiles,
// for grids that leave CUs idle) and chunks of up to 320 rows, 256 columns wide.

// Tile `bid` of max_row_blocks * slices -> (row block, column slice); false
// past the live row blocks. Live tiles are spread over the XCDs in contiguous
// ranges, row blocks in groups (tile_coords).
__device__ __forceinline__ bool row_block_tile(int bid, int slices, const GatedLayout& l, Chunk* ch, int* slice) {
  const int live_rb = scalar_load(l.padded_offsets + l.num_experts) / kBS;
  if (live_rb > l.max_row_blocks || bid >= live_rb * slices) return false;
  int rb;
  tile_coords(xcd_remap(bid, live_rb * slices), live_rb, slices, kTileGroup, &rb, slice);
  const int32_t e = scalar_load(l.row_block_expert + rb);
  if (e < 0 || e >= l.num_experts) return false;
  const int32_t n = scalar_load(l.tokens_per_expert + e);
  const int32_t first = rb * kBS - scalar_load(l.padded_offsets + e);
  if (first < 0 || first >= n) return false;  // not a routing layout
  *ch = Chunk{e, rb * kBS, min(n - first, kBS), 4};
  return true;
}

// The chunk form's tiles: chunks of 256 rows, the last of up to 320, x slices of
// 256 columns, 8 waves in two rows of 4 (128 x 64 a wave at 256 rows). Each tile
// is cut to its chunk's rows in steps of R = 2 row groups of 32 (one row of 8 waves would
// take odd R too, but reads more LDS fragments per MFMA than R + 1 groups in
// two rows). An expert's weights are streamed once per 256 rows, and padding
// rows past a chunk's last 64 are neither computed nor read.
//   gated (W1, its rows along K): K steps of 32 through a 4-stage ring, A two
//     steps at a time (APAIR).
//   BT (rows of W1 or W2 as columns): K steps of 64, since a row's piece of 32
//     is half a cache line (D = 4096, F = 14336, 512 rows an expert: 1592 us
//     with steps of 32); 160 KB hold 2 stages of A and 3 of B at R = 8. Weights
//     past the caches up to R = 4, where an expert has no other chunk to share
//     them with (slope of 128 rows an expert 207 -> 198 us; taller ones 990 -> 1067).
constexpr int kGatedRmax = 10, kGatedBN = 256;
template <int R>
using GatedUpCfg = DmaCfg<32 * R, kGatedBN, 32, 4, 2, 4, 0, 2, 5, 1, 1, 0, 0, 0, 0, 1>;
template <int R>
using BtChunkCfg = std::conditional_t<
    (R >= 6), DmaCfg<32 * R, kGatedBN, 64, 2, 2, 4, 0, 0, 5, 1, 0, (R <= 8 ? 3 : 0), 0, 0, 1>,
    DmaCfg<32 * R, kGatedBN, 64, (R == 4 ? 3 : 4), 2, 4, 0, 2, 5, 1, 0, 0, 0, 0, 1>>;

// The last slice may be half a slice (columns are multiples of 128).
__host__ __device__ __forceinline__ int gated_slices(int64_t columns) {
  return static_cast<int>((columns + kGatedBN - 1) / kGatedBN);
}

// f(integral_constant<int, R>) for a chunk of `groups` row groups.
template <class F>
__device__ __forceinline__ void with_chunk_groups(int groups, F&& f) {
  static_for<1, kGatedRmax / 2 + 1>([&](auto rc) {
    constexpr int R = 2 * decltype(rc)::value;
    if (groups == R - 1 || groups == R) f(std::integral_constant<int, R>{});
  });
}

// Tile `bid` of the chunk form; false past its tiles. Experts of several chunks
// come first, in order, then the others, largest first, so that the last tiles
// to start are short. Workgroups go to the XCDs one by one, so whatever the
// routing every XCD gets a like share of full tiles and small ones (with a
// contiguous range of tiles an XCD, two chunks leave six XCDs idle: D = 4096,
// F = 14336, one token, 222 against 71 us). An expert of c chunks runs in bands of
// 8 slices, chunk by chunk: a slice's chunks follow each other on one XCD, if
// the slices are a multiple of 8, and meet its weights in that L2.
__device__ __forceinline__ bool gated_chunk_tile(int bid, int slices, const GatedLayout& l, Chunk* ch, int* slice) {
  const int32_t first = expert_counts(l.tokens_per_expert, l.num_experts, 0);
  auto counts = [&](int base) { return base == 0 ? first : expert_counts(l.tokens_per_expert, l.num_experts, base); };
  auto chunks_of = [](int32_t n) { return n > 32 * kGatedRmax ? Chunking<kGatedRmax>::count(n) : 0; };  // several
  int several = 0;
#pragma unroll 1
  for (int base = 0; base < l.num_experts; base += 64) several += wave_inclusive_scan_total(chunks_of(counts(base)));
  const int c = uniform(bid / slices);
  if (c >= several) {
    int32_t hist[kGatedRmax + 1];
    single_chunk_hist<kGatedRmax>(l.tokens_per_expert, l.num_experts, first, hist);
    *ch = find_single_chunk_by_size<kGatedRmax>(l.tokens_per_expert, l.num_experts, c - several, first, hist);
    *slice = uniform(bid - c * slices);
  } else {
    int before = 0, rows_before = 0;
#pragma unroll 1
    for (int base = 0; base < l.num_experts; base += 64) {
      const int32_t n = counts(base);
      const int mine = chunks_of(n);
      const int incl = wave_inclusive_scan(mine), padded = wave_inclusive_scan(padded_rows(n));
      const uint64_t reach = __ballot(before + incl > c);
      if (reach != 0) {
        const int e = __builtin_ctzll(reach);
        const int count = lane_value(mine, e);
        const int t = bid - (before + lane_value(incl, e) - count) * slices;  // among the expert's tiles
        const int band = uniform(t / (kNumXcd * count));
        const int width = min(kNumXcd, slices - band * kNumXcd);
        const int in = t - band * kNumXcd * count;
        const int i = uniform(in / width);
        *slice = uniform(band * kNumXcd + in - i * width);
        const int start = i * Chunking<kGatedRmax>::kRows;
        ch->expert = uniform(base + e);
        ch->row0 = uniform(rows_before + lane_value(padded - padded_rows(n), e) + start);
        ch->rows = uniform(i + 1 < count ? Chunking<kGatedRmax>::kRows : lane_value(n, e) - start);
        ch->groups = (ch->rows + 31) / 32;
        break;
      }
      before += lane_value(incl, 63);
      rows_before += lane_value(padded, 63);
    }
  }
  // None, or not a routing layout (the chunk would leave the buffers): skip it.
  return ch->expert >= 0 && ch->row0 >= 0 && ch->rows >= 1 && ch->groups <= kGatedRmax &&
         ch->row0 + ch->rows <= l.max_row_blocks * kBS;
}

// How a product of `columns` columns and a reduction over k runs on a layout.
struct GatedForm {
  bool chunks;    // the chunk form, else row blocks in 128-wide tiles
  int32_t parts;  // of the reduction, each a workgroup's
  int64_t grid;
};

// Row blocks while their 128-wide tiles have a CU each (each live row block
// holds a copy at least), chunks once those fill the CUs too; in between, and
// for the parts of the reduction, whatever this estimate of the time makes
// shortest. A round of workgroups takes 3 us and 0.65 us for 64 of the reduction
// (128 x 128 tiles; up to 4 times that for chunks of 256 rows), and the sum of
// the parts 6 us and its bytes at 5 TB/s. (E = 3, D = 384, F = 6400, 54 copies: y = H
// W2 in 9 tiles 61 us, in 16 parts 9 and their sum 6.5; E = 8, D = 256, F = 6016, 16704
// copies: dXr in 66 chunk tiles 364 us, in 3 parts 181 and 11.) The CUs are
// counted as 256 whatever the device, so that the workspace's size and the order
// of the sums do not depend on it.
inline GatedForm gated_form(int64_t max_row_blocks, int64_t num_experts, int64_t num_copies, int64_t columns,
                            int64_t k, bool splits) {
  constexpr int64_t kCus = 256;
  const int64_t narrow = std::min(max_row_blocks, num_copies) * (columns / 128);
  // An expert of n rows has ceil(n / 256) chunks, or one less if the last piece
  // joins the one before, so N copies at most N / 256 + min(E, N).
  const int64_t chunks =
      std::min(max_row_blocks, num_copies / Chunking<kGatedRmax>::kRows + std::min(num_experts, num_copies));
  const int64_t wide = chunks * gated_slices(columns);
  GatedForm best{true, 1, wide};
  double least = std::numeric_limits<double>::infinity();
  auto consider = [&](bool is_chunks, int64_t busy, int64_t tiles, double step_us) {
    const int64_t most = splits ? std::min<int64_t>(16, k / 256) : 1;
    for (int64_t parts = 1; parts <= std::max<int64_t>(1, most); ++parts) {
      const int64_t rounds = (busy * parts + kCus - 1) / kCus, steps = (k / 64 + parts - 1) / parts;
      const double sum_us = parts > 1 ? 6.0 + static_cast<double>(parts * num_copies) * columns * 8 / 5e6 : 0.0;
      const double us = rounds * (3.0 + step_us * steps) + sum_us;
      if (us < least) best = GatedForm{is_chunks, static_cast<int32_t>(parts), tiles * parts}, least = us;
    }
  };
  if (narrow <= kCus || wide < kCus) consider(false, narrow, max_row_blocks * (columns / 128), 0.65);
  if (narrow > kCus && wide < kCus)
    consider(true, wide, wide, 0.65 * (1.0 + 3.0 * std::min(1.0, static_cast<double>(num_copies) / (256.0 * chunks))));
  return best;
}

// Where a split product's parts go: [parts, P, columns] sums.
struct SplitOut {
  float* partial;
  int32_t parts, tiles;  // tiles of each part
};
inline SplitOut split_out(const GatedForm& f, float* partial) {
  return {partial, f.parts, static_cast<int32_t>(f.grid / f.parts)};
}

// Workgroup *tile of a split product -> its tile and part.
__device__ __forceinline__ void split_tile(const SplitOut& s, int* tile, int* part) {
  *part = uniform(*tile / s.tiles);
  *tile -= *part * s.tiles;
}

// The first of `blocks` that part i of `parts` takes.
__device__ __forceinline__ int split_start(int i, int parts, int blocks) {
  return static_cast<int>(static_cast<int64_t>(i) * blocks / parts);
}

// A tile of part `part`, straight from the accumulators: a lane's 4 columns of
// a row at a time (the two halves of the wave side by side).
template <class Cfg>
__device__ __forceinline__ void store_part(const SplitOut& s, const typename DmaMainloop<Cfg>::Acc& acc, int part,
                                           const GatedLayout& l, const Chunk& ch, int n0, int columns) {
  using ML = DmaMainloop<Cfg>;
  float* out = s.partial + (static_cast<int64_t>(part) * l.max_row_blocks * kBS + ch.row0) * columns + n0;
#pragma unroll
  for (int i = 0; i < Cfg::TM; ++i) {
    const int r = ML::out_row(i);
    if (r >= ch.rows) continue;
#pragma unroll
    for (int jn = 0; jn < Cfg::TN; ++jn)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int col = ML::out_col(jn, g);
        if (n0 + col < columns)
          *reinterpret_cast<f32x4_t*>(out + static_cast<int64_t>(r) * columns + col) = f32x4_t{
              acc[jn][i][4 * g], acc[jn][i][4 * g + 1], acc[jn][i][4 * g + 2], acc[jn][i][4 * g + 3]};
      }
  }
}

// LDS offset of 16-byte chunk `chunk` of row r in a staged tile of ROW_BYTES
// a row: the rows that one store instruction touches spread over the banks.
template <int ROW_BYTES>
__device__ __forceinline__ int staged_at(int r, int chunk) {
  constexpr int kMask = (ROW_BYTES / 16 < 32 ? ROW_BYTES / 16 : 32) - 1;
  return r * ROW_BYTES + ((chunk ^ (r & kMask)) << 4);
}

}  // namespace sb
