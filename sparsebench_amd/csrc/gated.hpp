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

// Per copy c = t k + j in row r: grad_gates[c] = <grad_out[t], y[r]>; per row:
// row_gate[r] = gates[c], xg[r] = x[t], gog[r] = grad_out[t].
int launch_grad_rows(const void* x, const void* grad_out, const void* y, const GatedLayout& layout,
                     const int32_t* copy_row, const void* gates, int32_t gate_dtype, void* grad_gates, float* row_gate,
                     void* xg, void* gog, int64_t num_tokens, int32_t k, int64_t d_model,
                     const int32_t* valid_tokens, hipStream_t stream);

// dH = row_gate gog W2[e]^T; grad_gu = dH U a'(G) | dH a(G); wh [P, F] = row_gate a(G) U.
int launch_gated_slope(const void* gog, const void* w2, const void* gu, const float* row_gate,
                       const GatedLayout& layout, void* grad_gu, void* wh, int64_t num_copies, int64_t d_model,
                       int64_t ffn_dim, int32_t act, hipStream_t stream);

// out[P, N] = a[P, K] b[e]^T, b [E, N, K].
int launch_rows_bt(const void* a, const void* b, const GatedLayout& layout, void* out, int64_t num_copies, int64_t n,
                   int64_t k, hipStream_t stream);

// out[e] [M, N] = sum over e's rows of a[r]^T b[r], a [P, M], b [P, N]; zeros for an expert with no rows.
int launch_expert_outer(const void* a, const void* b, const GatedLayout& layout, void* out, int64_t m, int64_t n,
                        hipStream_t stream);

// out[t] = sum_j y[copy_row[t k + j]], fp32 sums (combine.hip).
int launch_sum_copies(const void* y, const int32_t* copy_row, void* out, int64_t num_tokens, int32_t k,
                      int64_t d_model, int64_t y_rows, const int32_t* valid_tokens, hipStream_t stream);

// ------------------------------------------------------------- in tiles ---

// The row block of a tile: its expert, first padded row and real rows (1 .. 128).
struct RowBlock {
  int32_t expert, row0, rows;
};

// Tile `bid` of max_row_blocks * slices -> (row block, column slice); false
// past the live row blocks. Live tiles are spread over the XCDs in contiguous
// ranges, row blocks in groups (tile_coords).
__device__ __forceinline__ bool row_block_tile(int bid, int slices, const GatedLayout& l, int group, RowBlock* b,
                                               int* slice) {
  const int live_rb = __builtin_amdgcn_readfirstlane(l.padded_offsets[l.num_experts]) / kBS;
  if (live_rb > l.max_row_blocks || bid >= live_rb * slices) return false;
  int rb;
  tile_coords(xcd_remap(bid, live_rb * slices), live_rb, slices, group, &rb, slice);
  const int32_t e = __builtin_amdgcn_readfirstlane(l.row_block_expert[rb]);
  if (e < 0 || e >= l.num_experts) return false;
  const int32_t n = __builtin_amdgcn_readfirstlane(l.tokens_per_expert[e]);
  const int32_t first = rb * kBS - __builtin_amdgcn_readfirstlane(l.padded_offsets[e]);
  if (first < 0 || first >= n) return false;  // not a routing layout
  b->expert = e;
  b->row0 = rb * kBS;
  b->rows = min(n - first, kBS);
  return true;
}

// LDS offset of 16-byte chunk `chunk` of row r in a staged tile of ROW_BYTES
// a row: the rows that one store instruction touches spread over the banks.
template <int ROW_BYTES>
__device__ __forceinline__ int staged_at(int r, int chunk) {
  constexpr int kMask = (ROW_BYTES / 16 < 32 ? ROW_BYTES / 16 : 32) - 1;
  return r * ROW_BYTES + ((chunk ^ (r & kMask)) << 4);
}

}  // namespace sb
