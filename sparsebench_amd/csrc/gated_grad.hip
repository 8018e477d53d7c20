// The backward pass of the gated experts on a routing layout, P padded rows:
//
//   grad_rows     grad_gates[t, j] = <grad_out[t], y[r]>, and x's and
//                 grad_out's rows gathered by padded row (xg, gog [P, D])
//   gated_slope   dH = w[r] gog W2[e]^T;  dG = dH U a'(G), dU = dH a(G)
//                 (grad_gu [P, 2F]), and wh = w[r] a(G) U (bf16, one rounding)
//   rows_bt       dXr = [dG | dU] W1[e]^T
//   expert_outer  dW1[e] = xg^T [dG | dU],  dW2[e] = wh^T gog over e's rows
//
// and dx[t] = sum over t's rows of dXr (combine.hip). The products run on the
// LDS-DMA main loop: rows_bt and gated_slope with B's columns as rows (BT:
// W1 and W2 are read as they are stored), expert_outer with both operands
// along K (AT). Rows past an expert's real rows are read as zeros (past the
// buffer's end) and not written.
//
// Gathering x and grad_out once (2 P D values, a few percent of the weights'
// bytes) lets expert_outer's loads be plain: its K runs over rows, so a
// gather inside would need other addresses at every K step.

#include "gated.hpp"
#include "gated_act.hpp"

namespace sb {
namespace {

// ------------------------------------------------------------- rows ---

template <typename G>
__device__ __forceinline__ float load_gate(const G* g, int64_t i);
template <>
__device__ __forceinline__ float load_gate<uint16_t>(const uint16_t* g, int64_t i) {
  return bf16_to_f32(g[i]);
}
template <>
__device__ __forceinline__ float load_gate<_Float16>(const _Float16* g, int64_t i) {
  return static_cast<float>(g[i]);
}
template <>
__device__ __forceinline__ float load_gate<float>(const float* g, int64_t i) {
  return g[i];
}
__device__ __forceinline__ void store_gate(uint16_t* g, int64_t i, float v) { g[i] = f32_to_bf16(v); }
__device__ __forceinline__ void store_gate(_Float16* g, int64_t i, float v) { g[i] = static_cast<_Float16>(v); }
__device__ __forceinline__ void store_gate(float* g, int64_t i, float v) { g[i] = v; }

// One wave per padded row, then one lane per copy for those without a row
// (gradient 0). The row's copy is the one of its token's k that sits in it.
// Bound by memory: reads x, grad_out and y, writes xg and gog, 16 bytes a lane.
template <typename G>
__global__ void __launch_bounds__(256)
    grad_rows_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ grad_out,
                     const uint16_t* __restrict__ y, GatedLayout layout, const int32_t* __restrict__ copy_row,
                     const G* __restrict__ gates, G* __restrict__ grad_gates, float* __restrict__ row_gate,
                     uint16_t* __restrict__ xg, uint16_t* __restrict__ gog, int64_t num_tokens, int32_t k,
                     int32_t d_model, int32_t row_groups, const int32_t* __restrict__ valid_tokens) {
  if (static_cast<int32_t>(blockIdx.x) >= row_groups) {
    const int64_t c = (static_cast<int64_t>(blockIdx.x) - row_groups) * 256 + threadIdx.x;
    const int64_t limit = valid_tokens ? min(num_tokens, static_cast<int64_t>(*valid_tokens)) : num_tokens;
    if (c < limit * k && copy_row[c] < 0) store_gate(grad_gates, c, 0.0f);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int32_t r = uniform(static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 6));
  if (r >= layout.max_row_blocks * kBS) return;
  const int32_t t = uniform(layout.row_token[r]);
  if (t < 0 || t >= num_tokens) return;
  int64_t copy = -1;
  for (int32_t j0 = 0; j0 < k; j0 += 64) {
    const bool here = j0 + lane < k && copy_row[static_cast<int64_t>(t) * k + j0 + lane] == r;
    const uint64_t found = __ballot(here);
    if (found) copy = static_cast<int64_t>(t) * k + j0 + __builtin_ctzll(found);
  }
  const int64_t from = static_cast<int64_t>(t) * d_model, to = static_cast<int64_t>(r) * d_model;
  float dot = 0.0f;
  for (int32_t c = lane * 8; c < d_model; c += 512) {
    const u32x4_t go = *reinterpret_cast<const u32x4_t*>(grad_out + from + c);
    const u32x4_t yr = *reinterpret_cast<const u32x4_t*>(y + to + c);
    const u32x4_t xr = *reinterpret_cast<const u32x4_t*>(x + from + c);
    *reinterpret_cast<u32x4_t*>(gog + to + c) = go;
    *reinterpret_cast<u32x4_t*>(xg + to + c) = xr;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      dot = fmaf(__uint_as_float(go[q] << 16), __uint_as_float(yr[q] << 16), dot);
      dot = fmaf(__uint_as_float(go[q] & 0xffff0000u), __uint_as_float(yr[q] & 0xffff0000u), dot);
    }
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) dot += __shfl_xor(dot, s);
  if (lane == 0 && copy >= 0) {
    store_gate(grad_gates, copy, dot);
    row_gate[r] = load_gate(gates, copy);
  }
}

template <typename G>
int run_grad_rows(const void* x, const void* grad_out, const void* y, const GatedLayout& layout,
                  const int32_t* copy_row, const void* gates, void* grad_gates, float* row_gate, void* xg, void* gog,
                  int64_t num_tokens, int32_t k, int64_t d_model, const int32_t* valid_tokens, hipStream_t stream) {
  const int32_t row_groups = layout.max_row_blocks * (kBS / 4);
  const int64_t groups = row_groups + (num_tokens * k + 255) / 256;
  grad_rows_kernel<G><<<static_cast<uint32_t>(groups), 256, 0, stream>>>(
      static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(grad_out), static_cast<const uint16_t*>(y), layout,
      copy_row, static_cast<const G*>(gates), static_cast<G*>(grad_gates), row_gate, static_cast<uint16_t*>(xg),
      static_cast<uint16_t*>(gog), num_tokens, k, static_cast<int32_t>(d_model), row_groups, valid_tokens);
  return check_launch("gated backward: rows");
}

// ------------------------------------------------- products with W^T ---

// A: rows row0 .. of a [P, K] (rows past `rows` read as zeros); B: rows n0 ..
// of b[e] [N, K]. Both advance BK * 2 bytes a K step.
template <class Cfg>
struct RowsBtSrc {
  __amdgpu_buffer_rsrc_t ra, rb;
  uint32_t a_off[Cfg::kAInstr], b_off[Cfg::kBInstr];
  __device__ __forceinline__ uint32_t a_voff(int q) const { return a_off[q]; }
  __device__ __forceinline__ uint32_t b_voff(int q) const { return b_off[q]; }
  __device__ __forceinline__ void a_src(int t, __amdgpu_buffer_rsrc_t* r, uint32_t* s) const {
    *r = ra;
    *s = static_cast<uint32_t>(t) * (Cfg::BK * 2);
  }
  __device__ __forceinline__ void b_src(int t, __amdgpu_buffer_rsrc_t* r, uint32_t* s) const {
    *r = rb;
    *s = static_cast<uint32_t>(t) * (Cfg::BK * 2);
  }
  __device__ __forceinline__ RowsBtSrc(const uint16_t* a, const uint16_t* b, const RowBlock& block, int32_t n0,
                                       int32_t n, int32_t k) {
    ra = make_rsrc(a + static_cast<int64_t>(block.row0) * k, static_cast<uint32_t>(block.rows) * k * 2u);
    rb = make_rsrc(b + static_cast<int64_t>(block.expert) * n * k,
                   static_cast<uint32_t>(n) * static_cast<uint32_t>(k) * 2u);
    const ADmaPos<Cfg> ap;
#pragma unroll
    for (int q = 0; q < Cfg::kAInstr; ++q)
      a_off[q] = ap.row[q] < block.rows ? (static_cast<uint32_t>(ap.row[q]) * k + ap.chunk[q] * 8) * 2u : kOutOfRange;
    const BtDmaPos<Cfg> bp;
#pragma unroll
    for (int q = 0; q < Cfg::kBInstr; ++q)
      b_off[q] = (static_cast<uint32_t>(n0 + bp.row[q]) * k + bp.chunk[q] * 8) * 2u;
  }
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads)
    rows_bt_kernel(const uint16_t* __restrict__ a, const uint16_t* __restrict__ b, GatedLayout layout,
                   uint16_t* __restrict__ out, int32_t n, int32_t k) {
  using ML = DmaMainloop<Cfg>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsAlloc];
  RowBlock block;
  int slice;
  if (!row_block_tile(static_cast<int>(blockIdx.x), n / Cfg::BN, layout, kTileGroup, &block, &slice)) return;
  const int n0 = slice * Cfg::BN;
  const RowsBtSrc<Cfg> src(a, b, block, n0, n, k);
  typename ML::Acc acc;
  ML::run(lds, src, k / Cfg::BK, acc);
  ML::stage_tile(lds, acc, [](float v) { return v; });
  uint16_t* rows = out + static_cast<int64_t>(block.row0) * n + n0;
  ML::for_each_staged_chunk(lds, [&](int r, int col, u32x4_t v) {
    if (r < block.rows) *reinterpret_cast<u32x4_t*>(rows + static_cast<int64_t>(r) * n + col) = v;
  });
}

// The epilogue stages the tile as fp32 (a lane's results are 4 columns of 32
// rows), then each lane takes 8 columns of a row: 16-byte loads of G and U,
// 16-byte stores of dG, dU and wh.
template <class Cfg, int ACT>
__global__ void __launch_bounds__(Cfg::kThreads)
    gated_slope_kernel(const uint16_t* __restrict__ gog, const uint16_t* __restrict__ w2,
                       const uint16_t* __restrict__ gu, const float* __restrict__ row_gate, GatedLayout layout,
                       uint16_t* __restrict__ grad_gu, uint16_t* __restrict__ wh, int32_t d_model, int32_t ffn_dim) {
  using ML = DmaMainloop<Cfg>;
  constexpr int BN = Cfg::BN, kRowBytes = BN * 4;
  constexpr int kLds = Cfg::kLdsAlloc > kBS * kRowBytes ? Cfg::kLdsAlloc : kBS * kRowBytes;
  static_assert(Cfg::BM == kBS && kLds <= 160 * 1024, "the fp32 tile fits LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
  RowBlock block;
  int slice;
  if (!row_block_tile(static_cast<int>(blockIdx.x), ffn_dim / BN, layout, kTileGroup, &block, &slice)) return;
  const int n0 = slice * BN;
  const RowsBtSrc<Cfg> src(gog, w2, block, n0, ffn_dim, d_model);
  typename ML::Acc acc;
  ML::run(lds, src, d_model / Cfg::BK, acc);

  __syncthreads();  // every wave is done reading the ring
#pragma unroll
  for (int jn = 0; jn < Cfg::TN; ++jn)
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i) {
      const int m = ML::out_row(i);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4_t v = {acc[jn][i][4 * g], acc[jn][i][4 * g + 1], acc[jn][i][4 * g + 2], acc[jn][i][4 * g + 3]};
        *reinterpret_cast<f32x4_t*>(lds + staged_at<kRowBytes>(m, ML::out_col(jn, g) >> 2)) = v;
      }
    }
  __syncthreads();
  constexpr int kChunksPerRow = BN / 8;
  for (int q = threadIdx.x; q < block.rows * kChunksPerRow; q += Cfg::kThreads) {
    const int r = q / kChunksPerRow, c = q % kChunksPerRow;
    const int64_t row = block.row0 + r;
    const int64_t at = row * 2 * ffn_dim + n0 + c * 8;
    const u32x4_t gv = *reinterpret_cast<const u32x4_t*>(gu + at);
    const u32x4_t uv = *reinterpret_cast<const u32x4_t*>(gu + at + ffn_dim);
    const float w = row_gate[row];
    const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(lds + staged_at<kRowBytes>(r, 2 * c));
    const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(lds + staged_at<kRowBytes>(r, 2 * c + 1));
    u32x4_t dg, du, hw;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      float og[2], ou[2], oh[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float g = __uint_as_float(e ? gv[p] & 0xffff0000u : gv[p] << 16);
        const float u = __uint_as_float(e ? uv[p] & 0xffff0000u : uv[p] << 16);
        const float dh = w * (p < 2 ? lo[2 * p + e] : hi[2 * p - 4 + e]);
        const ActSlope a = gated_act_slope<ACT>(g);
        og[e] = dh * u * a.slope;
        ou[e] = dh * a.value;
        oh[e] = w * (a.value * u);
      }
      dg[p] = pack_bf16x2(og[0], og[1]);
      du[p] = pack_bf16x2(ou[0], ou[1]);
      hw[p] = pack_bf16x2(oh[0], oh[1]);
    }
    *reinterpret_cast<u32x4_t*>(grad_gu + at) = dg;
    *reinterpret_cast<u32x4_t*>(grad_gu + at + ffn_dim) = du;
    *reinterpret_cast<u32x4_t*>(wh + row * ffn_dim + n0 + c * 8) = hw;
  }
}

// ------------------------------------------------- weight gradients ---

// K step t: rows t BK .. of the expert's `rows` rows of a [P, M] and b [P, N].
// Each step's buffers start at its first row and end at the expert's last
// one, so rows past it read as zeros.
template <class Cfg>
struct OuterSrc {
  const uint16_t *a, *b;  // the expert's first row, at the tile's first column
  int32_t rows, m, n;
  uint32_t a_off[Cfg::kAInstr], b_off[Cfg::kBInstr];
  __device__ __forceinline__ uint32_t a_voff(int q) const { return a_off[q]; }
  __device__ __forceinline__ uint32_t b_voff(int q) const { return b_off[q]; }
  // The bytes from a tile's first column in a step's first row to its last
  // column in the last row that is there.
  __device__ __forceinline__ static uint32_t bytes(int32_t left, int32_t stride, int32_t width) {
    return static_cast<uint32_t>((min(left, static_cast<int32_t>(Cfg::BK)) - 1) * stride + width) * 2u;
  }
  __device__ __forceinline__ void a_src(int t, __amdgpu_buffer_rsrc_t* r, uint32_t* s) const {
    *r = make_rsrc(a + static_cast<int64_t>(t) * Cfg::BK * m, bytes(rows - t * Cfg::BK, m, Cfg::BM));
    *s = 0;
  }
  __device__ __forceinline__ void b_src(int t, __amdgpu_buffer_rsrc_t* r, uint32_t* s) const {
    *r = make_rsrc(b + static_cast<int64_t>(t) * Cfg::BK * n, bytes(rows - t * Cfg::BK, n, Cfg::BN));
    *s = 0;
  }
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads)
    expert_outer_kernel(const uint16_t* __restrict__ a, const uint16_t* __restrict__ b, GatedLayout layout,
                        uint16_t* __restrict__ out, int32_t m, int32_t n) {
  using ML = DmaMainloop<Cfg>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsAlloc];
  const int slices = n / Cfg::BN, row_tiles = m / Cfg::BM;
  const int per_expert = slices * row_tiles;
  const int tile = xcd_remap(static_cast<int>(blockIdx.x), layout.num_experts * per_expert);
  const int e = uniform(tile / per_expert);
  int mt, nt;
  tile_coords(tile - e * per_expert, row_tiles, slices, kTileGroup, &mt, &nt);
  const int m0 = mt * Cfg::BM, n0 = nt * Cfg::BN;
  const int32_t rows = uniform(layout.tokens_per_expert[e]);
  const int32_t row0 = uniform(layout.padded_offsets[e]);
  uint16_t* tile_out = out + (static_cast<int64_t>(e) * m + m0) * n + n0;

  OuterSrc<Cfg> src;
  src.a = a + static_cast<int64_t>(row0) * m + m0;
  src.b = b + static_cast<int64_t>(row0) * n + n0;
  src.rows = rows;
  src.m = m;
  src.n = n;
  const AtDmaPos<Cfg> ap;
#pragma unroll
  for (int q = 0; q < Cfg::kAInstr; ++q) src.a_off[q] = (static_cast<uint32_t>(ap.row[q]) * m + ap.col[q]) * 2u;
  const BDmaPos<Cfg> bp;
#pragma unroll
  for (int q = 0; q < Cfg::kBInstr; ++q) src.b_off[q] = (static_cast<uint32_t>(bp.row[q]) * n + bp.col[q]) * 2u;

  typename ML::Acc acc;
  ML::run(lds, src, (rows + Cfg::BK - 1) / Cfg::BK, acc);  // no rows: zeros
  ML::stage_tile(lds, acc, [](float v) { return v; });
  ML::for_each_staged_chunk(lds, [&](int r, int col, u32x4_t v) {
    *reinterpret_cast<u32x4_t*>(tile_out + static_cast<int64_t>(r) * n + col) = v;
  });
}

using BtWide = DmaCfg<128, 256, 64, 3, 2, 4, 0, 0, 3, 1, 0, 0, 0, 0, 1>;
using BtNarrow = DmaCfg<128, 128, 64, 3, 2, 2, 0, 0, 5, 1, 0, 0, 0, 0, 1>;
using OuterWide = DmaCfg<128, 256, 32, 3, 2, 4, 0, 0, 5, 1, 0, 0, 0, 1>;
using OuterNarrow = DmaCfg<128, 128, 32, 3, 2, 2, 0, 0, 5, 1, 0, 0, 0, 1>;

template <class Cfg, int ACT>
int run_slope(const void* gog, const void* w2, const void* gu, const float* row_gate, const GatedLayout& layout,
              void* grad_gu, void* wh, int64_t d_model, int64_t ffn_dim, hipStream_t stream) {
  const int64_t tiles = layout.max_row_blocks * (ffn_dim / Cfg::BN);
  gated_slope_kernel<Cfg, ACT><<<static_cast<uint32_t>(tiles), Cfg::kThreads, 0, stream>>>(
      static_cast<const uint16_t*>(gog), static_cast<const uint16_t*>(w2), static_cast<const uint16_t*>(gu), row_gate,
      layout, static_cast<uint16_t*>(grad_gu), static_cast<uint16_t*>(wh), static_cast<int32_t>(d_model),
      static_cast<int32_t>(ffn_dim));
  return check_launch("gated backward: slope");
}

template <class Cfg>
int run_rows_bt(const void* a, const void* b, const GatedLayout& layout, void* out, int64_t n, int64_t k,
                hipStream_t stream) {
  const int64_t tiles = layout.max_row_blocks * (n / Cfg::BN);
  rows_bt_kernel<Cfg><<<static_cast<uint32_t>(tiles), Cfg::kThreads, 0, stream>>>(
      static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(b), layout, static_cast<uint16_t*>(out),
      static_cast<int32_t>(n), static_cast<int32_t>(k));
  return check_launch("gated backward: rows @ w^T");
}

template <class Cfg>
int run_outer(const void* a, const void* b, const GatedLayout& layout, void* out, int64_t m, int64_t n,
              hipStream_t stream) {
  const int64_t tiles = layout.num_experts * (m / Cfg::BM) * (n / Cfg::BN);
  if (tiles > 2147483647LL) return fail(SB_ERR_INVALID, "gated backward: too many tiles");
  expert_outer_kernel<Cfg><<<static_cast<uint32_t>(tiles), Cfg::kThreads, 0, stream>>>(
      static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(b), layout, static_cast<uint16_t*>(out),
      static_cast<int32_t>(m), static_cast<int32_t>(n));
  return check_launch("gated backward: weight gradient");
}

// 256 columns, or 128 when 256 do not divide them or leave CUs without a tile.
int bt_width(const GatedLayout& layout, int64_t num_copies, int64_t n, int* width) {
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  *width = std::min(256, fit_width(std::min<int64_t>(layout.max_row_blocks, num_copies), n, cus));
  return SB_OK;
}

}  // namespace

int launch_grad_rows(const void* x, const void* grad_out, const void* y, const GatedLayout& layout,
                     const int32_t* copy_row, const void* gates, int32_t gate_dtype, void* grad_gates, float* row_gate,
                     void* xg, void* gog, int64_t num_tokens, int32_t k, int64_t d_model,
                     const int32_t* valid_tokens, hipStream_t stream) {
  auto run = [&](auto tag) {
    return run_grad_rows<decltype(tag)>(x, grad_out, y, layout, copy_row, gates, grad_gates, row_gate, xg, gog,
                                        num_tokens, k, d_model, valid_tokens, stream);
  };
  switch (gate_dtype) {
    case SB_DTYPE_BF16: return run(uint16_t{});
    case SB_DTYPE_F16: return run(_Float16{});
    default: return run(float{});
  }
}

int launch_gated_slope(const void* gog, const void* w2, const void* gu, const float* row_gate,
                       const GatedLayout& layout, void* grad_gu, void* wh, int64_t num_copies, int64_t d_model,
                       int64_t ffn_dim, int32_t act, hipStream_t stream) {
  int width = 0;
  if (const int rc = bt_width(layout, num_copies, ffn_dim, &width)) return rc;
  auto run = [&](auto launch) {
    return launch(gog, w2, gu, row_gate, layout, grad_gu, wh, d_model, ffn_dim, stream);
  };
  if (width == 256) return run(act == SB_ACT_SILU ? run_slope<BtWide, SB_ACT_SILU> : run_slope<BtWide, SB_ACT_GELU>);
  return run(act == SB_ACT_SILU ? run_slope<BtNarrow, SB_ACT_SILU> : run_slope<BtNarrow, SB_ACT_GELU>);
}

int launch_rows_bt(const void* a, const void* b, const GatedLayout& layout, void* out, int64_t num_copies, int64_t n,
                   int64_t k, hipStream_t stream) {
  int width = 0;
  if (const int rc = bt_width(layout, num_copies, n, &width)) return rc;
  return width == 256 ? run_rows_bt<BtWide>(a, b, layout, out, n, k, stream)
                      : run_rows_bt<BtNarrow>(a, b, layout, out, n, k, stream);
}

int launch_expert_outer(const void* a, const void* b, const GatedLayout& layout, void* out, int64_t m, int64_t n,
                        hipStream_t stream) {
  return n % 256 == 0 ? run_outer<OuterWide>(a, b, layout, out, m, n, stream)
                      : run_outer<OuterNarrow>(a, b, layout, out, m, n, stream);
}

}  // namespace sb
