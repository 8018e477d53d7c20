// The backward pass of the gated experts on a routing layout, P padded rows:
//
//   grad_rows     grad_gates[t, j] = <grad_out[t], y[r]>, and x's and
//                 grad_out's rows gathered by padded row (xg, gog [P, D])
//   gated_slope   dH = w[r] gog W2[e]^T;  dG = dH U a'(G), dU = dH a(G)
//                 (grad_gu [P, 2F]), and wh = w[r] a(G) U (bf16, one rounding)
//   rows_bt       dXr = [dG | dU] W1[e]^T
//   outers        dW1[e] = xg^T [dG | dU],  dW2[e] = wh^T gog over e's rows
//
// and dx[t] = sum over t's rows of dXr (combine.hip). The products run on the
// LDS-DMA main loop: rows_bt and gated_slope with B's columns as rows (BT:
// W1 and W2 are read as they are stored), the outer products (gated_outer.hip)
// with both operands along K (AT). Rows past an expert's real rows are read as zeros (past the
// buffer's end) and not written.
//
// Gathering x and grad_out once (2 P D values, a few percent of the weights'
// bytes) lets the outer products' loads be plain: its K runs over rows, so a
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

// One lane per expert: its place among the experts by rows, most first
// (expert_order, which the weight gradients' tiles follow). Then one wave per
// padded row, then one lane per copy for those without a row (gradient 0). The
// row's copy is the one of its token's k that sits in it. Bound by memory: reads
// x, grad_out and y, writes xg and gog, 16 bytes a lane (16380 rows of D = 2048 57
// us, 5.9 TB/s).
template <typename G>
__global__ void __launch_bounds__(256)
    grad_rows_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ grad_out,
                     const uint16_t* __restrict__ y, GatedLayout layout, const int32_t* __restrict__ copy_row,
                     const G* __restrict__ gates, G* __restrict__ grad_gates, float* __restrict__ row_gate,
                     uint16_t* __restrict__ xg, uint16_t* __restrict__ gog, int64_t num_tokens, int32_t k,
                     int32_t d_model, int32_t row_groups, int32_t* __restrict__ expert_order,
                     const int32_t* __restrict__ valid_tokens) {
  const int32_t order_groups = (layout.num_experts + 255) / 256;
  if (static_cast<int32_t>(blockIdx.x) < order_groups) {
    const int32_t e = static_cast<int32_t>(blockIdx.x) * 256 + threadIdx.x;
    if (e >= layout.num_experts) return;
    const int32_t mine = layout.tokens_per_expert[e];
    int32_t place = 0;
#pragma unroll 8
    for (int32_t i = 0; i < layout.num_experts; ++i) {
      const int32_t n = scalar_load(layout.tokens_per_expert + i);
      place += n > mine || (n == mine && i < e) ? 1 : 0;
    }
    expert_order[place] = e;
    return;
  }
  const int32_t group = static_cast<int32_t>(blockIdx.x) - order_groups;
  if (group >= row_groups) {
    const int64_t c = (static_cast<int64_t>(group) - row_groups) * 256 + threadIdx.x;
    const int64_t limit = valid_tokens ? min(num_tokens, static_cast<int64_t>(*valid_tokens)) : num_tokens;
    if (c < limit * k && copy_row[c] < 0) store_gate(grad_gates, c, 0.0f);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int32_t r = uniform(group * 4 + static_cast<int>(threadIdx.x >> 6));
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
                  int64_t num_tokens, int32_t k, int64_t d_model, int32_t* expert_order, const int32_t* valid_tokens,
                  hipStream_t stream) {
  const int32_t row_groups = layout.max_row_blocks * (kBS / 4);
  const int64_t groups = (layout.num_experts + 255) / 256 + row_groups + (num_tokens * k + 255) / 256;
  grad_rows_kernel<G><<<static_cast<uint32_t>(groups), 256, 0, stream>>>(
      static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(grad_out), static_cast<const uint16_t*>(y), layout,
      copy_row, static_cast<const G*>(gates), static_cast<G*>(grad_gates), row_gate, static_cast<uint16_t*>(xg),
      static_cast<uint16_t*>(gog), num_tokens, k, static_cast<int32_t>(d_model), row_groups, expert_order,
      valid_tokens);
  return check_launch("gated backward: rows");
}

// ------------------------------------------------- products with W^T ---

// A: rows row0 .. of a [P, K] (rows past `rows` read as zeros); B: rows n0 ..
// of b[e] [N, K] (past N: zeros). Both advance BK * 2 bytes a K step.
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
  // The reduction starts at column k0 of the k.
  __device__ __forceinline__ RowsBtSrc(const uint16_t* a, const uint16_t* b, const Chunk& ch, int32_t n0, int32_t n,
                                       int32_t k, int32_t k0) {
    ra = make_rsrc(a + static_cast<int64_t>(ch.row0) * k + k0, (static_cast<uint32_t>(ch.rows) * k - k0) * 2u);
    rb = make_rsrc(b + static_cast<int64_t>(ch.expert) * n * k + k0,
                   (static_cast<uint32_t>(n) * static_cast<uint32_t>(k) - k0) * 2u);
    const ADmaPos<Cfg> ap;
#pragma unroll
    for (int q = 0; q < Cfg::kAInstr; ++q)
      a_off[q] = ap.row[q] < ch.rows ? (static_cast<uint32_t>(ap.row[q]) * k + ap.chunk[q] * 8) * 2u : kOutOfRange;
    const BtDmaPos<Cfg> bp;
#pragma unroll
    for (int q = 0; q < Cfg::kBInstr; ++q)
      b_off[q] = (static_cast<uint32_t>(n0 + bp.row[q]) * k + bp.chunk[q] * 8) * 2u;
  }
};

struct RowsBtArgs {
  const uint16_t *a, *b;
  GatedLayout layout;
  uint16_t* out;
  SplitOut split;
  int32_t n, k;
};

template <class Cfg, bool kSplit>
__device__ __forceinline__ void rows_bt_tile(uint8_t* __restrict__ lds, const RowsBtArgs& p, const Chunk& ch, int n0,
                                             int part) {
  using ML = DmaMainloop<Cfg>;
  const int k0 = kSplit ? split_start(part, p.split.parts, p.k / kBS) * kBS : 0;
  const int k1 = kSplit ? split_start(part + 1, p.split.parts, p.k / kBS) * kBS : p.k;
  const RowsBtSrc<Cfg> src(p.a, p.b, ch, n0, p.n, p.k, k0);
  typename ML::Acc acc;
  ML::run(lds, src, (k1 - k0) / Cfg::BK, acc);
  if constexpr (kSplit) {
    store_part<Cfg>(p.split, acc, part, p.layout, ch, n0, p.n);
  } else {
    ML::stage_tile(lds, acc, [](float v) { return v; });
    uint16_t* rows = p.out + static_cast<int64_t>(ch.row0) * p.n + n0;
    ML::for_each_staged_chunk(lds, [&](int r, int col, u32x4_t v) {
      if (r < ch.rows && n0 + col < p.n) *reinterpret_cast<u32x4_t*>(rows + static_cast<int64_t>(r) * p.n + col) = v;
    });
  }
}

struct SlopeArgs {
  const uint16_t *gog, *w2, *gu;
  const float* row_gate;
  GatedLayout layout;
  uint16_t *grad_gu, *wh;
  int32_t d_model, ffn_dim;
};

// The epilogue stages the tile as fp32, up to 128 rows at a time (a lane's
// results are 4 columns of 32 rows), then each lane takes 8 columns of a row:
// 16-byte loads of G and U, 16-byte stores of dG, dU and wh.
template <class Cfg, int ACT>
__device__ __forceinline__ void gated_slope_tile(uint8_t* __restrict__ lds, const SlopeArgs& p, const Chunk& ch,
                                                 int n0) {
  using ML = DmaMainloop<Cfg>;
  constexpr int BN = Cfg::BN, kRowBytes = BN * 4;
  // Row groups of a wave in one part, and the part's rows: Cfg::WM runs of them.
  constexpr int kGroups = 4 / Cfg::WM < Cfg::TM ? 4 / Cfg::WM : Cfg::TM;
  constexpr int kParts = (Cfg::TM + kGroups - 1) / kGroups;
  const RowsBtSrc<Cfg> src(p.gog, p.w2, ch, n0, p.ffn_dim, p.d_model, 0);
  typename ML::Acc acc;
  ML::run(lds, src, p.d_model / Cfg::BK, acc);

  const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) / Cfg::WN;
  static_for<0, kParts>([&](auto pc) {
    constexpr int i0 = decltype(pc)::value * kGroups;
    constexpr int kRun = 32 * (Cfg::TM - i0 < kGroups ? Cfg::TM - i0 : kGroups);  // rows of each wave row in this part
    __syncthreads();  // every wave is done reading the ring, or the part before
#pragma unroll
    for (int jn = 0; jn < Cfg::TN; ++jn)
#pragma unroll
      for (int i = i0; i < i0 + kRun / 32; ++i) {
        const int m = wm * kRun + 32 * (i - i0) + (lane & 31);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4_t v = {acc[jn][i][4 * g], acc[jn][i][4 * g + 1], acc[jn][i][4 * g + 2], acc[jn][i][4 * g + 3]};
          *reinterpret_cast<f32x4_t*>(lds + staged_at<kRowBytes>(m, ML::out_col(jn, g) >> 2)) = v;
        }
      }
    __syncthreads();
    constexpr int kChunksPerRow = BN / 8;
    for (int q = threadIdx.x; q < Cfg::WM * kRun * kChunksPerRow; q += Cfg::kThreads) {
      const int m = q / kChunksPerRow, c = q % kChunksPerRow;
      const int r = m / kRun * Cfg::WTM + 32 * i0 + m % kRun;  // of the chunk
      if (r >= ch.rows || n0 + c * 8 >= p.ffn_dim) continue;
      const int64_t row = ch.row0 + r;
      const int64_t at = row * 2 * p.ffn_dim + n0 + c * 8;
      const u32x4_t gv = *reinterpret_cast<const u32x4_t*>(p.gu + at);
      const u32x4_t uv = *reinterpret_cast<const u32x4_t*>(p.gu + at + p.ffn_dim);
      const float w = p.row_gate[row];
      const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(lds + staged_at<kRowBytes>(m, 2 * c));
      const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(lds + staged_at<kRowBytes>(m, 2 * c + 1));
      u32x4_t dg, du, hw;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        float og[2], ou[2], oh[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float g = __uint_as_float(e ? gv[h] & 0xffff0000u : gv[h] << 16);
          const float u = __uint_as_float(e ? uv[h] & 0xffff0000u : uv[h] << 16);
          const float dh = w * (h < 2 ? lo[2 * h + e] : hi[2 * h - 4 + e]);
          const ActSlope a = gated_act_slope<ACT>(g);
          og[e] = dh * u * a.slope;
          ou[e] = dh * a.value;
          oh[e] = w * (a.value * u);
        }
        dg[h] = pack_bf16x2(og[0], og[1]);
        du[h] = pack_bf16x2(ou[0], ou[1]);
        hw[h] = pack_bf16x2(oh[0], oh[1]);
      }
      *reinterpret_cast<u32x4_t*>(p.grad_gu + at) = dg;
      *reinterpret_cast<u32x4_t*>(p.grad_gu + at + p.ffn_dim) = du;
      *reinterpret_cast<u32x4_t*>(p.wh + row * p.ffn_dim + n0 + c * 8) = hw;
    }
  });
}

// Both products' row-block form: 128 x 128 tiles.
using BtNarrow = DmaCfg<128, 128, 64, 3, 2, 2, 0, 0, 5, 1, 0, 0, 0, 0, 1>;

template <int BN>
constexpr int slope_lds(int ring) { return ring > kBS * BN * 4 ? ring : kBS * BN * 4; }

template <bool kSplit>
__global__ void __launch_bounds__(BtNarrow::kThreads) rows_bt_kernel(RowsBtArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[BtNarrow::kLdsAlloc];
  Chunk ch;
  int slice, part = 0, tile = static_cast<int>(blockIdx.x);
  if constexpr (kSplit) split_tile(p.split, &tile, &part);
  if (!row_block_tile(tile, p.n / BtNarrow::BN, p.layout, &ch, &slice)) return;
  rows_bt_tile<BtNarrow, kSplit>(lds, p, ch, slice * BtNarrow::BN, part);
}

template <bool kSplit>
__global__ void __launch_bounds__(512) rows_bt_chunk_kernel(RowsBtArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[160 * 1024];
  Chunk ch{-1, 0, 0, 0};
  int slice = 0, part = 0, tile = static_cast<int>(blockIdx.x);
  if constexpr (kSplit) split_tile(p.split, &tile, &part);
  if (!gated_chunk_tile(tile, gated_slices(p.n), p.layout, &ch, &slice)) return;
  with_chunk_groups(ch.groups, [&](auto rc) {
    using Cfg = BtChunkCfg<decltype(rc)::value>;
    static_assert(Cfg::kLdsAlloc <= sizeof(lds) && Cfg::kThreads == 512, "one workgroup for all heights");
    rows_bt_tile<Cfg, kSplit>(lds, p, ch, slice * kGatedBN, part);
  });
}

template <int ACT>
__global__ void __launch_bounds__(BtNarrow::kThreads) gated_slope_kernel(SlopeArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[slope_lds<BtNarrow::BN>(BtNarrow::kLdsAlloc)];
  Chunk ch;
  int slice;
  if (!row_block_tile(static_cast<int>(blockIdx.x), p.ffn_dim / BtNarrow::BN, p.layout, &ch, &slice)) return;
  gated_slope_tile<BtNarrow, ACT>(lds, p, ch, slice * BtNarrow::BN);
}

template <int ACT>
__global__ void __launch_bounds__(512) gated_slope_chunk_kernel(SlopeArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[160 * 1024];
  Chunk ch{-1, 0, 0, 0};
  int slice = 0;
  if (!gated_chunk_tile(static_cast<int>(blockIdx.x), gated_slices(p.ffn_dim), p.layout, &ch, &slice)) return;
  with_chunk_groups(ch.groups, [&](auto rc) {
    using Cfg = BtChunkCfg<decltype(rc)::value>;
    static_assert(Cfg::kLdsAlloc <= sizeof(lds) && Cfg::kThreads == 512, "one workgroup for all heights");
    gated_slope_tile<Cfg, ACT>(lds, p, ch, slice * kGatedBN);
  });
}

// A product's launch in its form.
template <class Args>
int launch_bt(void (*row_blocks)(Args), void (*chunk_form)(Args), const Args& args, const GatedForm& form, int64_t k,
              hipStream_t stream) {
  if (!reduction_fits<BtNarrow>(k) || !reduction_fits<BtChunkCfg<kGatedRmax>>(k))
    return fail(SB_ERR_INVALID, "gated backward: not whole K steps");
  if (form.grid > 2147483647LL) return fail(SB_ERR_INVALID, "problem too large");
  if (form.chunks) chunk_form<<<static_cast<uint32_t>(form.grid), 512, 0, stream>>>(args);
  else row_blocks<<<static_cast<uint32_t>(form.grid), BtNarrow::kThreads, 0, stream>>>(args);
  return check_launch("gated backward");
}

}  // namespace

int launch_grad_rows(const void* x, const void* grad_out, const void* y, const GatedLayout& layout,
                     const int32_t* copy_row, const void* gates, int32_t gate_dtype, void* grad_gates, float* row_gate,
                     void* xg, void* gog, int64_t num_tokens, int32_t k, int64_t d_model, int32_t* expert_order,
                     const int32_t* valid_tokens, hipStream_t stream) {
  auto run = [&](auto tag) {
    return run_grad_rows<decltype(tag)>(x, grad_out, y, layout, copy_row, gates, grad_gates, row_gate, xg, gog,
                                        num_tokens, k, d_model, expert_order, valid_tokens, stream);
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
  const SlopeArgs args{static_cast<const uint16_t*>(gog), static_cast<const uint16_t*>(w2),
                       static_cast<const uint16_t*>(gu), row_gate, layout, static_cast<uint16_t*>(grad_gu),
                       static_cast<uint16_t*>(wh), static_cast<int32_t>(d_model), static_cast<int32_t>(ffn_dim)};
  // dG and dU are products with the whole sum: not split.
  const GatedForm form = gated_form(layout.max_row_blocks, layout.num_experts, num_copies, ffn_dim, d_model, false);
  return act == SB_ACT_SILU ? launch_bt(gated_slope_kernel<SB_ACT_SILU>, gated_slope_chunk_kernel<SB_ACT_SILU>, args,
                                        form, d_model, stream)
                            : launch_bt(gated_slope_kernel<SB_ACT_GELU>, gated_slope_chunk_kernel<SB_ACT_GELU>, args,
                                        form, d_model, stream);
}

int launch_rows_bt(const void* a, const void* b, const GatedLayout& layout, void* out, float* partial,
                   int64_t num_copies, int64_t n, int64_t k, hipStream_t stream) {
  const GatedForm form = gated_form(layout.max_row_blocks, layout.num_experts, num_copies, n, k, true);
  const RowsBtArgs args{static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(b), layout,
                        static_cast<uint16_t*>(out), split_out(form, partial), static_cast<int32_t>(n),
                        static_cast<int32_t>(k)};
  if (form.parts == 1) return launch_bt(rows_bt_kernel<false>, rows_bt_chunk_kernel<false>, args, form, k, stream);
  if (const int rc = launch_bt(rows_bt_kernel<true>, rows_bt_chunk_kernel<true>, args, form, kBS, stream)) return rc;
  return launch_join_parts(partial, layout, out, form.parts, n, stream);
}

}  // namespace sb
