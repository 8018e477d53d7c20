// The gated experts' first product on a routing layout:
//
//   G | U = x[row_token] [P, D] @ W1[e] [D, 2F],   H = a(G) U
//
// One workgroup computes 128 rows x BN columns of one row block on the
// LDS-DMA main loop: BN / 2 gate columns and the same BN / 2 up columns, in
// one B tile (its columns from n0 and from F + n0 of W1[e]). A wave's blocks
// of 32 columns alternate between the two (GATED, gemm_dma.hpp), so a lane
// holds G and U of the same elements and H is formed from its fp32
// accumulators, rounded once. x's rows are gathered by the loads themselves
// (SddDmaSrc), padding rows read as zeros without a read of memory.
// With `gu` the tile's G | U are written too (bf16: what the backward pass
// reads; the products' operands are bf16 and so is its own next product).

#include "gated.hpp"
#include "gated_act.hpp"
#include "sdd_tile.hpp"

namespace sb {
namespace {

template <class Cfg, bool kWideX, bool kKeep, int ACT>
__global__ void __launch_bounds__(Cfg::kThreads)
    gated_up_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ w1, GatedLayout layout,
                    uint16_t* __restrict__ h, uint16_t* __restrict__ gu, int32_t num_tokens, int32_t d_model,
                    int32_t ffn_dim) {
  using ML = DmaMainloop<Cfg>;
  constexpr int kHalf = Cfg::BN / 2;  // columns of F
  static_assert(Cfg::BM == kBS && Cfg::GATED && Cfg::EPI_PARTS == 1, "one row block per tile");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsAlloc];
  const int slices = ffn_dim / kHalf;
  RowBlock b;
  int slice;
  if (!row_block_tile(static_cast<int>(blockIdx.x), slices, layout, kTileGroup, &b, &slice)) return;
  const int n0 = slice * kHalf;

  SddDmaSrc<Cfg, kWideX> src;
  src.x_rsrc = make_rsrc(x, kWideX ? 0u : static_cast<uint32_t>(num_tokens) * static_cast<uint32_t>(d_model) * 2u);
  src.w_rsrc = make_rsrc(w1 + static_cast<int64_t>(b.expert) * d_model * (2 * static_cast<int64_t>(ffn_dim)),
                         static_cast<uint32_t>(d_model) * static_cast<uint32_t>(ffn_dim) * 4u);
  src.b_step_bytes = static_cast<uint32_t>(Cfg::BK) * static_cast<uint32_t>(ffn_dim) * 4u;
  const ADmaPos<Cfg> ap;
#pragma unroll
  for (int q = 0; q < Cfg::kAInstr; ++q) {
    const int32_t tok = ap.row[q] < b.rows ? layout.row_token[b.row0 + ap.row[q]] : -1;
    src.set_row(q, tok < num_tokens ? tok : -1, ap.chunk[q], x, d_model);
  }
  const BDmaPos<Cfg> bp;
#pragma unroll
  for (int q = 0; q < Cfg::kBInstr; ++q) {
    const int col = bp.col[q] < kHalf ? n0 + bp.col[q] : ffn_dim + n0 + bp.col[q] - kHalf;
    src.b_off[q] = (static_cast<uint32_t>(bp.row[q]) * (2 * ffn_dim) + col) * 2u;
  }

  typename ML::Acc acc;
  ML::run(lds, src, d_model / Cfg::BK, acc);

  // Staged as bf16 rows of kHalf columns: G, then U below it, then (over
  // both) H; each written row by row in 16-byte chunks.
  const int lane = threadIdx.x & 63, wn = (threadIdx.x >> 6) % Cfg::WN;
  constexpr int kRowBytes = kHalf * 2;
  auto stage = [&](int base, auto value) {
#pragma unroll
    for (int j = 0; j < Cfg::TN / 2; ++j)
#pragma unroll
      for (int i = 0; i < Cfg::TM; ++i) {
        const int m = ML::out_row(i);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int n = 32 * (wn * (Cfg::TN / 2) + j) + 8 * g + 4 * (lane >> 5);
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = value(acc[2 * j][i][4 * g + e], acc[2 * j + 1][i][4 * g + e]);
          *reinterpret_cast<u32x2_t*>(lds + base + staged_at<kRowBytes>(m, n >> 3) + (n & 7) * 2) =
              u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        }
      }
  };
  constexpr int kChunksPerRow = kHalf / 8;
  auto write = [&](int base, auto to) {
    for (int q = threadIdx.x; q < b.rows * kChunksPerRow; q += Cfg::kThreads) {
      const int r = q / kChunksPerRow, c = q % kChunksPerRow;
      *reinterpret_cast<u32x4_t*>(to(r, c * 8)) =
          *reinterpret_cast<const u32x4_t*>(lds + base + staged_at<kRowBytes>(r, c));
    }
  };
  __syncthreads();  // every wave is done reading the ring
  if constexpr (kKeep) {
    constexpr int kUp = kBS * kRowBytes;
    stage(0, [](float g, float) { return g; });
    stage(kUp, [](float, float u) { return u; });
    __syncthreads();
    uint16_t* rows = gu + static_cast<int64_t>(b.row0) * 2 * ffn_dim + n0;
    write(0, [&](int r, int col) { return rows + static_cast<int64_t>(r) * 2 * ffn_dim + col; });
    write(kUp, [&](int r, int col) { return rows + static_cast<int64_t>(r) * 2 * ffn_dim + ffn_dim + col; });
    __syncthreads();
  }
  stage(0, [](float g, float u) { return gated_act<ACT>(g) * u; });
  __syncthreads();
  uint16_t* blocks = h + static_cast<int64_t>(b.row0) * ffn_dim;  // the row block's first BSR block
  write(0, [&](int r, int col) {
    const int f = n0 + col;
    return blocks + static_cast<int64_t>(f / kBS) * kBS * kBS + r * kBS + f % kBS;
  });
}

// The per-row-block SDD's tile shapes, gated: 512 columns (256 of F), and 256
// and 128 where F or the number of tiles asks for narrower ones.
using GatedWide = DmaCfg<128, 512, 32, 3, 2, 4, 0, 2, 3, 1, 1, 0, 0, 0, 0, 1>;
using GatedMid = DmaCfg<128, 256, 64, 3, 2, 4, 0, 2, 3, 1, 0, 0, 0, 0, 0, 1>;
using GatedNarrow = DmaCfg<128, 128, 64, 3, 2, 2, 0, 2, 5, 1, 0, 0, 0, 0, 0, 1>;

struct UpArgs {
  const void *x, *w1;
  GatedLayout layout;
  void *h, *gu;
  int64_t num_tokens, d_model, ffn_dim;
  hipStream_t stream;
};

template <class Cfg, bool kWideX, bool kKeep, int ACT>
int launch_up(const UpArgs& a) {
  if (!reduction_fits<Cfg>(a.d_model)) return fail(SB_ERR_INVALID, "gated experts: D is not whole K steps");
  const int64_t tiles = a.layout.max_row_blocks * (a.ffn_dim / (Cfg::BN / 2));
  if (tiles > 2147483647LL) return fail(SB_ERR_INVALID, "gated experts: too many tiles");
  gated_up_kernel<Cfg, kWideX, kKeep, ACT><<<static_cast<uint32_t>(tiles), Cfg::kThreads, 0, a.stream>>>(
      static_cast<const uint16_t*>(a.x), static_cast<const uint16_t*>(a.w1), a.layout, static_cast<uint16_t*>(a.h),
      static_cast<uint16_t*>(a.gu), static_cast<int32_t>(a.num_tokens), static_cast<int32_t>(a.d_model),
      static_cast<int32_t>(a.ffn_dim));
  return check_launch("gated experts");
}

template <bool kWideX, bool kKeep, int ACT>
int launch_up_width(const UpArgs& a, int width) {
  switch (width) {
    case 512: return launch_up<GatedWide, kWideX, kKeep, ACT>(a);
    case 256: return launch_up<GatedMid, kWideX, kKeep, ACT>(a);
    default: return launch_up<GatedNarrow, kWideX, kKeep, ACT>(a);
  }
}

template <bool kWideX, bool kKeep>
int launch_up_act(const UpArgs& a, int width, int32_t act) {
  return act == SB_ACT_SILU ? launch_up_width<kWideX, kKeep, SB_ACT_SILU>(a, width)
                            : launch_up_width<kWideX, kKeep, SB_ACT_GELU>(a, width);
}

}  // namespace

int launch_gated_up(const void* x, const void* w1, const GatedLayout& layout, void* h, void* gu, int64_t num_tokens,
                    int64_t num_copies, int64_t d_model, int64_t ffn_dim, int32_t act, hipStream_t stream) {
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  const UpArgs a{x, w1, layout, h, gu, num_tokens, d_model, ffn_dim, stream};
  // Each live row block holds a copy at least.
  const int width = fit_width(std::min<int64_t>(layout.max_row_blocks, num_copies), 2 * ffn_dim, cus);
  if (sdd_wide_x(num_tokens, d_model))
    return gu ? launch_up_act<true, true>(a, width, act) : launch_up_act<true, false>(a, width, act);
  return gu ? launch_up_act<false, true>(a, width, act) : launch_up_act<false, false>(a, width, act);
}

}  // namespace sb
