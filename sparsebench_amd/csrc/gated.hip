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

struct UpArgs {
  const uint16_t *x, *w1;
  GatedLayout layout;
  uint16_t *h, *gu;
  int32_t num_tokens, d_model, ffn_dim;
};

// Rows ch of H and (kKeep) G | U, their columns n0 .. n0 + BN / 2 of F. LDS: bytes of lds.
template <class Cfg, bool kWideX, bool kKeep, int ACT, int LDS>
__device__ __forceinline__ void gated_up_tile(uint8_t* __restrict__ lds, const UpArgs& a, const Chunk& ch, int n0) {
  using ML = DmaMainloop<Cfg>;
  constexpr int kHalf = Cfg::BN / 2;
  static_assert(Cfg::GATED && Cfg::EPI_PARTS == 1, "gated tiles");
  SddDmaSrc<Cfg, kWideX> src;
  src.x_rsrc =
      make_rsrc(a.x, kWideX ? 0u : static_cast<uint32_t>(a.num_tokens) * static_cast<uint32_t>(a.d_model) * 2u);
  src.w_rsrc = make_rsrc(a.w1 + static_cast<int64_t>(ch.expert) * a.d_model * (2 * static_cast<int64_t>(a.ffn_dim)),
                         static_cast<uint32_t>(a.d_model) * static_cast<uint32_t>(a.ffn_dim) * 4u);
  src.b_step_bytes = static_cast<uint32_t>(Cfg::BK) * static_cast<uint32_t>(a.ffn_dim) * 4u;
  const ADmaPos<Cfg> ap;
#pragma unroll
  for (int q = 0; q < Cfg::kAInstr; ++q) {
    const int32_t tok = ap.row[q] < ch.rows ? a.layout.row_token[ch.row0 + ap.row[q]] : -1;
    src.set_row(q, tok < a.num_tokens ? tok : -1, ap.chunk[q], a.x, a.d_model);
  }
  const BDmaPos<Cfg> bp;
#pragma unroll
  for (int q = 0; q < Cfg::kBInstr; ++q) {
    const int col = bp.col[q] < kHalf ? n0 + bp.col[q] : a.ffn_dim + n0 + bp.col[q] - kHalf;
    src.b_off[q] = (static_cast<uint32_t>(bp.row[q]) * (2 * a.ffn_dim) + col) * 2u;
  }

  typename ML::Acc acc;
  ML::run(lds, src, a.d_model / Cfg::BK, acc);

  // Staged as bf16 rows of kHalf columns, G, U below it, H below both if they
  // fit in LDS bytes; each written row by row in 16-byte chunks.
  const int lane = threadIdx.x & 63, wn = (threadIdx.x >> 6) % Cfg::WN;
  constexpr int kRowBytes = kHalf * 2;
  auto stage = [&](int base, auto value) {
    if (!ML::computes()) return;
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
    for (int q = threadIdx.x; q < ch.rows * kChunksPerRow; q += Cfg::kThreads) {
      const int r = q / kChunksPerRow, c = q % kChunksPerRow;
      *reinterpret_cast<u32x4_t*>(to(r, c * 8)) =
          *reinterpret_cast<const u32x4_t*>(lds + base + staged_at<kRowBytes>(r, c));
    }
  };
  constexpr int kUp = Cfg::BM * kRowBytes;
  constexpr int kH = 3 * kUp <= LDS ? 2 * kUp : 0;  // H over G where the three do not fit
  auto product = [](float g, float u) { return gated_act<ACT>(g) * u; };
  __syncthreads();  // every wave is done reading the ring
  if constexpr (kKeep) {
    stage(0, [](float g, float) { return g; });
    stage(kUp, [](float, float u) { return u; });
    if constexpr (kH != 0) stage(kH, product);
    __syncthreads();
    uint16_t* rows = a.gu + static_cast<int64_t>(ch.row0) * 2 * a.ffn_dim + n0;
    write(0, [&](int r, int col) { return rows + static_cast<int64_t>(r) * 2 * a.ffn_dim + col; });
    write(kUp, [&](int r, int col) { return rows + static_cast<int64_t>(r) * 2 * a.ffn_dim + a.ffn_dim + col; });
    if constexpr (kH == 0) __syncthreads();
  }
  if constexpr (!kKeep || kH == 0) {
    stage(kH, product);
    __syncthreads();
  }
  uint16_t* blocks = a.h + static_cast<int64_t>(ch.row0) * a.ffn_dim;  // the first row block's first BSR block
  write(kH, [&](int r, int col) {
    const int f = n0 + col;
    return blocks + static_cast<int64_t>(r / kBS) * kBS * a.ffn_dim + static_cast<int64_t>(f / kBS) * kBS * kBS +
           (r % kBS) * kBS + f % kBS;
  });
}

template <class Cfg, bool kWideX, bool kKeep, int ACT>
__global__ void __launch_bounds__(Cfg::kThreads) gated_up_kernel(UpArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsAlloc];
  Chunk ch;
  int slice;
  if (!row_block_tile(static_cast<int>(blockIdx.x), a.ffn_dim / (Cfg::BN / 2), a.layout, &ch, &slice)) return;
  gated_up_tile<Cfg, kWideX, kKeep, ACT, sizeof(lds)>(lds, a, ch, slice * (Cfg::BN / 2));
}

template <bool kKeep, int ACT>
__global__ void __launch_bounds__(512) gated_up_chunk_kernel(UpArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[GatedUpCfg<kGatedRmax>::kLdsAlloc];
  Chunk ch{-1, 0, 0, 0};
  int slice = 0;
  if (!gated_chunk_tile(static_cast<int>(blockIdx.x), a.ffn_dim / (kGatedBN / 2), a.layout, &ch, &slice)) return;
  with_chunk_groups(ch.groups, [&](auto rc) {
    using Cfg = GatedUpCfg<decltype(rc)::value>;
    static_assert(Cfg::kLdsAlloc <= sizeof(lds) && Cfg::kThreads == 512, "one workgroup for all heights");
    gated_up_tile<Cfg, false, kKeep, ACT, sizeof(lds)>(lds, a, ch, slice * (kGatedBN / 2));
  });
}

// Row-block tiles: 128 columns (64 of F), and 256 for x of 2 GiB or more,
// which the chunk form's 32-bit offsets do not reach.
using GatedNarrow = DmaCfg<128, 128, 64, 3, 2, 2, 0, 2, 5, 1, 0, 0, 0, 0, 0, 1>;
using GatedMid = DmaCfg<128, 256, 64, 3, 2, 4, 0, 2, 3, 1, 0, 0, 0, 0, 0, 1>;

template <class Cfg, bool kWideX, bool kKeep, int ACT>
int launch_up(const UpArgs& a, hipStream_t stream) {
  const int64_t tiles = int64_t{a.layout.max_row_blocks} * (a.ffn_dim / (Cfg::BN / 2));
  if (!reduction_fits<Cfg>(a.d_model) || tiles > 2147483647LL) return fail(SB_ERR_INVALID, "problem too large");
  gated_up_kernel<Cfg, kWideX, kKeep, ACT><<<static_cast<uint32_t>(tiles), Cfg::kThreads, 0, stream>>>(a);
  return check_launch("gated experts");
}

template <bool kKeep, int ACT>
int launch_up_form(const UpArgs& a, const GatedForm& form, hipStream_t stream) {
  if (sdd_wide_x(a.num_tokens, a.d_model)) return launch_up<GatedMid, true, kKeep, ACT>(a, stream);
  if (!form.chunks) return launch_up<GatedNarrow, false, kKeep, ACT>(a, stream);
  if (!reduction_fits<GatedUpCfg<kGatedRmax>>(a.d_model) || form.grid > 2147483647LL)
    return fail(SB_ERR_INVALID, "problem too large");
  gated_up_chunk_kernel<kKeep, ACT><<<static_cast<uint32_t>(form.grid), 512, 0, stream>>>(a);
  return check_launch("gated experts");
}

}  // namespace

int launch_gated_up(const void* x, const void* w1, const GatedLayout& layout, void* h, void* gu, int64_t num_tokens,
                    int64_t num_copies, int64_t d_model, int64_t ffn_dim, int32_t act, hipStream_t stream) {
  const UpArgs a{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(w1), layout,
                 static_cast<uint16_t*>(h), static_cast<uint16_t*>(gu), static_cast<int32_t>(num_tokens),
                 static_cast<int32_t>(d_model), static_cast<int32_t>(ffn_dim)};
  // H is a product of two sums: not split.
  const GatedForm form = gated_form(layout.max_row_blocks, layout.num_experts, num_copies, 2 * ffn_dim, d_model, false);
  if (gu)
    return act == SB_ACT_SILU ? launch_up_form<true, SB_ACT_SILU>(a, form, stream)
                              : launch_up_form<true, SB_ACT_GELU>(a, form, stream);
  return act == SB_ACT_SILU ? launch_up_form<false, SB_ACT_SILU>(a, form, stream)
                            : launch_up_form<false, SB_ACT_GELU>(a, form, stream);
}

}  // namespace sb
