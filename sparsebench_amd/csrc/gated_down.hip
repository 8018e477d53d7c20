// The gated experts' second product, y = H W2[e], where the layer's own
// kernel (experts.hip) does not take the shape or leaves most CUs idle, and the
// sum that ends a product whose reduction is split over workgroups.
//
// A tile reduces over all of F. Few rows and a narrow output make few tiles: 18
// tokens of 3 copies, E = 3, D = 384, F = 6400 are 9 tiles of 128 columns, whose
// 1.6 MB of weights one CU each reads in 61 us. Split in parts of F, each adds
// up its part in fp32 into rows of its own (partial [splits, P, D]), and one
// more pass adds the parts in order (no atomics: the same bits every time).

#include "chunk_tiles.hpp"
#include "gated.hpp"

namespace sb {
namespace {

struct DownArgs {
  const uint16_t *h, *w2;
  GatedLayout layout;
  uint16_t* out;
  SplitOut split;
  int32_t ffn_dim, d_model;
};

template <class Cfg, bool kSplit>
__device__ __forceinline__ void gated_down_tile(uint8_t* __restrict__ lds, const DownArgs& p, const Chunk& ch, int n0,
                                                int part) {
  using ML = DmaMainloop<Cfg>;
  // The part's columns of F: whole blocks of H.
  const int blocks = p.ffn_dim / kBS;
  const int first = kSplit ? split_start(part, p.split.parts, blocks) : 0;
  const int last = kSplit ? split_start(part + 1, p.split.parts, blocks) : blocks;
  const uint32_t block_bytes = kBS * kBS * 2;
  DsdChunkSrc<Cfg> src;
  src.h_rsrc = make_rsrc(p.h + static_cast<int64_t>(ch.row0) * p.ffn_dim + static_cast<int64_t>(first) * kBS * kBS,
                         static_cast<uint32_t>((ch.rows + kBS - 1) / kBS * blocks - first) * block_bytes);
  src.h_base = 0;
  src.w_rsrc = make_rsrc(p.w2 + (static_cast<int64_t>(ch.expert) * p.ffn_dim + first * kBS) * p.d_model,
                         static_cast<uint32_t>(p.ffn_dim - first * kBS) * static_cast<uint32_t>(p.d_model) * 2u);
  src.w_step_bytes = static_cast<uint32_t>(Cfg::BK) * static_cast<uint32_t>(p.d_model) * 2u;
  src.n0_bytes = 0;
  const ADmaPos<Cfg> ap;
#pragma unroll
  for (int q = 0; q < Cfg::kAInstr; ++q) {
    const uint32_t j = static_cast<uint32_t>(ap.row[q]);
    src.a_off[q] = static_cast<int>(j) < ch.rows
                       ? (j / kBS) * blocks * block_bytes + (j % kBS) * (kBS * 2) + ap.chunk[q] * 16u
                       : kOutOfRange;
  }
  const BDmaPos<Cfg> bp;
#pragma unroll
  for (int q = 0; q < Cfg::kBInstr; ++q)
    src.b_off[q] = n0 + bp.col[q] < p.d_model ? (static_cast<uint32_t>(bp.row[q]) * p.d_model + n0 + bp.col[q]) * 2u
                                              : kOutOfRange;

  typename ML::Acc acc;
  ML::run(lds, src, (last - first) * (kBS / Cfg::BK), acc);
  if constexpr (kSplit) {
    store_part<Cfg>(p.split, acc, part, p.layout, ch, n0, p.d_model);
  } else {
    ML::stage_tile(lds, acc, [](float v) { return v; });
    uint16_t* rows = p.out + static_cast<int64_t>(ch.row0) * p.d_model + n0;
    ML::for_each_staged_chunk(lds, [&](int r, int col, u32x4_t v) {
      if (r < ch.rows && n0 + col < p.d_model)
        *reinterpret_cast<u32x4_t*>(rows + static_cast<int64_t>(r) * p.d_model + col) = v;
    });
  }
}

using DownNarrow = DmaCfg<128, 128, 64, 3, 2, 2, 0, 2, 5, 1>;
template <int R>
using DownChunkCfg = DmaCfg<32 * R, kGatedBN, 32, 4, 2, 4, 0, 2, 5, 1, 1>;

template <bool kSplit>
__global__ void __launch_bounds__(DownNarrow::kThreads) gated_down_kernel(DownArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[DownNarrow::kLdsAlloc];
  Chunk ch;
  int slice, part = 0, tile = static_cast<int>(blockIdx.x);
  if constexpr (kSplit) split_tile(p.split, &tile, &part);
  if (!row_block_tile(tile, p.d_model / DownNarrow::BN, p.layout, &ch, &slice)) return;
  gated_down_tile<DownNarrow, kSplit>(lds, p, ch, slice * DownNarrow::BN, part);
}

template <bool kSplit>
__global__ void __launch_bounds__(512) gated_down_chunk_kernel(DownArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[DownChunkCfg<kGatedRmax>::kLdsAlloc];
  Chunk ch{-1, 0, 0, 0};
  int slice = 0, part = 0, tile = static_cast<int>(blockIdx.x);
  if constexpr (kSplit) split_tile(p.split, &tile, &part);
  if (!gated_chunk_tile(tile, gated_slices(p.d_model), p.layout, &ch, &slice)) return;
  with_chunk_groups(ch.groups, [&](auto rc) {
    using Cfg = DownChunkCfg<decltype(rc)::value>;
    static_assert(Cfg::kLdsAlloc <= sizeof(lds) && Cfg::kThreads == 512, "one workgroup for all heights");
    gated_down_tile<Cfg, kSplit>(lds, p, ch, slice * kGatedBN, part);
  });
}

// out[r] = the sum of row r's parts, in order; rows without a token are left.
// Rounded to bf16 as an unsplit product's rows are: the sum over a token's copies
// that follows reads the same rows either way. Bound by memory; 8 columns a lane.
__global__ void __launch_bounds__(256)
    join_parts_kernel(const float* __restrict__ partial, const int32_t* __restrict__ row_token,
                      uint16_t* __restrict__ out, int64_t rows, int32_t chunks_per_row, int32_t parts) {
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t r = item / chunks_per_row;
  if (r >= rows || row_token[r] < 0) return;
  f32x4_t lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
  for (int s = 0; s < parts; ++s) {
    const auto* from = reinterpret_cast<const f32x4_t*>(partial + (s * rows * chunks_per_row + item) * 8);
    lo += from[0];
    hi += from[1];
  }
  *reinterpret_cast<u32x4_t*>(out + item * 8) =
      u32x4_t{pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3])};
}

}  // namespace

int launch_gated_down(const void* h, const void* w2, const GatedLayout& layout, void* out, float* partial,
                      int64_t num_copies, int64_t d_model, int64_t ffn_dim, hipStream_t stream) {
  const GatedForm form = gated_form(layout.max_row_blocks, layout.num_experts, num_copies, d_model, ffn_dim, true);
  if (form.grid > 2147483647LL || !reduction_fits<DownNarrow>(kBS) || !reduction_fits<DownChunkCfg<kGatedRmax>>(kBS))
    return fail(SB_ERR_INVALID, "problem too large");
  const DownArgs args{static_cast<const uint16_t*>(h), static_cast<const uint16_t*>(w2), layout,
                      static_cast<uint16_t*>(out), split_out(form, partial), static_cast<int32_t>(ffn_dim),
                      static_cast<int32_t>(d_model)};
  auto run = [&](auto kernel, int threads) { kernel<<<static_cast<uint32_t>(form.grid), threads, 0, stream>>>(args); };
  if (form.chunks) form.parts > 1 ? run(gated_down_chunk_kernel<true>, 512) : run(gated_down_chunk_kernel<false>, 512);
  else form.parts > 1 ? run(gated_down_kernel<true>, DownNarrow::kThreads)
                      : run(gated_down_kernel<false>, DownNarrow::kThreads);
  if (const int rc = check_launch("gated experts: second product")) return rc;
  return form.parts > 1 ? launch_join_parts(partial, layout, out, form.parts, d_model, stream) : SB_OK;
}

int launch_join_parts(const float* partial, const GatedLayout& layout, void* out, int32_t parts, int64_t columns,
                      hipStream_t stream) {
  const int64_t rows = int64_t{layout.max_row_blocks} * kBS;
  join_parts_kernel<<<static_cast<uint32_t>((rows * (columns / 8) + 255) / 256), 256, 0, stream>>>(
      partial, layout.row_token, static_cast<uint16_t*>(out), rows, static_cast<int32_t>(columns / 8), parts);
  return check_launch("gated experts: sum of parts");
}

}  // namespace sb
