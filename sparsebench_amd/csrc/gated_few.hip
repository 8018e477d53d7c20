// The gated layer for one or two tokens (decode steps): each expert's weights
// are read for a row or two, so the time is the weights' bytes and the
// launches. No routing layout, no MFMA tiles (which would be padding for the
// most part):
//
//   few_up     gu[s][c] = the s-th part of D of x[t] [G | U][e]
//   few_down   part[s][c] = h[c] W2[e] over the s-th part of F,
//              h[c] = a(sum_s G) * (sum_s U)
//   few_out    out[t] = sum_j gates[t, j] sum_s part[s][t k + j]; with few
//              workgroups by the last of few_down's for each 128 columns
//
// A workgroup of few_up / few_down belongs to a copy c, and does the rows of
// all copies of its expert, if c is the first of them (a ballot over the ids);
// so an expert's weights are read once for both tokens. A lane owns 8 columns
// (16 bytes of a weight row) and 8 consecutive k at a time: 8 weight loads (16
// in few_up) are under way together, then 64 fused multiply-adds a row each.
// The lanes of a column then add up their sums, in an order that depends on the
// shape alone. fp32 throughout: the products are exact, h is not rounded.
//
// Bound by memory where the weights are large, by the launches where
// small. D and F are split among workgroups until they are about three a CU.
// Against the routed tiles (which win from three tokens on: 424 against 657 us
// for 8 tokens at D = 4096, F = 14336, E = 8, 50 against 49 for 4 at D = 1024, F =
// 4096, E = 64), k = 2, us a call:
//   one token   D = 256 F = 512 E = 8 13.6 (tiles 19.8), D = 1024 F = 4096 E = 64 24
//     (40), D = 2048 F = 768 E = 128 18 (35), D = 4096 F = 14336 E = 8 129 (142)
//   two tokens  12 (19), 31 (44), 19 (35), 212 (213)

#include "gated_act.hpp"
#include "gated.hpp"

namespace sb {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kStep = 8;  // k of a lane at a time
constexpr int kMaxUpSplits = 8, kMaxSplits = 16;
// few_down's workgroups up to which the last of them write out: a workgroup's
// write-back before its ticket takes 0.3 to 0.5 us, one after another in an XCD
// (256 of them 10 us, 1024 68), a launch more 2.4 us of the GPU and 2.7 of the host
// (D = 256, F = 512, one token, 16 workgroups: 13.6 us a call against 15.5).
constexpr uint32_t kTicketMost = 32;

struct FewArgs {
  const uint16_t *x, *w1, *w2;
  const void *expert_idx, *gates;
  const int32_t* valid_tokens;
  float *gu, *part;
  int32_t* tickets;  // one per 128 columns of out
  uint16_t* out;
  int32_t idx_is_i64, num_tokens, k, num_experts, d_model, ffn_dim, up_splits, splits, gate_dtype;
};

// The expert of copy c, or -1 for a copy that is not routed.
__device__ __forceinline__ int32_t expert_of(const FewArgs& a, int32_t c, int32_t limit) {
  if (c >= limit * a.k) return -1;
  const int64_t e = a.idx_is_i64 ? static_cast<const int64_t*>(a.expert_idx)[c]
                                 : static_cast<const int32_t*>(a.expert_idx)[c];
  return e >= 0 && e < a.num_experts ? static_cast<int32_t>(e) : -1;
}

__device__ __forceinline__ int32_t token_limit(const FewArgs& a) {
  return a.valid_tokens ? min(a.num_tokens, max(0, *a.valid_tokens)) : a.num_tokens;
}

// The copies (bits) of copy c's expert, 0 unless c is the first of them.
__device__ __forceinline__ uint64_t copies_with(const FewArgs& a, int32_t c, int32_t* expert) {
  const int32_t mine = expert_of(a, static_cast<int32_t>(threadIdx.x & 63), token_limit(a));
  *expert = __builtin_amdgcn_readlane(mine, c);
  const uint64_t all = __ballot(mine == *expert);
  return *expert >= 0 && __builtin_ctzll(all) == c ? all : 0;
}

// acc[r][e] += sum over k0 .. k0 + 7 of row r's values and the lane's 8 columns.
template <int RM>
__device__ __forceinline__ void multiply_add(float (&acc)[RM][8], const float (&v)[RM][kStep], const u32x4_t (&w)[kStep]) {
#pragma unroll
  for (int j = 0; j < kStep; ++j) {
    float f[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f[2 * q] = __uint_as_float(w[j][q] << 16);
      f[2 * q + 1] = __uint_as_float(w[j][q] & 0xffff0000u);
    }
#pragma unroll
    for (int r = 0; r < RM; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(v[r][j], f[e], acc[r][e]);
  }
}

// The sum over the lanes of a wave that own the same columns (its four rows of
// 16 lanes), in every lane.
constexpr int kLanes = 16, kColumns = 8 * kLanes, kGroups = kThreads / kLanes;
__device__ __forceinline__ float column_sum(float v) {
  // Rows 0 and 1, 2 and 3, then the halves of the wave, change places.
  const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  v = __int_as_float(rows[0]) + __int_as_float(rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return __int_as_float(halves[0]) + __int_as_float(halves[1]);
}

// The next up to RM copies of `left` (missing ones repeat the first); their number.
template <int RM>
__device__ __forceinline__ int take_copies(uint64_t* left, int32_t (&copy)[RM]) {
  int rows = 0;
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    copy[r] = *left ? __builtin_ctzll(*left) : copy[0];
    rows += *left ? 1 : 0;
    *left &= *left - 1;
  }
  return rows;
}

template <int RM>
__device__ __forceinline__ int32_t pick(const int32_t (&copy)[RM], int r) {
  int32_t c = copy[0];
#pragma unroll
  for (int i = 1; i < RM; ++i) c = r == i ? copy[i] : c;
  return c;
}

// Part `split` of `splits` of n, in whole blocks of 128.
__device__ __forceinline__ int part_start(int n, int split, int splits) { return 128 * (n / 128 * split / splits); }

template <int RM>
__global__ void __launch_bounds__(kThreads) few_up_kernel(FewArgs a) {
  __shared__ float sums[kWaves][RM][2][kColumns];
  if (blockIdx.x == 0)  // few_down's tickets
    for (int i = threadIdx.x; i < a.d_model / kColumns; i += kThreads) a.tickets[i] = 0;
  const int slices = a.ffn_dim / kColumns;
  const int unit = uniform(static_cast<int>(blockIdx.x) / slices), slice = uniform(static_cast<int>(blockIdx.x) % slices);
  const int c = uniform(unit / a.up_splits), split = uniform(unit % a.up_splits);
  int32_t expert;
  uint64_t left = copies_with(a, c, &expert);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane % kLanes, group = threadIdx.x / kLanes;
  const int n0 = slice * kColumns;
  const int from = part_start(a.d_model, split, a.up_splits), to = part_start(a.d_model, split + 1, a.up_splits);
  const int64_t stride = 2 * static_cast<int64_t>(a.ffn_dim), copies = static_cast<int64_t>(a.num_tokens) * a.k;
  while (left) {
    const uint16_t* w = a.w1 + static_cast<int64_t>(expert) * a.d_model * stride + n0 + 8 * col;
    int32_t copy[RM];
    const int rows = take_copies<RM>(&left, copy);
    float g[RM][8] = {}, u[RM][8] = {};
    for (int k0 = from + group * kStep; k0 < to; k0 += kGroups * kStep) {
      u32x4_t wg[kStep], wu[kStep], xr[RM];
#pragma unroll
      for (int r = 0; r < RM; ++r)
        xr[r] = *reinterpret_cast<const u32x4_t*>(a.x + static_cast<int64_t>(copy[r] / a.k) * a.d_model + k0);
#pragma unroll
      for (int j = 0; j < kStep; ++j) {
        wg[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(w + (k0 + j) * stride));
        wu[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(w + (k0 + j) * stride + a.ffn_dim));
      }
      float v[RM][kStep];
#pragma unroll
      for (int r = 0; r < RM; ++r)
#pragma unroll
        for (int j = 0; j < kStep; ++j)
          v[r][j] = __uint_as_float(j & 1 ? xr[r][j / 2] & 0xffff0000u : xr[r][j / 2] << 16);
      multiply_add<RM>(g, v, wg);
      multiply_add<RM>(u, v, wu);
    }
#pragma unroll
    for (int r = 0; r < RM; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float gs = column_sum(g[r][e]), us = column_sum(u[r][e]);
        if (lane < kLanes) {
          sums[wave][r][0][8 * col + e] = gs;
          sums[wave][r][1][8 * col + e] = us;
        }
      }
    __syncthreads();
    for (int q = threadIdx.x; q < rows * 2 * kColumns; q += kThreads) {
      const int r = q / (2 * kColumns), half = q / kColumns % 2, n = q % kColumns;
      float s = 0.0f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) s += sums[v][r][half][n];
      a.gu[(split * copies + pick<RM>(copy, r)) * stride + half * static_cast<int64_t>(a.ffn_dim) + n0 + n] = s;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ float few_gate(const FewArgs& a, int32_t i) {
  if (a.gate_dtype == SB_DTYPE_F32) return static_cast<const float*>(a.gates)[i];
  const uint16_t bits = static_cast<const uint16_t*>(a.gates)[i];
  return a.gate_dtype == SB_DTYPE_BF16 ? bf16_to_f32(bits) : static_cast<float>(__builtin_bit_cast(_Float16, bits));
}

// Columns n0 .. n0 + 127 of out, by one workgroup: four lanes per 4 columns of
// a token, each with every fourth part of F; their sums are added last.
__device__ __forceinline__ void few_out(const FewArgs& a, int n0, f32x4_t* __restrict__ lds) {
  constexpr int kShare = 4, kParts = kMaxSplits / kShare, kQuads = kColumns / 4;
  static_assert(kThreads == 2 * kShare * kQuads, "two tokens at most");
  const int q = threadIdx.x % kQuads, share = threadIdx.x / kQuads % kShare, t = threadIdx.x / (kQuads * kShare);
  const int32_t limit = token_limit(a);
  const int64_t copies = static_cast<int64_t>(a.num_tokens) * a.k;
  const float* from = a.part + n0 + 4 * q;
  f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if (t < limit) {
#pragma unroll 2
    for (int j = 0; j < a.k; ++j) {
      const int32_t c = t * a.k + j;
      const bool routed = expert_of(a, c, limit) >= 0;
      f32x4_t y[kParts];
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const int s = share + i * kShare;
        y[i] = routed && s < a.splits ? *reinterpret_cast<const f32x4_t*>(from + (s * copies + c) * a.d_model)
                                      : f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      }
#pragma unroll
      for (int i = 1; i < kParts; ++i) y[0] += y[i];
      if (routed) sum += few_gate(a, c) * y[0];
    }
  }
  lds[threadIdx.x] = sum;
  __syncthreads();
  if (share == 0 && t < limit) {
#pragma unroll
    for (int i = 1; i < kShare; ++i) sum += lds[threadIdx.x + i * kQuads];
    *reinterpret_cast<u32x2_t*>(a.out + static_cast<int64_t>(t) * a.d_model + n0 + 4 * q) =
        u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
  }
}

template <int RM, int ACT, bool TICKET>
__global__ void __launch_bounds__(kThreads) few_down_kernel(FewArgs a) {
  constexpr int kRange = 2048;  // of F, whose h is worked out once per workgroup
  __shared__ float sums[kWaves][RM][kColumns];
  __shared__ __attribute__((aligned(16))) float h[RM][kRange];
  const int slices = a.d_model / kColumns;
  const int unit = uniform(static_cast<int>(blockIdx.x) / slices), slice = uniform(static_cast<int>(blockIdx.x) % slices);
  const int c = uniform(unit / a.splits), split = uniform(unit % a.splits);
  int32_t expert;
  uint64_t left = copies_with(a, c, &expert);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane % kLanes, group = threadIdx.x / kLanes;
  const int n0 = slice * kColumns;
  const int from = part_start(a.ffn_dim, split, a.splits), to = part_start(a.ffn_dim, split + 1, a.splits);
  const int64_t stride = a.d_model, copies = static_cast<int64_t>(a.num_tokens) * a.k;
  while (left) {
    const uint16_t* w = a.w2 + static_cast<int64_t>(expert) * a.ffn_dim * stride + n0 + 8 * col;
    int32_t copy[RM];
    const int rows = take_copies<RM>(&left, copy);
    float y[RM][8] = {};
    for (int f0 = from; f0 < to; f0 += kRange) {
      const int count = min(kRange, to - f0);
      u32x4_t wr[kStep];
      auto load = [&](int k0) {
#pragma unroll
        for (int j = 0; j < kStep; ++j)
          wr[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(w + (f0 + k0 + j) * stride));
      };
      int k0 = group * kStep;
      if (k0 < count) load(k0);  // under way while h is worked out
      __syncthreads();           // the range before has been read
#pragma unroll
      for (int r = 0; r < RM; ++r)
        for (int f = threadIdx.x; f < count; f += kThreads) {
          const float* at = a.gu + copy[r] * 2 * static_cast<int64_t>(a.ffn_dim) + f0 + f;
          float g[kMaxUpSplits], u[kMaxUpSplits];
#pragma unroll
          for (int s = 0; s < kMaxUpSplits; ++s) {
            const bool there = s < a.up_splits;
            g[s] = there ? at[s * copies * 2 * a.ffn_dim] : 0.0f;
            u[s] = there ? at[s * copies * 2 * a.ffn_dim + a.ffn_dim] : 0.0f;
          }
#pragma unroll
          for (int s = 1; s < kMaxUpSplits; ++s) g[0] += g[s], u[0] += u[s];
          h[r][f] = gated_act<ACT>(g[0]) * u[0];
        }
      __syncthreads();
      while (k0 < count) {
        float v[RM][kStep];
#pragma unroll
        for (int r = 0; r < RM; ++r)
#pragma unroll
          for (int j = 0; j < kStep; ++j) v[r][j] = h[r][k0 + j];
        multiply_add<RM>(y, v, wr);
        k0 += kGroups * kStep;
        if (k0 < count) load(k0);
      }
    }
#pragma unroll
    for (int r = 0; r < RM; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = column_sum(y[r][e]);
        if (lane < kLanes) sums[wave][r][8 * col + e] = s;
      }
    __syncthreads();
    for (int q = threadIdx.x; q < rows * kColumns; q += kThreads) {
      const int r = q / kColumns, n = q % kColumns;
      float s = 0.0f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) s += sums[v][r][n];
      a.part[(split * copies + pick<RM>(copy, r)) * a.d_model + n0 + n] = s;
    }
    __syncthreads();
  }

  if constexpr (TICKET) {
    // The last of the slice's workgroups (all copies and parts) adds them up:
    // the others' sums are written back before their ticket is drawn, and read
    // from memory after the last one. Each wave waits for its own stores to be
    // in this XCD's L2, which the barrier does not do, so that the one write-back
    // behind it takes all of the workgroup's along.
    __shared__ int32_t last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      last = atomicAdd(a.tickets + slice, 1) == static_cast<int32_t>(copies) * a.splits - 1 ? 1 : 0;
      __threadfence();
    }
    __syncthreads();
    if (!last) return;
    auto* lds = reinterpret_cast<f32x4_t*>(&h[0][0]);
    static_assert(sizeof(h) >= kThreads * sizeof(f32x4_t), "room for the lanes' sums");
    few_out(a, n0, lds);
  }
}

__global__ void __launch_bounds__(kThreads) few_out_kernel(FewArgs a) {
  __shared__ f32x4_t lds[kThreads];
  few_out(a, static_cast<int>(blockIdx.x) * kColumns, lds);
}

// Parts of n for `units` workgroups each: until they are about three a CU, in
// whole blocks of 128.
int few_splits(int64_t units, int64_t n, int most, int cus) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({3 * cus / units, n / 128, most})));
}

template <int RM>
int run_few(const FewArgs& a, int32_t act, hipStream_t stream) {
  const uint32_t copies = static_cast<uint32_t>(a.num_tokens) * a.k;
  few_up_kernel<RM><<<copies * a.up_splits * (a.ffn_dim / 128), kThreads, 0, stream>>>(a);
  if (const int rc = check_launch("gated experts: few copies")) return rc;
  const uint32_t down = copies * a.splits * (a.d_model / 128);
  const bool ticket = down <= kTicketMost;
  auto launch = [&](auto kernel) { kernel<<<down, kThreads, 0, stream>>>(a); };
  if (act == SB_ACT_SILU) {
    if (ticket) launch(few_down_kernel<RM, SB_ACT_SILU, true>);
    else launch(few_down_kernel<RM, SB_ACT_SILU, false>);
  } else {
    if (ticket) launch(few_down_kernel<RM, SB_ACT_GELU, true>);
    else launch(few_down_kernel<RM, SB_ACT_GELU, false>);
  }
  if (ticket) return check_launch("gated experts: few copies");
  if (const int rc = check_launch("gated experts: few copies")) return rc;
  few_out_kernel<<<static_cast<uint32_t>(a.d_model / kColumns), kThreads, 0, stream>>>(a);
  return check_launch("gated experts: few copies");
}

}  // namespace

bool few_copies(int64_t num_tokens, int32_t k) { return num_tokens <= 2 && num_tokens * k <= 64; }

int64_t few_workspace_floats(int64_t num_copies, int64_t d_model, int64_t ffn_dim) {
  return num_copies * (kMaxUpSplits * 2 * ffn_dim + kMaxSplits * d_model) + d_model / kColumns;
}

int launch_few(const void* x, const void* expert_idx, int32_t idx_is_i64, const void* gates, int32_t gate_dtype,
               const void* w1, const void* w2, void* out, float* workspace, int64_t num_tokens, int32_t k,
               int64_t num_experts, int64_t d_model, int64_t ffn_dim, int32_t act, const int32_t* valid_tokens,
               hipStream_t stream) {
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  const int64_t copies = num_tokens * k;
  FewArgs a{};
  a.x = static_cast<const uint16_t*>(x);
  a.w1 = static_cast<const uint16_t*>(w1);
  a.w2 = static_cast<const uint16_t*>(w2);
  a.expert_idx = expert_idx;
  a.gates = gates;
  a.valid_tokens = valid_tokens;
  a.gu = workspace;
  a.part = workspace + copies * kMaxUpSplits * 2 * ffn_dim;
  a.tickets = reinterpret_cast<int32_t*>(a.part + copies * kMaxSplits * d_model);
  a.out = static_cast<uint16_t*>(out);
  a.gate_dtype = gate_dtype;
  a.idx_is_i64 = idx_is_i64;
  a.num_tokens = static_cast<int32_t>(num_tokens);
  a.k = k;
  a.num_experts = static_cast<int32_t>(num_experts);
  a.d_model = static_cast<int32_t>(d_model);
  a.ffn_dim = static_cast<int32_t>(ffn_dim);
  a.up_splits = few_splits(copies * (ffn_dim / 128), d_model, kMaxUpSplits, cus);
  a.splits = few_splits(copies * (d_model / 128), ffn_dim, kMaxSplits, cus);
  return num_tokens == 1 ? run_few<1>(a, act, stream) : run_few<2>(a, act, stream);
}

}  // namespace sb
