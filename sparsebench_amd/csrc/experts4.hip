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
// A workgroup of up4 / down4 owns 32 columns (in up4, of both halves) of one
// expert and the rows of its copies, 32 at a time; its 8 waves share the
// reduction, 64 k each in turn, and add up through LDS in a fixed order. A lane's
// 16 bytes of codes are 32 k of a column: one load and one scale feed four
// 32 x 32 x 16 products whose k are taken in that order on both sides.
// No routing kernel: a workgroup collects its expert's copies from the ids.

#include "gated_act.hpp"
#include "gated.hpp"
#include "workspace.hpp"

namespace sb {
namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kCols = 32, kRows = 32, kStepK = 64;
constexpr int kMaxCopies = 2048, kMaxSplits = 8, kMaxRowGroups = 8;
constexpr int kTileBytes = kCols * kStepK / 2;  // codes of a step: 16 bytes a lane

struct Few4Args {
  const uint16_t* x;
  const void *expert_idx, *gates;
  const uint8_t *w1, *s1, *w2, *s2;
  const int32_t* valid_tokens;
  uint16_t *h, *out;
  float* part;
  int32_t idx_is_i64, num_tokens, k, num_experts, d_model, ffn_dim, splits, gate_dtype, units;
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

struct Copies {
  int32_t counts[kWaves];
  uint16_t list[kMaxCopies];
};

// The copies of a unit's expert, in order, and their number; *expert. A unit is
// an expert, or, where there are fewer copies than experts, the copy that is the
// first of its expert (0 copies for the others).
__device__ __forceinline__ int collect(const Few4Args& a, int unit, Copies& lds, int* expert) {
  const int32_t limit = copy_limit(a);
  int e = unit;
  if (a.units < a.num_experts) e = unit < limit ? uniform(expert_of(a, unit)) : -1;
  *expert = e;
  if (e < 0) return 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int found = 0;
  for (int c0 = 0; c0 < limit; c0 += kThreads) {
    const int c = c0 + static_cast<int>(threadIdx.x);
    const bool mine = c < limit && expert_of(a, c) == e;
    const uint64_t all = __ballot(mine);
    if (lane == 0) lds.counts[wave] = __builtin_popcountll(all);
    __syncthreads();
    int at = found + __builtin_popcountll(all & ((uint64_t{1} << lane) - 1));
    for (int w = 0; w < kWaves; ++w) {
      const int n = lds.counts[w];
      at += w < wave ? n : 0;
      found += n;
    }
    if (mine) lds.list[at] = static_cast<uint16_t>(c);
    __syncthreads();
  }
  if (a.units < a.num_experts && (found == 0 || lds.list[0] != unit)) return 0;
  return uniform(found);
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

// acc[p] += rows . column tile p over steps first, first + kWaves, ... < last.
// row: the lane's row of A (its lane % 32), at k = 32 (lane / 32), or null;
// codes, scales: column tile p's, at the lane's place.
template <int P>
__device__ __forceinline__ void multiply(f32x16_t (&acc)[P], const uint16_t* row, const uint8_t* const (&codes)[P],
                                         const uint8_t* const (&scales)[P], int first, int last) {
  struct Step {
    u32x4_t w[P], a[4];
    uint8_t s[P];
  };
  auto load = [&](int t, Step& s) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      s.w[p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(codes[p] + static_cast<int64_t>(t) * kTileBytes));
      s.s[p] = scales[p][t * 64];
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      s.a[q] = row ? *reinterpret_cast<const u32x4_t*>(row + t * kStepK + 8 * q) : u32x4_t{0u, 0u, 0u, 0u};
  };
  auto use = [&](const Step& s) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const float scale = scale_of(s.s[p]);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        acc[p] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, s.a[q]),
                                                         dequantize(s.w[p][q], scale), acc[p], 0, 0, 0);
    }
  };
  Step now, next;
  int t = first;
  if (t >= last) return;
  load(t, now);
  for (; t + kWaves < last; t += kWaves) {
    load(t + kWaves, next);
    use(now);
    now = next;
  }
  use(now);
}

// The row of acc[.][v] in a tile: a lane holds one column (lane % 32).
__device__ __forceinline__ int acc_row(int v, int lane) { return 8 * (v / 4) + 4 * (lane >> 5) + v % 4; }

using Sums = float[kWaves][16][64];

template <int P>
__device__ __forceinline__ void put_sums(Sums (&sums)[P], const f32x16_t (&acc)[P], int rows) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int v = 0; v < 16; ++v)
    if (v / 4 * 8 < rows)
#pragma unroll
      for (int p = 0; p < P; ++p) sums[p][wave][v][lane] = acc[p][v];
}

__device__ __forceinline__ float get_sum(const Sums& sums, int v, int lane) {
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s += sums[w][v][lane];
  return s;
}

template <int ACT>
__global__ void __launch_bounds__(kThreads) up4_kernel(Few4Args a) {
  __shared__ Copies copies;
  __shared__ Sums sums[2];
  const int tiles = a.ffn_dim / kCols;
  const int unit = uniform(static_cast<int>(blockIdx.x) / tiles), tile = uniform(static_cast<int>(blockIdx.x) % tiles);
  int expert;
  const int count = collect(a, unit, copies, &expert);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int steps = a.d_model / kStepK;
  for (int r0 = static_cast<int>(blockIdx.y) * kRows; r0 < count; r0 += static_cast<int>(gridDim.y) * kRows) {
    const int rows = min(kRows, count - r0), m = lane % kRows;
    const uint16_t* row =
        m < rows ? a.x + static_cast<int64_t>(copies.list[r0 + m] / a.k) * a.d_model + 32 * (lane >> 5) : nullptr;
    const uint8_t *codes[2], *scales[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int64_t at = (static_cast<int64_t>(expert) * 2 * tiles + p * tiles + tile) * steps;
      codes[p] = a.w1 + at * kTileBytes + lane * 16;
      scales[p] = a.s1 + at * 64 + lane;
    }
    f32x16_t acc[2] = {};
    multiply<2>(acc, row, codes, scales, wave, steps);
    put_sums<2>(sums, acc, rows);
    __syncthreads();
    for (int v = wave; v < 16; v += kWaves) {
      const int r = acc_row(v, lane);
      if (r >= rows) continue;
      const float g = get_sum(sums[0], v, lane), u = get_sum(sums[1], v, lane);
      a.h[static_cast<int64_t>(copies.list[r0 + r]) * a.ffn_dim + tile * kCols + lane % kCols] =
          f32_to_bf16(gated_act<ACT>(g) * u);
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads) down4_kernel(Few4Args a) {
  __shared__ Copies copies;
  __shared__ Sums sums[1];
  const int tiles = a.d_model / kCols;
  int at = static_cast<int>(blockIdx.x);
  const int tile = uniform(at % tiles);
  at /= tiles;
  const int split = uniform(at % a.splits), unit = uniform(at / a.splits);
  int expert;
  const int count = collect(a, unit, copies, &expert);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int steps = a.ffn_dim / kStepK;
  const int first = static_cast<int>(static_cast<int64_t>(steps) * split / a.splits);
  const int last = static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / a.splits);
  const int64_t num_copies = static_cast<int64_t>(a.num_tokens) * a.k;
  for (int r0 = static_cast<int>(blockIdx.y) * kRows; r0 < count; r0 += static_cast<int>(gridDim.y) * kRows) {
    const int rows = min(kRows, count - r0), m = lane % kRows;
    const uint16_t* row =
        m < rows ? a.h + static_cast<int64_t>(copies.list[r0 + m]) * a.ffn_dim + 32 * (lane >> 5) : nullptr;
    const int64_t from = (static_cast<int64_t>(expert) * tiles + tile) * steps;
    const uint8_t* const codes[1] = {a.w2 + from * kTileBytes + lane * 16};
    const uint8_t* const scales[1] = {a.s2 + from * 64 + lane};
    f32x16_t acc[1] = {};
    multiply<1>(acc, row, codes, scales, first + wave, last);
    put_sums<1>(sums, acc, rows);
    __syncthreads();
    for (int v = wave; v < 16; v += kWaves) {
      const int r = acc_row(v, lane);
      if (r < rows)
        a.part[(split * num_copies + copies.list[r0 + r]) * a.d_model + tile * kCols + lane % kCols] =
            get_sum(sums[0], v, lane);
    }
    __syncthreads();
  }
}

__device__ __forceinline__ float gate_of(const Few4Args& a, int64_t i) {
  if (a.gate_dtype == SB_DTYPE_F32) return static_cast<const float*>(a.gates)[i];
  const uint16_t bits = static_cast<const uint16_t*>(a.gates)[i];
  return a.gate_dtype == SB_DTYPE_BF16 ? bf16_to_f32(bits) : static_cast<float>(__builtin_bit_cast(_Float16, bits));
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

// Workgroups share the rows of an expert that has many, and the reduction of
// the second product until there are about four a CU.
struct Few4Form {
  int units, row_groups, splits;
};

Few4Form few4_form(int64_t copies, int64_t num_experts, int64_t d_model, int64_t ffn_dim, int cus) {
  Few4Form f;
  f.units = static_cast<int>(std::min(copies, num_experts));
  f.row_groups = static_cast<int>(
      std::min<int64_t>(kMaxRowGroups, std::max<int64_t>(1, copies / f.units / kRows)));
  const int64_t groups = f.units * f.row_groups * (d_model / kCols);
  f.splits = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>({kMaxSplits, 4 * cus / groups, ffn_dim / kStepK / kWaves})));
  return f;
}

struct Few4Buffers {
  uint16_t* h;
  float* part;
  int64_t used;
};

Few4Buffers carve_few4(void* workspace, int64_t copies, int64_t d_model, int64_t ffn_dim, int splits) {
  Carver ws{static_cast<uint8_t*>(workspace)};
  Few4Buffers b;
  b.h = ws.take<uint16_t>(copies * ffn_dim);
  b.part = ws.take<float>(splits * copies * d_model);
  b.used = ws.used;
  return b;
}

int check_few4(int64_t num_tokens, int32_t k, int32_t num_experts, int64_t d_model, int64_t ffn_dim) {
  if (num_tokens <= 0 || k <= 0 || num_tokens > kMaxCopies / k)
    return fail(SB_ERR_INVALID, "4-bit experts: T, k > 0 and at most %d copies, got %lld x %d", kMaxCopies,
                static_cast<long long>(num_tokens), k);
  if (num_experts <= 0 || num_experts > 1024)
    return fail(SB_ERR_INVALID, "4-bit experts: num_experts must be in [1, 1024], got %d", num_experts);
  if (d_model <= 0 || d_model % 128 != 0 || ffn_dim <= 0 || ffn_dim % 128 != 0 || d_model > (1 << 20) ||
      ffn_dim > (1 << 20))
    return fail(SB_ERR_INVALID, "4-bit experts: D (%lld) and F (%lld) must be multiples of 128, up to 2^20",
                static_cast<long long>(d_model), static_cast<long long>(ffn_dim));
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
  if (workspace_bytes) *workspace_bytes = carve_few4(nullptr, copies, d_model, ffn_dim, f.splits).used;
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
  const Few4Buffers b = carve_few4(workspace, copies, d_model, ffn_dim, f.splits);
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
  const dim3 up(static_cast<uint32_t>(f.units * (ffn_dim / kCols)), static_cast<uint32_t>(f.row_groups));
  if (act == SB_ACT_SILU) up4_kernel<SB_ACT_SILU><<<up, kThreads, 0, s>>>(a);
  else up4_kernel<SB_ACT_GELU><<<up, kThreads, 0, s>>>(a);
  if (const int rc = check_launch("4-bit experts")) return rc;
  const dim3 down(static_cast<uint32_t>(f.units * f.splits * (d_model / kCols)), static_cast<uint32_t>(f.row_groups));
  down4_kernel<<<down, kThreads, 0, s>>>(a);
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
