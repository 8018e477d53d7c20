// Root-mean-square norms before and after a block, fused with the block's gate,
// its scale and the residual sum (norm.hpp has the formulas).
//
// Bound by memory: norm_out with the next norm reads two rows and writes two.
// One pass: the row stays in registers (norm.hpp) between its sum of squares and its use,
// and so does `out` for the next norm's sum, which is taken of the rounded
// values: the next block starts from those, so norm_in of `out` gives the same
// bits. Sums in fp32.
//
// Rows of up to 2048 values are a wave's (no barrier, four rows a workgroup), longer ones
// a workgroup's of 4 or 16 waves; workgroups stay and take every so many rows, so that
// the weights are read once. Both norms, bf16: 4001 rows of 4096 in 22.7 us (5.8 TB/s of
// reads and writes; a large copy reaches 4.9), 8192 of 1024 in 15.3 (4.4), fp32 rows of
// 1001, loaded value by value, 2047 in 9.0 (3.6), one row of 2048 or less in 3.3. Beyond
// D = 8192 rows go through scratch: bf16, 4096 rows of 8192 in 46 us (5.8 TB/s), 4092 of
// 8200 in 260 (1.0), 2048 of 16384 in 189, 1024 of 32768 in 164.

#include "norm.hpp"

namespace sb {

int check_norm(const char* what, int32_t dtype, int64_t num_tokens, int64_t d, float eps,
               std::initializer_list<int32_t> dtypes, std::initializer_list<int64_t> strides) {
  auto known = [](int32_t t) { return t == SB_DTYPE_BF16 || t == SB_DTYPE_F16 || t == SB_DTYPE_F32; };
  if (!known(dtype)) return fail(SB_ERR_INVALID, "%s: unsupported dtype code %d", what, dtype);
  for (int32_t t : dtypes)
    if (!known(t)) return fail(SB_ERR_INVALID, "%s: unsupported dtype code %d", what, t);
  if (num_tokens < 0 || num_tokens > 2147483647LL || d <= 0 || d > kNormMaxD)
    return fail(SB_ERR_INVALID, "%s: 0 <= T < 2^31 and 0 < D <= %lld, got %lld and %lld", what,
                static_cast<long long>(kNormMaxD), static_cast<long long>(num_tokens), static_cast<long long>(d));
  if (!(eps >= 0.0f)) return fail(SB_ERR_INVALID, "%s: eps must not be negative", what);
  for (int64_t s : strides)
    if (s < 0) return fail(SB_ERR_INVALID, "%s: negative stride", what);
  return SB_OK;
}

namespace {

template <int DTYPE, int G, int NCH, bool VEC, bool OUT, bool NEXT>
__global__ void __launch_bounds__(norm_threads(G)) norm_kernel(NormArgs a) {
  using S = Share<G, NCH, VEC>;
  constexpr int kGroups = norm_threads(G) / G;
  constexpr int kElem = DTYPE == SB_DTYPE_F32 ? 4 : 2;
  __shared__ float sums[2][G > 64 ? G / 64 : 1][1];
  GroupSum<G, 1> sum(sums);
  const int t = threadIdx.x % G;
  const int64_t limit = a.valid_tokens ? min(a.num_tokens, static_cast<int64_t>(max(0, *a.valid_tokens))) : a.num_tokens;
  float w[OUT ? S::kValues : 1], v[NEXT ? S::kValues : 1];
  if constexpr (OUT) {
    load_vector<S, VEC>(a.weight, a.weight_dtype, 0, a.d, t, 1.0f, w);
    if (a.gate_kind == SB_GATE_CHANNEL) {
      float g[S::kValues];
      load_vector<S, VEC>(a.gate, a.gate_dtype, 0, a.d, t, 0.0f, g);
#pragma unroll
      for (int i = 0; i < S::kValues; ++i) w[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < S::kValues; ++i) w[i] *= a.scale;
  }
  if constexpr (NEXT) load_vector<S, VEC>(a.next_weight, a.next_dtype, 0, a.d, t, 1.0f, v);

  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / G; row < limit;
       row += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t to = row * a.d * kElem;
    float x[S::kValues];
    load_row<S, DTYPE, VEC>(static_cast<const uint8_t*>(a.x) + row * a.x_stride * kElem, a.d, t, x);
    if constexpr (OUT) {
      float y[S::kValues];
      load_row<S, DTYPE, VEC>(static_cast<const uint8_t*>(a.y) + row * a.y_stride * kElem, a.d, t, y);
      float ss[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < S::kValues; ++i) ss[0] = fmaf(y[i], y[i], ss[0]);
      sum(ss);
      float r = 1.0f / sqrtf(ss[0] * a.inv_d + a.eps);
      if (a.gate_kind == SB_GATE_TOKEN) r *= load_as_f32(a.gate, a.gate_dtype, row * a.gate_stride);
      if (a.gate_kind == SB_GATE_FULL) {
        float g[S::kValues];
        load_vector<S, VEC>(a.gate, a.gate_dtype, row * a.gate_stride, a.d, t, 0.0f, g);
#pragma unroll
        for (int i = 0; i < S::kValues; ++i) y[i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < S::kValues; ++i) x[i] = rounded<DTYPE>(fmaf(y[i] * r, w[i], x[i]));
      store_row<S, DTYPE, VEC>(static_cast<uint8_t*>(a.out) + to, a.d, t, x);
    }
    if constexpr (NEXT) {
      float ss[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < S::kValues; ++i) ss[0] = fmaf(x[i], x[i], ss[0]);
      sum(ss);
      const float r = 1.0f / sqrtf(ss[0] * a.inv_d + a.eps);
#pragma unroll
      for (int i = 0; i < S::kValues; ++i) x[i] = x[i] * r * v[i];
      store_row<S, DTYPE, VEC>(static_cast<uint8_t*>(a.next) + to, a.d, t, x);
    }
  }
}

template <bool OUT, bool NEXT>
int launch_norm(const NormArgs& a, int32_t dtype, bool vec, hipStream_t stream) {
  if (a.num_tokens == 0) return SB_OK;
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  return with_dtype(dtype, [&](auto type) {
    with_norm_form<false>(a.d, vec, [&](auto g, auto chunks, auto vectors) {
      constexpr int G = decltype(g)::value, kThreads = norm_threads(G), kGroups = kThreads / G;
      const int64_t groups = (a.num_tokens + kGroups - 1) / kGroups;
      const uint32_t grid = static_cast<uint32_t>(std::min<int64_t>(groups, int64_t{2048 / kThreads} * cus));
      norm_kernel<decltype(type)::value, G, decltype(chunks)::value, decltype(vectors)::value, OUT, NEXT>
          <<<grid, kThreads, 0, stream>>>(a);
    });
    return check_launch("norm");
  });
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_norm_in(const void* x, int64_t x_stride, const void* weight, int32_t weight_dtype, void* out,
                          int32_t dtype, int64_t num_tokens, int64_t d_model, float eps, const int32_t* valid_tokens,
                          void* stream) {
  if (const int rc = check_norm("norm_in", dtype, num_tokens, d_model, eps, {weight_dtype}, {x_stride})) return rc;
  if (num_tokens > 0 && (!x || !out)) return fail(SB_ERR_INVALID, "norm_in: null buffer");
  NormArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.next_weight = weight;
  a.next_dtype = weight_dtype;
  a.next = out;
  a.num_tokens = num_tokens;
  a.d = static_cast<int32_t>(d_model);
  a.eps = eps;
  a.inv_d = 1.0f / static_cast<float>(d_model);
  a.valid_tokens = valid_tokens;
  const bool vec = norm_vectors(d_model, {{x, x_stride, dtype}, {out, 0, dtype}, {weight, 0, weight_dtype}});
  if (const int rc = launch_norm<false, true>(a, dtype, vec, as_stream(stream))) return rc;
  return clear_ok();
}

extern "C" int sb_norm_out(const void* y, int64_t y_stride, const void* x, int64_t x_stride, const void* weight,
                           int32_t weight_dtype, const void* gate, int32_t gate_dtype, int32_t gate_kind,
                           int64_t gate_stride, float scale, const void* next_weight, int32_t next_dtype, void* out,
                           void* next, int32_t dtype, int64_t num_tokens, int64_t d_model, float eps,
                           const int32_t* valid_tokens, void* stream) {
  if (const int rc = check_norm("norm_out", dtype, num_tokens, d_model, eps, {weight_dtype, gate_dtype, next_dtype},
                                {y_stride, x_stride, gate_stride}))
    return rc;
  if (gate_kind < SB_GATE_NONE || gate_kind > SB_GATE_FULL || (gate_kind != SB_GATE_NONE && !gate && num_tokens > 0))
    return fail(SB_ERR_INVALID, "norm_out: gate kind %d", gate_kind);
  if (num_tokens > 0 && (!y || !x || !out)) return fail(SB_ERR_INVALID, "norm_out: null buffer");
  NormArgs a{};
  a.y = y;
  a.x = x;
  a.y_stride = y_stride;
  a.x_stride = x_stride;
  a.weight = weight;
  a.weight_dtype = weight_dtype;
  a.gate = gate;
  a.gate_dtype = gate_dtype;
  a.gate_kind = gate_kind;
  a.gate_stride = gate_stride;
  a.scale = scale;
  a.next_weight = next_weight;
  a.next_dtype = next_dtype;
  a.out = out;
  a.next = next;
  a.num_tokens = num_tokens;
  a.d = static_cast<int32_t>(d_model);
  a.eps = eps;
  a.inv_d = 1.0f / static_cast<float>(d_model);
  a.valid_tokens = valid_tokens;
  const bool vec = norm_vectors(
      d_model, {{y, y_stride, dtype}, {x, x_stride, dtype}, {out, 0, dtype}, {next, 0, dtype}, {weight, 0, weight_dtype},
                {gate_kind == SB_GATE_TOKEN ? nullptr : gate, gate_kind == SB_GATE_FULL ? gate_stride : 0, gate_dtype},
                {next_weight, 0, next_dtype}});
  if (const int rc = next ? launch_norm<true, true>(a, dtype, vec, as_stream(stream))
                          : launch_norm<true, false>(a, dtype, vec, as_stream(stream)))
    return rc;
  return clear_ok();
}
