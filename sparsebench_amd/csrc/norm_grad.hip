// The backward pass of the norms before and after a block (norm.hpp). With
// o = out (norm_in: x), rn and r the rows' reciprocal roots:
//
//   do' = do + rn (v dn - on mean(v dn on)),      on = o rn,  dx = do'
//   p   = s n(y) do'                               n(y) = y r
//   dy  = r (s g w do' - n(y) mean(g w p))
//   dw  = sum_t g p,  dg = w p summed over what g is broadcast to,  dv = sum_t dn on
//
// One pass: the sums of a row that need no other sum (o^2, y^2, v dn o) are
// taken together, then sum(g w p). Rows are read once and kept in registers up to D = 4096.
// dw and dv are summed over a workgroup's rows in registers, over its groups in
// LDS, and over the workgroups by a second kernel, in a fixed order: the same
// bits every time. A gate of the channels has dg = w q and dw = g q with one
// sum q = sum_t p. Bound by memory: 4 rows read, 2 written; the next row is loaded while
// one is worked on. 8192 rows of 1024, bf16: 21.9 us (4.6 TB/s), and the sums of 512
// workgroups 4.0; 8192 of 4096 91 (4.4 TB/s). Beyond D = 4096 part of them goes through
// scratch (norm.hpp): 6553 rows of 5120 181 us (2.2 TB/s), 4096 of 8192 147 (2.7), 4092 of 8200 654
// (0.6), 2048 of 16384 381 (1.1), 1024 of 32768 792 (0.5).

#include "norm.hpp"
#include "workspace.hpp"

namespace sb {
namespace {

template <int DTYPE, int G, int NCH, bool VEC, bool OUT, bool NEXT>
__global__ void __launch_bounds__(norm_threads(G)) norm_grad_kernel(NormArgs a) {
  using S = Share<G, NCH, VEC>;
  constexpr int N = S::kValues;
  constexpr int kThreads = norm_threads(G), kGroups = kThreads / G;
  constexpr int kElem = DTYPE == SB_DTYPE_F32 ? 4 : 2;
  __shared__ float sums3[2][G > 64 ? G / 64 : 1][3];
  __shared__ float sums1[2][G > 64 ? G / 64 : 1][1];
  GroupSum<G, 3> sum3(sums3);
  GroupSum<G, 1> sum1(sums1);
  const int t = threadIdx.x % G;
  const int64_t limit = a.valid_tokens ? min(a.num_tokens, static_cast<int64_t>(max(0, *a.valid_tokens))) : a.num_tokens;
  struct Rows {
    RowRegs<S, DTYPE, VEC> d, o, dn, y;
  };
  auto load = [&](int64_t row, Rows& r) {
    auto one = [&](RowRegs<S, DTYPE, VEC>& regs, const void* p, int64_t stride) {
      regs.load(static_cast<const uint8_t*>(p) + row * stride * kElem, a.d, t);
    };
    if (OUT || a.grad_out) one(r.d, a.grad_out, a.grad_out_stride);
    if constexpr (NEXT) {
      one(r.o, a.x, a.x_stride);
      one(r.dn, a.grad_next, a.grad_next_stride);
    }
    if constexpr (OUT) one(r.y, a.y, a.y_stride);
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / G;
  Rows ahead;
  if (VEC && row < limit) load(row, ahead);  // before the weights: they are waited for first
  // w: the weight, times the gate where that is one of the channels.
  float w[OUT ? N : 1], v[NEXT ? N : 1], q[OUT ? N : 1], dv[NEXT ? N : 1];
  if constexpr (OUT) {
    load_vector<S, VEC>(a.weight, a.weight_dtype, 0, a.d, t, 1.0f, w);
    if (a.gate_kind == SB_GATE_CHANNEL) {
      float g[N];
      load_vector<S, VEC>(a.gate, a.gate_dtype, 0, a.d, t, 0.0f, g);
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = 0.0f;
  }
  if constexpr (NEXT) {
    load_vector<S, VEC>(a.next_weight, a.next_dtype, 0, a.d, t, 1.0f, v);
#pragma unroll
    for (int i = 0; i < N; ++i) dv[i] = 0.0f;
  }

  for (; row < limit; row += step) {
    const int64_t to = row * a.d * kElem;
    float d[N], o[NEXT ? N : 1], dn[NEXT ? N : 1], y[OUT ? N : 1];
    if constexpr (!VEC) load(row, ahead);
    if (OUT || a.grad_out) {
      ahead.d.take(d);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = 0.0f;
    }
    if constexpr (NEXT) {
      ahead.o.take(o);
      ahead.dn.take(dn);
    }
    if constexpr (OUT) ahead.y.take(y);
    if (VEC && row + step < limit) load(row + step, ahead);  // under way while this row is worked on
    float s[3] = {0.0f, 0.0f, 0.0f};  // sums of o^2, y^2 and v dn o
    if constexpr (OUT) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[1] = fmaf(y[i], y[i], s[1]);
    }
    if constexpr (NEXT) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s[0] = fmaf(o[i], o[i], s[0]);
        s[2] = fmaf(v[i] * dn[i], o[i], s[2]);
      }
    }
    sum3(s);
    if constexpr (NEXT) {
      const float rn = 1.0f / sqrtf(s[0] * a.inv_d + a.eps);
      const float back = rn * rn * (s[2] * a.inv_d);  // mean(v dn on) rn, of o
#pragma unroll
      for (int i = 0; i < N; ++i) {
        dv[i] = fmaf(dn[i] * rn, o[i], dv[i]);
        d[i] += rn * (v[i] * dn[i] - back * o[i]);
      }
      store_row<S, DTYPE, VEC>(static_cast<uint8_t*>(a.dx) + to, a.d, t, d);
    }
    if constexpr (OUT) {
      const float r = 1.0f / sqrtf(s[1] * a.inv_d + a.eps);
      const float token_gate =
          a.gate_kind == SB_GATE_TOKEN ? load_as_f32(a.gate, a.gate_dtype, row * a.gate_stride) : 1.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        y[i] *= r;
        d[i] *= a.scale;
      }
      if (a.gate_kind == SB_GATE_FULL) {
        float g[N], dg[N];
        load_vector<S, VEC>(a.gate, a.gate_dtype, row * a.gate_stride, a.d, t, 0.0f, g);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          dg[i] = w[i] * y[i] * d[i];
          d[i] *= g[i];
        }
        by_dtype(a.gate_dtype, [&](auto type) {
          constexpr int kType = decltype(type)::value;
          store_row<S, kType, VEC>(static_cast<uint8_t*>(a.dgate) + row * a.d * (kType == SB_DTYPE_F32 ? 4 : 2), a.d, t, dg);
        });
      }
      float p[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        p[0] = fmaf(w[i] * y[i], d[i], p[0]);
        q[i] = fmaf(token_gate * y[i], d[i], q[i]);
      }
      sum1(p);
      if (a.gate_kind == SB_GATE_TOKEN && t == 0) store_as(a.dgate, a.gate_dtype, row, p[0]);
      const float mean = p[0] * token_gate * a.inv_d, size = r * token_gate;
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = size * (w[i] * d[i]) - r * mean * y[i];
      store_row<S, DTYPE, VEC>(static_cast<uint8_t*>(a.dy) + to, a.d, t, y);
    }
  }

  // The workgroup's sums: its groups' one after another.
  float* const mine = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.d;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = S::column(i, t);
      if (at >= a.d) continue;
      if constexpr (OUT) mine[at] = q[i];
      if constexpr (NEXT) mine[a.d + at] = dv[i];
    }
  } else {
    __shared__ float part[kGroups][8 * G * NCH];
    auto join = [&](const float (&mine_of)[N], float* to) {
#pragma unroll
      for (int i = 0; i < N; ++i) part[threadIdx.x / G][S::column(i, t)] = mine_of[i];
      __syncthreads();
      for (int at = threadIdx.x; at < a.d; at += kThreads) {
        float s = part[0][at];
#pragma unroll
        for (int g = 1; g < kGroups; ++g) s += part[g][at];
        to[at] = s;
      }
      __syncthreads();
    };
    if constexpr (OUT) join(q, mine);
    if constexpr (NEXT) join(dv, mine + a.d);
  }
}

// The sums over the workgroups: 64 rows of 16 lanes take every 64th of them for
// 16 columns, then are added in order. blockIdx.y 0: the weight (and a gate of
// the channels), 1: the next weight.
struct SumArgs {
  const float* partial;
  const void *weight, *gate;
  void *dweight, *dgate, *dnext;
  int32_t parts, d, weight_dtype, gate_dtype, next_dtype;
};
constexpr int kSumRows = 64, kSumCols = 16;

__global__ void __launch_bounds__(kSumRows * kSumCols) norm_sum_kernel(SumArgs a) {
  __shared__ float sums[kSumRows][kSumCols];
  const int c = threadIdx.x % kSumCols, r = threadIdx.x / kSumCols;
  const int half = blockIdx.y, at = static_cast<int>(blockIdx.x) * kSumCols + c;
  if (half == 0 ? !a.dweight && !a.dgate : !a.dnext) return;
  float s = 0.0f;
  if (at < a.d) {
    const float* from = a.partial + static_cast<int64_t>(half) * a.d + at;
#pragma unroll 8
    for (int i = r; i < a.parts; i += kSumRows) s += from[static_cast<int64_t>(i) * 2 * a.d];
  }
  sums[r][c] = s;
  __syncthreads();
  if (r >= 4) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < kSumRows / 4; ++i) s += sums[i * 4 + r][c];
  // The four rows of lanes of the first wave.
  s += __shfl_xor(s, 16);
  s += __shfl_xor(s, 32);
  if (r != 0 || at >= a.d) return;
  if (half == 1) {
    store_as(a.dnext, a.next_dtype, at, s);
    return;
  }
  if (a.dweight) store_as(a.dweight, a.weight_dtype, at, a.gate ? s * load_as_f32(a.gate, a.gate_dtype, at) : s);
  if (a.dgate) store_as(a.dgate, a.gate_dtype, at, a.weight ? s * load_as_f32(a.weight, a.weight_dtype, at) : s);
}

// Workgroups of a backward pass: each leaves a partial sum, so no more than
// the device holds at once.
int64_t grad_workgroups(int64_t num_tokens, int64_t d, int cus) {
  int64_t grid = 1;
  with_norm_form<true>(d, true, [&](auto g, auto, auto) {
    constexpr int kThreads = norm_threads(decltype(g)::value), kGroups = kThreads / decltype(g)::value;
    grid = std::min<int64_t>((num_tokens + kGroups - 1) / kGroups, int64_t{std::max(1, 512 / kThreads)} * cus);
  });
  return std::max<int64_t>(1, grid);
}

template <bool OUT, bool NEXT>
int launch_grad(const NormArgs& a, int32_t dtype, bool vec, uint32_t grid, hipStream_t stream) {
  return with_dtype(dtype, [&](auto type) {
    with_norm_form<true>(a.d, vec, [&](auto g, auto chunks, auto vectors) {
      constexpr int G = decltype(g)::value;
      norm_grad_kernel<decltype(type)::value, G, decltype(chunks)::value, decltype(vectors)::value, OUT, NEXT>
          <<<grid, norm_threads(G), 0, stream>>>(a);
    });
    return check_launch("norm gradients");
  });
}

int run_grad(NormArgs& a, int32_t dtype, bool out, bool next, bool vec, void* dweight, void* dnext, void* workspace,
             int64_t workspace_bytes, hipStream_t stream) {
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  const int64_t grid = grad_workgroups(a.num_tokens, a.d, cus);
  if (const int rc = check_workspace(workspace, workspace_bytes, grid * 2 * a.d * 4)) return rc;
  a.partial = static_cast<float*>(workspace);
  a.inv_d = 1.0f / static_cast<float>(a.d);
  const uint32_t groups = static_cast<uint32_t>(grid);
  const int rc = out && next ? launch_grad<true, true>(a, dtype, vec, groups, stream)
                 : out       ? launch_grad<true, false>(a, dtype, vec, groups, stream)
                             : launch_grad<false, true>(a, dtype, vec, groups, stream);
  if (rc) return rc;
  const bool channel = a.gate_kind == SB_GATE_CHANNEL;
  const SumArgs s{a.partial,      channel ? a.weight : nullptr, channel ? a.gate : nullptr,
                  dweight,        channel ? a.dgate : nullptr,  dnext,
                  static_cast<int32_t>(grid), a.d, a.weight_dtype, a.gate_dtype, a.next_dtype};
  if (!s.dweight && !s.dgate && !s.dnext) return SB_OK;
  norm_sum_kernel<<<dim3(static_cast<uint32_t>((a.d + kSumCols - 1) / kSumCols), 2), kSumRows * kSumCols, 0, stream>>>(s);
  return check_launch("norm gradients: sums");
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_norm_sizes(int64_t num_tokens, int64_t d_model, int64_t* workspace_bytes) {
  if (const int rc = check_norm("norm", SB_DTYPE_F32, num_tokens, d_model, 0.0f, {}, {})) return rc;
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  if (workspace_bytes) *workspace_bytes = grad_workgroups(num_tokens, d_model, cus) * 2 * d_model * 4;
  return clear_ok();
}

extern "C" int sb_norm_in_backward(const void* grad, int64_t grad_stride, const void* x, int64_t x_stride,
                                   const void* weight, int32_t weight_dtype, const void* grad_x, int64_t grad_x_stride,
                                   void* dx, void* dweight, int32_t dtype, int64_t num_tokens, int64_t d_model,
                                   float eps, const int32_t* valid_tokens, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  if (const int rc = check_norm("norm_in_backward", dtype, num_tokens, d_model, eps, {weight_dtype},
                                {grad_stride, x_stride, grad_x_stride}))
    return rc;
  if (num_tokens > 0 && (!grad || !x || !dx)) return fail(SB_ERR_INVALID, "norm_in_backward: null buffer");
  NormArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.grad_next = grad;
  a.grad_next_stride = grad_stride;
  a.grad_out = grad_x;
  a.grad_out_stride = grad_x_stride;
  a.next_weight = weight;
  a.next_dtype = weight_dtype;
  a.dx = dx;
  a.num_tokens = num_tokens;
  a.d = static_cast<int32_t>(d_model);
  a.eps = eps;
  a.valid_tokens = valid_tokens;
  const bool vec = norm_vectors(d_model, {{grad, grad_stride, dtype}, {x, x_stride, dtype}, {dx, 0, dtype},
                                          {grad_x, grad_x_stride, dtype}, {weight, 0, weight_dtype}});
  if (const int rc = run_grad(a, dtype, false, true, vec, nullptr, dweight, workspace, workspace_bytes, as_stream(stream)))
    return rc;
  return clear_ok();
}

extern "C" int sb_norm_out_backward(const void* grad_out, int64_t grad_out_stride, const void* grad_next,
                                    int64_t grad_next_stride, const void* y, int64_t y_stride, const void* out,
                                    int64_t out_stride, const void* weight, int32_t weight_dtype, const void* gate,
                                    int32_t gate_dtype, int32_t gate_kind, int64_t gate_stride, float scale,
                                    const void* next_weight, int32_t next_dtype, void* dy, void* dx, void* dweight,
                                    void* dgate, void* dnext_weight, int32_t dtype, int64_t num_tokens,
                                    int64_t d_model, float eps, const int32_t* valid_tokens, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  if (const int rc = check_norm("norm_out_backward", dtype, num_tokens, d_model, eps,
                                {weight_dtype, gate_dtype, next_dtype},
                                {grad_out_stride, grad_next_stride, y_stride, out_stride, gate_stride}))
    return rc;
  const bool next = grad_next != nullptr;
  if (gate_kind < SB_GATE_NONE || gate_kind > SB_GATE_FULL ||
      (gate_kind != SB_GATE_NONE && ((!gate && num_tokens > 0) || (!dgate && num_tokens > 0))))
    return fail(SB_ERR_INVALID, "norm_out_backward: gate kind %d", gate_kind);
  if (num_tokens > 0 && (!grad_out || !y || !dy || (next && (!out || !dx))))
    return fail(SB_ERR_INVALID, "norm_out_backward: null buffer");
  NormArgs a{};
  a.y = y;
  a.y_stride = y_stride;
  a.x = out;
  a.x_stride = out_stride;
  a.grad_out = grad_out;
  a.grad_out_stride = grad_out_stride;
  a.grad_next = grad_next;
  a.grad_next_stride = grad_next_stride;
  a.weight = weight;
  a.weight_dtype = weight_dtype;
  a.gate = gate;
  a.gate_dtype = gate_dtype;
  a.gate_kind = gate_kind;
  a.gate_stride = gate_stride;
  a.scale = scale;
  a.next_weight = next_weight;
  a.next_dtype = next_dtype;
  a.dy = dy;
  a.dx = dx;
  a.dgate = dgate;
  a.num_tokens = num_tokens;
  a.d = static_cast<int32_t>(d_model);
  a.eps = eps;
  a.valid_tokens = valid_tokens;
  const bool vec = norm_vectors(
      d_model, {{grad_out, grad_out_stride, dtype}, {y, y_stride, dtype}, {dy, 0, dtype}, {grad_next, grad_next_stride, dtype},
                {next ? out : nullptr, out_stride, dtype}, {next ? dx : nullptr, 0, dtype}, {weight, 0, weight_dtype},
                {gate_kind == SB_GATE_TOKEN ? nullptr : gate, gate_kind == SB_GATE_FULL ? gate_stride : 0, gate_dtype},
                {gate_kind == SB_GATE_FULL ? dgate : nullptr, 0, gate_dtype}, {next_weight, 0, next_dtype}});
  if (const int rc = run_grad(a, dtype, true, next, vec, dweight, next ? dnext_weight : nullptr, workspace,
                              workspace_bytes, as_stream(stream)))
    return rc;
  return clear_ok();
}
