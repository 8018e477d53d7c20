// What the norms' forward and backward kernels share.
//
//   n(v)     v / sqrt(mean(v^2) + eps) over a row of D values
//   norm_in  next = v n(x)
//   norm_out out = x + s g w n(y);  next = v n(out), of out as it is rounded
//
// A group of G threads takes a row at a time, and always the same columns, so
// the weights stay in registers over all its rows and the weights' gradients
// are summed there. The row itself stays in registers too, and is read once, up to
// D = 8192 forward and 4096 backward. Beyond, a group of 1024 threads leaves a thread 128
// registers, and part of the row and the weights goes through scratch memory (bytes a
// lane, with the next norm, forward 284 to 476; backward 96 to 184 up to D = 8192, 512 to
// 680 up to 16384, 1472 to 1960 beyond): norm.hip and norm_grad.hip have the times.
#pragma once

#include <initializer_list>

#include "common.hpp"

namespace sb {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct NormArgs {
  // Forward: y, x -> out, next. Backward: grad_out, grad_next, y, x (norm_out's
  // out, norm_in's x) -> dy, dx, dgate, and the partial sums of the weights' gradients.
  const void *y, *x, *grad_out, *grad_next;
  const void *weight, *gate, *next_weight;
  void *out, *next;  // forward
  void *dy, *dx, *dgate;
  float* partial;    // [workgroups][2][D]: the weight's, then the next weight's
  const int32_t* valid_tokens;
  int64_t y_stride, x_stride, grad_out_stride, grad_next_stride, gate_stride;
  int64_t num_tokens;
  int32_t d, weight_dtype, gate_dtype, next_dtype, gate_kind;
  float scale, eps, inv_d;
};

// One value of an array of a dtype known at run time (uniform), as fp32.
__device__ __forceinline__ float load_as_f32(const void* p, int32_t dtype, int64_t i) {
  if (dtype == SB_DTYPE_F32) return static_cast<const float*>(p)[i];
  const uint16_t bits = static_cast<const uint16_t*>(p)[i];
  return dtype == SB_DTYPE_BF16 ? bf16_to_f32(bits) : static_cast<float>(__builtin_bit_cast(_Float16, bits));
}

// An fp32 result rounded to fp16: in two steps, as a result that was stored in fp32 in
// between. Without the barrier the compiler fuses the last operation and the conversion
// into one rounding, which takes other values at about one in 2^13.
__device__ __forceinline__ uint16_t f32_to_f16(float v) {
  asm("" : "+v"(v));
  return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

__device__ __forceinline__ void store_as(void* p, int32_t dtype, int64_t i, float v) {
  if (dtype == SB_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == SB_DTYPE_BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
  else static_cast<uint16_t*>(p)[i] = f32_to_f16(v);
}

template <int DTYPE>
__device__ __forceinline__ float rounded(float v) {
  if constexpr (DTYPE == SB_DTYPE_F32) return v;
  else if constexpr (DTYPE == SB_DTYPE_BF16) return bf16_to_f32(f32_to_bf16(v));
  else return static_cast<float>(__builtin_bit_cast(_Float16, f32_to_f16(v)));
}

// A row's share of a thread, 8 NCH values. VEC: chunks of 8 consecutive values
// (D a multiple of 8, every address a multiple of 16 bytes); otherwise every
// G-th value, so that the lanes of a load are neighbours in any case.
template <int G, int NCH, bool VEC>
struct Share {
  static constexpr int kValues = 8 * NCH;
  __device__ __forceinline__ static int column(int i, int t) {
    return VEC ? (i / 8) * (8 * G) + 8 * t + i % 8 : i * G + t;
  }
};

// The row's values that belong to thread t, 0 past its end: loaded, and then taken,
// so that the next row's loads may be under way while one is worked on.
template <class S, int DTYPE, bool VEC>
struct RowRegs {
  static constexpr int kPerVector = DTYPE == SB_DTYPE_F32 ? 4 : 8;
  std::conditional_t<VEC, u32x4_t, float> raw[VEC ? S::kValues / kPerVector : S::kValues];

  __device__ __forceinline__ void load(const void* row, int d, int t) {
    if constexpr (VEC) {
#pragma unroll
      for (int c = 0; c < S::kValues / 8; ++c) {
        const int at = S::column(8 * c, t);
        const bool there = at < d;
        const auto* p = reinterpret_cast<const u32x4_t*>(static_cast<const uint8_t*>(row) +
                                                         (there ? at : 0) * (DTYPE == SB_DTYPE_F32 ? 4 : 2));
#pragma unroll
        for (int q = 0; q < 8 / kPerVector; ++q) {
          const u32x4_t a = p[q];
          raw[c * (8 / kPerVector) + q] = there ? a : u32x4_t{0u, 0u, 0u, 0u};
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < S::kValues; ++i) {
        const int at = S::column(i, t);
        raw[i] = at < d ? load_as_f32(row, DTYPE, at) : 0.0f;
      }
    }
  }
  __device__ __forceinline__ void take(float (&v)[S::kValues]) const {
#pragma unroll
    for (int i = 0; i < S::kValues; ++i) {
      if constexpr (!VEC) {
        v[i] = raw[i];
      } else if constexpr (DTYPE == SB_DTYPE_F32) {
        v[i] = __uint_as_float(raw[i / 4][i % 4]);
      } else {
        const uint32_t pair = raw[i / 8][i % 8 / 2];
        if constexpr (DTYPE == SB_DTYPE_BF16) v[i] = __uint_as_float(i & 1 ? pair & 0xffff0000u : pair << 16);
        else v[i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(pair >> (16 * (i & 1)))));
      }
    }
  }
};

template <class S, int DTYPE, bool VEC>
__device__ __forceinline__ void load_row(const void* row, int d, int t, float (&v)[S::kValues]) {
  RowRegs<S, DTYPE, VEC> r;
  r.load(row, d, t);
  r.take(v);
}

template <class S, int DTYPE, bool VEC>
__device__ __forceinline__ void store_row(void* row, int d, int t, const float (&v)[S::kValues]) {
  if constexpr (VEC) {
#pragma unroll
    for (int c = 0; c < S::kValues / 8; ++c) {
      const int at = S::column(8 * c, t);
      if (at >= d) continue;
      if constexpr (DTYPE == SB_DTYPE_F32) {
        f32x4_t* p = reinterpret_cast<f32x4_t*>(static_cast<float*>(row) + at);
        p[0] = f32x4_t{v[8 * c], v[8 * c + 1], v[8 * c + 2], v[8 * c + 3]};
        p[1] = f32x4_t{v[8 * c + 4], v[8 * c + 5], v[8 * c + 6], v[8 * c + 7]};
      } else {
        u32x4_t a;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float lo = v[8 * c + 2 * q], hi = v[8 * c + 2 * q + 1];
          if constexpr (DTYPE == SB_DTYPE_BF16) {
            a[q] = pack_bf16x2(lo, hi);
          } else {
            a[q] = f32_to_f16(lo) | static_cast<uint32_t>(f32_to_f16(hi)) << 16;
          }
        }
        *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(row) + at) = a;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < S::kValues; ++i) {
      const int at = S::column(i, t);
      if (at < d) store_as(row, DTYPE, at, v[i]);
    }
  }
}

// f(integral_constant of a dtype known at run time, uniform).
template <class F>
__device__ __forceinline__ void by_dtype(int32_t dtype, F&& f) {
  if (dtype == SB_DTYPE_BF16) f(std::integral_constant<int, SB_DTYPE_BF16>{});
  else if (dtype == SB_DTYPE_F32) f(std::integral_constant<int, SB_DTYPE_F32>{});
  else f(std::integral_constant<int, SB_DTYPE_F16>{});
}

// A row's or a [D] vector's share in a dtype known at run time (weights, gates);
// `otherwise` where there is none, 0 past the end.
template <class S, bool VEC>
__device__ __forceinline__ void load_vector(const void* p, int32_t dtype, int64_t first, int d, int t, float otherwise,
                                            float (&v)[S::kValues]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < S::kValues; ++i) v[i] = otherwise;
    return;
  }
  by_dtype(dtype, [&](auto type) {
    constexpr int kType = decltype(type)::value;
    load_row<S, kType, VEC>(static_cast<const uint8_t*>(p) + first * (kType == SB_DTYPE_F32 ? 4 : 2), d, t, v);
  });
}

// The sum over the wave's lanes, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
  const auto dpp = [&](auto ctrl) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v += dpp(std::integral_constant<int, 0xB1>{});   // quad_perm [1, 0, 3, 2]
  v += dpp(std::integral_constant<int, 0x4E>{});   // quad_perm [2, 3, 0, 1]
  v += dpp(std::integral_constant<int, 0x141>{});  // row_half_mirror
  v += dpp(std::integral_constant<int, 0x140>{});  // row_mirror
  const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  v = __int_as_float(rows[0]) + __int_as_float(rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return __int_as_float(halves[0]) + __int_as_float(halves[1]);
}

// Sums of N values over a row's group. Two buffers in turn: a wave that writes
// one again has passed the barrier that every reader of it came to after reading.
template <int G, int N>
struct GroupSum {
  static constexpr int kWaves = G / 64;
  float (*lds)[kWaves > 1 ? kWaves : 1][N];
  int turn = 0;
  __device__ __forceinline__ explicit GroupSum(float (*buffers)[kWaves > 1 ? kWaves : 1][N]) : lds(buffers) {}
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (kWaves > 1) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) lds[turn][wave][i] = v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.0f;
      for (int w = 0; w < kWaves; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += lds[turn][w][i];
      turn ^= 1;
    }
  }
};

// f(G, NCH, VEC as integral constants) for rows of d values; false if d is too long.
// Backward rows take more registers a value, so that fewer are a thread's.
template <bool GRAD, class F>
bool with_norm_form(int64_t d, bool vec, F&& f) {
  auto form = [&](auto g, auto chunks) {
    if (d > int64_t{8} * decltype(g)::value * decltype(chunks)::value) return false;
    if (vec) f(g, chunks, std::true_type{});
    else f(g, chunks, std::false_type{});
    return true;
  };
  using std::integral_constant;
  constexpr integral_constant<int, 64> wave{};
  constexpr integral_constant<int, 256> four{};
  constexpr integral_constant<int, 1024> sixteen{};
  constexpr integral_constant<int, 1> one{};
  constexpr integral_constant<int, 2> two{};
  constexpr integral_constant<int, 4> quad{};
  if (form(wave, one) || form(wave, two)) return true;
  if constexpr (GRAD) return form(four, one) || form(four, two) || form(sixteen, one) || form(sixteen, two) || form(sixteen, quad);
  else return form(wave, quad) || form(four, two) || form(four, quad) || form(sixteen, quad);
}

constexpr int64_t kNormMaxD = 32768;

// The workgroup of a form: one row's group, or four rows' waves.
constexpr int norm_threads(int g) { return g < 256 ? 256 : g; }

template <class F>
int with_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case SB_DTYPE_BF16: return f(std::integral_constant<int, SB_DTYPE_BF16>{});
    case SB_DTYPE_F16: return f(std::integral_constant<int, SB_DTYPE_F16>{});
    default: return f(std::integral_constant<int, SB_DTYPE_F32>{});
  }
}

// Where vectors of 8 may be used: every row of every operand starts at a multiple of 16 bytes.
struct NormOperand {
  const void* p;  // null: not there
  int64_t stride;
  int32_t dtype;
};
inline bool norm_vectors(int64_t d, std::initializer_list<NormOperand> operands) {
  bool ok = d % 8 == 0;
  for (const NormOperand& o : operands)
    ok = ok && (!o.p || (aligned16(o.p) && o.stride * (o.dtype == SB_DTYPE_F32 ? 4 : 2) % 16 == 0));
  return ok;
}

int check_norm(const char* what, int32_t dtype, int64_t num_tokens, int64_t d, float eps,
               std::initializer_list<int32_t> dtypes, std::initializer_list<int64_t> strides);

}  // namespace sb
