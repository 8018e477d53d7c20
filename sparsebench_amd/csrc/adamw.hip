// The AdamW step over a list of tensors, with fp32 or 8-bit states.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   g = grad * grad_scale
//   w = w (1 - lr wd) - lr / (1 - b1^s) * m / (sqrt(v / (1 - b2^s)) + eps)
//
// w is the fp32 master where there is one (the parameter is then written from
// it), else the parameter. All arithmetic in fp32, the powers in fp64.
//
// 8-bit states: blocks of 256 consecutive values with an fp32 scale each.
//   m       = c |c| scale,  c in -127 .. 127 (int8),  scale = max |m| / 127^2
//   sqrt(v) = c^2 scale,    c in 0 .. 255 (uint8),    scale = max sqrt(v) / 255^2
// The squares put the codes closer together towards zero (a value of 1% of
// its block's largest still has 25 steps below it). A value between two codes
// takes the upper one with a chance equal to its place between them in the
// root's measure: rounded to nearest, v would never move, as its relative
// change a step, about 1 - b2, is far below half a code. A v that is not zero
// never gets code 0, so that no later step divides by eps alone. The random
// bits are a hash of (seed, step, tensor, position): a call's result depends
// on its inputs alone. A NaN or an infinity in a block makes its scale, and
// so the whole block, NaN or infinite.
//
// Bound by memory: per value 16 bytes of states (4 with 8 bits) and the
// parameter, gradient and master. One workgroup takes 2048 values at a time,
// 8 a lane, so a block of 256 is half a wave. The tensors' addresses come
// with the launch (kTensorsPerLaunch of them), so nothing is kept between
// calls and a captured graph replays on the same tensors.

#include "common.hpp"

namespace sb {
namespace {

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kQuantBlock = 256;
constexpr int kValues = 8;                       // a lane's
constexpr int kThreads = 256;
constexpr int64_t kChunk = kValues * kThreads;   // values a workgroup takes at a time
constexpr int kTensorsPerLaunch = 40;            // 4 KB of kernel arguments
static_assert(kChunk % kQuantBlock == 0, "whole blocks");

struct Entry {
  void* param;
  const void* grad;
  float* master;
  void *m, *v;
  float *m_scale, *v_scale;
  int64_t numel;
  int64_t first_chunk;
  int32_t index;  // in the caller's list
  uint8_t param_dtype, grad_dtype, aligned, unused;
};

struct Table {
  Entry e[kTensorsPerLaunch];
  int64_t chunks;
  int32_t count, advance;
};
static_assert(sizeof(Table) <= 3600, "with the other arguments under 4 KB");

struct Hyper {
  const float* lr_ptr;     // device values, or null for lr and 1
  const float* grad_scale;
  int32_t* step;           // [steps done, workgroups done]
  double beta1, beta2;
  float lr, eps, weight_decay;
  uint32_t seed;
};

__device__ __forceinline__ uint32_t mix(uint32_t h) {
  h ^= h >> 16;
  h *= 0x6A09E667u;
  h ^= h >> 15;
  h *= 0xBB67AE85u;
  return h ^ (h >> 16);
}

// b^s by squaring (s > 0).
__device__ __forceinline__ double power(double b, uint32_t s) {
  double r = 1.0;
  for (; s; s >>= 1) {
    if (s & 1) r *= b;
    b *= b;
  }
  return r;
}

// Values i .. i + 7 of an array of dtype; `whole`: all eight are there and
// their address is a multiple of 16 bytes.
__device__ __forceinline__ void load8(const void* p, int dtype, int64_t i, int64_t n, bool whole, float (&out)[8]) {
  if (dtype == SB_DTYPE_F32) {
    const float* f = static_cast<const float*>(p) + i;
    if (whole) {
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(f), b = *reinterpret_cast<const f32x4_t*>(f + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = a[e], out[4 + e] = b[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = i + e < n ? f[e] : 0.0f;
    }
    return;
  }
  const uint16_t* h = static_cast<const uint16_t*>(p) + i;
  uint16_t bits[8];
  if (whole) {
    const u32x4_t a = *reinterpret_cast<const u32x4_t*>(h);
#pragma unroll
    for (int e = 0; e < 8; ++e) bits[e] = static_cast<uint16_t>(a[e / 2] >> (16 * (e & 1)));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) bits[e] = i + e < n ? h[e] : 0;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    out[e] = dtype == SB_DTYPE_BF16 ? bf16_to_f32(bits[e]) : static_cast<float>(__builtin_bit_cast(_Float16, bits[e]));
}

__device__ __forceinline__ void store8(void* p, int dtype, int64_t i, int64_t n, bool whole, const float (&v)[8]) {
  if (dtype == SB_DTYPE_F32) {
    float* f = static_cast<float*>(p) + i;
    if (whole) {
      *reinterpret_cast<f32x4_t*>(f) = f32x4_t{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4_t*>(f + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < n) f[e] = v[e];
    }
    return;
  }
  uint16_t* h = static_cast<uint16_t*>(p) + i;
  uint16_t bits[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    bits[e] = dtype == SB_DTYPE_BF16 ? f32_to_bf16(v[e]) : __builtin_bit_cast(uint16_t, static_cast<_Float16>(v[e]));
  if (whole) {
    u32x4_t a;
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = bits[2 * q] | (static_cast<uint32_t>(bits[2 * q + 1]) << 16);
    *reinterpret_cast<u32x4_t*>(h) = a;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < n) h[e] = bits[e];
  }
}

__device__ __forceinline__ void load_codes(const void* p, int64_t i, int64_t n, bool whole, uint8_t (&out)[8]) {
  const uint8_t* c = static_cast<const uint8_t*>(p) + i;
  if (whole) {
    const u32x2_t a = *reinterpret_cast<const u32x2_t*>(c);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = static_cast<uint8_t>(a[e / 4] >> (8 * (e & 3)));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = i + e < n ? c[e] : 0;
  }
}

__device__ __forceinline__ void store_codes(void* p, int64_t i, int64_t n, bool whole, const int32_t (&v)[8]) {
  uint8_t* c = static_cast<uint8_t*>(p) + i;
  if (whole) {
    u32x2_t a = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e / 4] |= static_cast<uint32_t>(v[e] & 255) << (8 * (e & 3));
    *reinterpret_cast<u32x2_t*>(c) = a;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < n) c[e] = static_cast<uint8_t>(v[e]);
  }
}

// The largest of the 32 lanes of a half wave, of values >= 0 given by their
// bits (whose order is the values', with infinity and then NaN last).
__device__ __forceinline__ float half_wave_max(uint32_t bits) {
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) bits = max(bits, static_cast<uint32_t>(__shfl_xor(static_cast<int>(bits), s)));
  return __uint_as_float(bits);
}

__device__ __forceinline__ float signed_value(uint8_t code, float scale) {
  const float c = static_cast<float>(static_cast<int8_t>(code));
  return c * fabsf(c) * scale;
}
__device__ __forceinline__ float root_value(uint8_t code, float scale) {
  const float c = static_cast<float>(code);
  return c * c * scale;
}

// The code of a value >= 0 on `inv` = 1 / scale: floor(root + bits / 2^16).
__device__ __forceinline__ int32_t code_of(float value, float inv, uint32_t bits, int32_t most) {
  const float root = __builtin_amdgcn_sqrtf(value * inv) + static_cast<float>(bits) * (1.0f / 65536.0f);
  return min(static_cast<int32_t>(root), most);
}

template <int BITS>
__global__ void __launch_bounds__(kThreads) adamw_kernel(Table t, Hyper h) {
  const uint32_t step = static_cast<uint32_t>(h.step[0]) + 1;
  const float lr = h.lr_ptr ? *h.lr_ptr : h.lr;
  const float scale = h.grad_scale ? *h.grad_scale : 1.0f;
  const float b1 = static_cast<float>(h.beta1), b2 = static_cast<float>(h.beta2);
  const float a1 = static_cast<float>(1.0 - h.beta1), a2 = static_cast<float>(1.0 - h.beta2);
  const float size = static_cast<float>(lr / (1.0 - power(h.beta1, step)));
  const float root_scale = static_cast<float>(1.0 / sqrt(1.0 - power(h.beta2, step)));
  const float keep = 1.0f - lr * h.weight_decay;
  const uint32_t step_key = mix(step * 0x9E3779B9u + h.seed);

  int at = 0;
  for (int64_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    while (at + 1 < t.count && c >= t.e[at + 1].first_chunk) ++at;
    const Entry& e = t.e[at];
    const int64_t n = e.numel;
    const int64_t i = (c - e.first_chunk) * kChunk + static_cast<int64_t>(threadIdx.x) * kValues;
    const bool whole = e.aligned && i + kValues <= n;
    float w[8], g[8], m[8], v[8];
    if (e.master) load8(e.master, SB_DTYPE_F32, i, n, whole, w);
    else load8(e.param, e.param_dtype, i, n, whole, w);
    load8(e.grad, e.grad_dtype, i, n, whole, g);
    float root[8];
    if constexpr (BITS == 32) {
      load8(e.m, SB_DTYPE_F32, i, n, whole, m);
      load8(e.v, SB_DTYPE_F32, i, n, whole, v);
    } else {
      uint8_t mc[8], vc[8];
      load_codes(e.m, i, n, whole, mc);
      load_codes(e.v, i, n, whole, vc);
      const float ms = i < n ? e.m_scale[i / kQuantBlock] : 0.0f, vs = i < n ? e.v_scale[i / kQuantBlock] : 0.0f;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        m[q] = signed_value(mc[q], ms);
        const float r = root_value(vc[q], vs);
        v[q] = r * r;
      }
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float gq = g[q] * scale;
      m[q] = b1 * m[q] + a1 * gq;
      v[q] = b2 * v[q] + a2 * gq * gq;
      root[q] = BITS == 32 ? sqrtf(v[q]) : __builtin_amdgcn_sqrtf(v[q]);
      const float under = root[q] * root_scale + h.eps;
      const float ratio = BITS == 32 ? m[q] / under : m[q] * __builtin_amdgcn_rcpf(under);
      w[q] = w[q] * keep - size * ratio;
    }
    if (e.master) store8(e.master, SB_DTYPE_F32, i, n, whole, w);
    store8(e.param, e.param_dtype, i, n, whole, w);
    if constexpr (BITS == 32) {
      store8(e.m, SB_DTYPE_F32, i, n, whole, m);
      store8(e.v, SB_DTYPE_F32, i, n, whole, v);
    } else {
      // Values past the tensor's end were loaded as zeros and so add nothing.
      uint32_t m_max = 0, v_max = 0;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        m_max = max(m_max, __float_as_uint(m[q]) & 0x7fffffffu);
        v_max = max(v_max, __float_as_uint(root[q]) & 0x7fffffffu);
      }
      float ms = half_wave_max(m_max) * (1.0f / 16129.0f);
      if (ms < 1e-37f) ms = 0.0f;  // 1 / ms would overflow: first moments under 1e-33 count as none
      const float vs = half_wave_max(v_max) * (1.0f / 65025.0f);
      const float m_inv = ms > 0.0f ? 1.0f / ms : 0.0f, v_inv = vs > 0.0f ? 1.0f / vs : 0.0f;
      const uint32_t key = mix(step_key ^ static_cast<uint32_t>(e.index)) + static_cast<uint32_t>(i >> 32);
      const uint32_t base = static_cast<uint32_t>(i) * 0x9E3779B9u + key;
      int32_t mc[8], vc[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint32_t bits = mix(base + q * 0x9E3779B9u);
        const int32_t cm = code_of(fabsf(m[q]), m_inv, bits & 0xffffu, 127);
        mc[q] = m[q] < 0.0f ? -cm : cm;
        const int32_t cv = code_of(root[q], v_inv, bits >> 16, 255);
        vc[q] = root[q] > 0.0f ? max(cv, 1) : cv;
      }
      store_codes(e.m, i, n, whole, mc);
      store_codes(e.v, i, n, whole, vc);
      if ((threadIdx.x & 31) == 0 && i < n) {
        e.m_scale[i / kQuantBlock] = ms;
        e.v_scale[i / kQuantBlock] = vs;
      }
    }
  }
  // The last workgroup of the list's last launch advances the step, after
  // every workgroup has read it.
  if (t.advance) {
    __syncthreads();
    if (threadIdx.x == 0 && atomicAdd(&h.step[1], 1) == static_cast<int32_t>(gridDim.x) - 1) {
      h.step[1] = 0;
      h.step[0] = static_cast<int32_t>(step);
    }
  }
}

// ---- the values that 8-bit states stand for ----

struct ValueEntry {
  const void* codes;
  const float* scales;
  void* out;
  int64_t numel, first_chunk;
  int32_t is_signed, aligned;
};
constexpr int kValuesPerLaunch = 64;
struct ValueTable {
  ValueEntry e[kValuesPerLaunch];
  int64_t chunks;
  int32_t count, dtype;
};
static_assert(sizeof(ValueTable) <= 3600, "under 4 KB of kernel arguments");

__global__ void __launch_bounds__(kThreads) dequantize_kernel(ValueTable t) {
  int at = 0;
  for (int64_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    while (at + 1 < t.count && c >= t.e[at + 1].first_chunk) ++at;
    const ValueEntry& e = t.e[at];
    const int64_t i = (c - e.first_chunk) * kChunk + static_cast<int64_t>(threadIdx.x) * kValues;
    if (i >= e.numel) continue;
    const bool whole = e.aligned && i + kValues <= e.numel;
    uint8_t code[8];
    load_codes(e.codes, i, e.numel, whole, code);
    const float scale = e.scales[i / kQuantBlock];
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = e.is_signed ? signed_value(code[q], scale) : root_value(code[q], scale);
    store8(e.out, t.dtype, i, e.numel, whole, v);
  }
}

bool known_dtype(int32_t d) { return d == SB_DTYPE_BF16 || d == SB_DTYPE_F16 || d == SB_DTYPE_F32; }

bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int64_t chunks_of(int64_t numel) { return (numel + kChunk - 1) / kChunk; }

// Workgroups of a launch: as many as the device holds at once, at most one per chunk.
uint32_t grid_for(int64_t chunks, int cus) {
  return static_cast<uint32_t>(std::max<int64_t>(1, std::min<int64_t>(chunks, int64_t{8} * cus)));
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_adamw(const SbAdamwTensor* tensors, int64_t count, int32_t state_bits, int32_t* step, float lr,
                        const float* lr_ptr, double beta1, double beta2, float eps, float weight_decay,
                        const float* grad_scale, uint32_t seed, void* stream) {
  if (count < 0 || (count > 0 && !tensors) || !step) return fail(SB_ERR_INVALID, "adamw: null buffer");
  if (state_bits != 32 && state_bits != 8)
    return fail(SB_ERR_INVALID, "adamw: states of 32 or 8 bits, got %d", state_bits);
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
    return fail(SB_ERR_INVALID, "adamw: betas must be in [0, 1)");
  if (count > 2147483647LL) return fail(SB_ERR_INVALID, "adamw: too many tensors");
  for (int64_t i = 0; i < count; ++i) {
    const SbAdamwTensor& a = tensors[i];
    if (a.numel < 0) return fail(SB_ERR_INVALID, "adamw: negative length");
    if (a.numel == 0) continue;
    if (!a.param || !a.grad || !a.exp_avg || !a.exp_avg_sq || (state_bits == 8 && (!a.exp_avg_scale || !a.exp_avg_sq_scale)))
      return fail(SB_ERR_INVALID, "adamw: null buffer");
    if (!known_dtype(a.param_dtype) || !known_dtype(a.grad_dtype))
      return fail(SB_ERR_INVALID, "adamw: unsupported dtype code");
  }
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  const Hyper h{lr_ptr, grad_scale, step, beta1, beta2, lr, eps, weight_decay, seed};
  int64_t i = 0;
  do {
    Table t{};
    for (; i < count && t.count < kTensorsPerLaunch; ++i) {
      const SbAdamwTensor& a = tensors[i];
      if (a.numel == 0) continue;
      const bool wide_states = state_bits == 32 ? aligned16(a.exp_avg) && aligned16(a.exp_avg_sq)
                                                : aligned_to(a.exp_avg, 8) && aligned_to(a.exp_avg_sq, 8);
      const bool wide = aligned16(a.param) && aligned16(a.grad) && (!a.master || aligned16(a.master)) && wide_states;
      t.e[t.count++] = Entry{a.param, a.grad, a.master, a.exp_avg, a.exp_avg_sq, a.exp_avg_scale, a.exp_avg_sq_scale,
                             a.numel, t.chunks, static_cast<int32_t>(i), static_cast<uint8_t>(a.param_dtype),
                             static_cast<uint8_t>(a.grad_dtype), static_cast<uint8_t>(wide), 0};
      t.chunks += chunks_of(a.numel);
    }
    t.advance = i == count;
    if (t.count == 0 && !t.advance) continue;
    const uint32_t grid = grid_for(t.chunks, cus);
    if (state_bits == 32) adamw_kernel<32><<<grid, kThreads, 0, as_stream(stream)>>>(t, h);
    else adamw_kernel<8><<<grid, kThreads, 0, as_stream(stream)>>>(t, h);
    if (const int rc = check_launch("adamw")) return rc;
  } while (i < count);
  return clear_ok();
}

extern "C" int sb_dequantize(const SbQuantized* tensors, int64_t count, int32_t out_dtype, void* stream) {
  if (count < 0 || (count > 0 && !tensors)) return fail(SB_ERR_INVALID, "dequantize: null buffer");
  if (!known_dtype(out_dtype)) return fail(SB_ERR_INVALID, "dequantize: unsupported dtype code %d", out_dtype);
  for (int64_t i = 0; i < count; ++i) {
    if (tensors[i].numel < 0) return fail(SB_ERR_INVALID, "dequantize: negative length");
    if (tensors[i].numel > 0 && (!tensors[i].codes || !tensors[i].scales || !tensors[i].out))
      return fail(SB_ERR_INVALID, "dequantize: null buffer");
  }
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  for (int64_t i = 0; i < count;) {
    ValueTable t{};
    t.dtype = out_dtype;
    for (; i < count && t.count < kValuesPerLaunch; ++i) {
      const SbQuantized& a = tensors[i];
      if (a.numel == 0) continue;
      t.e[t.count++] = ValueEntry{a.codes, a.scales, a.out, a.numel, t.chunks, static_cast<int32_t>(a.is_signed != 0),
                                  aligned_to(a.codes, 8) && aligned16(a.out)};
      t.chunks += chunks_of(a.numel);
    }
    if (t.count == 0) continue;
    dequantize_kernel<<<grid_for(t.chunks, cus), kThreads, 0, as_stream(stream)>>>(t);
    if (const int rc = check_launch("dequantize")) return rc;
  }
  return clear_ok();
}
