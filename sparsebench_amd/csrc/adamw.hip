// The AdamW step over a list of tensors, with fp32 or 8-bit states.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   g = grad * grad_scale
//   w = w (1 - lr wd) - lr / (1 - b1^s) * m / (sqrt(v / (1 - b2^s)) + eps)
//
// w is the fp32 master where there is one (the parameter is then written from
// it), else the parameter. All arithmetic in fp32, the powers in fp64.
//
// 8-bit states: blocks of 256 consecutive values with an fp32 scale each.
//   m       = c |c| scale,  c in -127 .. 127 (int8),  scale = max |m| fp32(1 / 127^2)
//   sqrt(v) = c^2 scale,    c in 0 .. 255 (uint8),    scale = max sqrt(v) fp32(1 / 255^2)
//   |c|     = floor(sqrt(value / scale) + 16 random bits / 2^16)
// These operations, and the moments' before them, are each rounded to nearest:
// a floor passes on the last bit as a whole code, so that over steps another
// order of roundings would give other states (and weights 6e-6 apart after 4).
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
// parameter, gradient and master: 200M bf16 values with masters 1190 us, 4.7
// TB/s, where a copy reaches 5.1; with 8-bit states and no masters 435 us, 4.6
// TB/s (there the arithmetic takes 345 us alone).
// A grid of 8 workgroups per CU that walk the chunks: with one workgroup per
// chunk the atomic that counts them is the bound (1212 and 1142 us).
// One workgroup takes 2048 values at a time,
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
  int32_t index;  // in the caller's list
  uint8_t param_dtype, grad_dtype, aligned, unused;
};

// The entries' first chunks stand apart: kernel arguments may lie in host
// memory, where each read that waits for another costs a microsecond or more,
// and one read by all lanes finds a chunk's tensor (a walk over the entries
// took a step of 60 small tensors, two launches, from 13 us to 31).
struct Table {
  int64_t first_chunk[kTensorsPerLaunch];
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

__host__ __device__ __forceinline__ int64_t chunks_of(int64_t numel) { return (numel + kChunk - 1) / kChunk; }

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

__device__ __forceinline__ void store_codes(void* p, int64_t i, int64_t n, bool whole, const uint32_t (&v)[8]) {
  uint8_t* c = static_cast<uint8_t*>(p) + i;
  if (whole) {
    u32x2_t a = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e / 4] |= (v[e] & 255u) << (8 * (e & 3));
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
  auto with = [&](uint32_t other) { bits = max(bits, other); };
  const auto dpp = [&](auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(bits), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  with(dpp(std::integral_constant<int, 0xB1>{}));   // quad_perm [1, 0, 3, 2]
  with(dpp(std::integral_constant<int, 0x4E>{}));   // quad_perm [2, 3, 0, 1]
  with(dpp(std::integral_constant<int, 0x141>{}));  // row_half_mirror
  with(dpp(std::integral_constant<int, 0x140>{}));  // row_mirror
  with(static_cast<uint32_t>(__shfl_xor(static_cast<int>(bits), 16)));
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

// The code of a value >= 0 by the rule, each operation rounded to nearest:
// floor(sqrt(value / scale) + bits / 2^16), at most `most`.
__device__ __forceinline__ uint32_t code_of(float value, float scale, uint32_t bits, float most) {
#pragma clang fp contract(off)
  const float root = sqrtf(value / (scale > 0.0f ? scale : 1.0f));
  return static_cast<uint32_t>(fminf(root + static_cast<float>(bits) * (1.0f / 65536.0f), most));
}

// 2^16 times the same before its floor, near enough: inv is about 2^32 / scale.
__device__ __forceinline__ uint32_t near_code(float value, float inv, uint32_t bits) {
  return static_cast<uint32_t>(__builtin_amdgcn_sqrtf(value * inv)) + bits;
}
// How far near_code and the rule's sum may lie apart, in units of 2^-16 of a code:
// 2^-23 of a root is 1 of them for 127 and 2 for 255. In 2^-23 of the root: 1 for
// near_code's square root (1 ulp), 0.75 for inv and its product (1.5 under the
// root), as much again for a second moment, which is a square root itself, and
// 1.25 for the rule's own roundings; then less than 1 unit from the conversion.
// That is less than 4 and 9 units: further than so from a border the floors agree.
constexpr uint32_t kFirstOff = 5, kSecondOff = 10;
__device__ __forceinline__ bool near_border(uint32_t code, uint32_t off) { return ((code + off) & 0xffffu) <= 2 * off; }

struct Coefficients {
  float scale, b1, a1, b2, a2, size, root_scale, eps, keep;
  uint32_t step_key;
};

// The moments' update and the weights' of 8 values. 8-bit states depend on a
// floor, where the last bit counts: there each operation is rounded on its own.
template <int BITS>
__device__ __forceinline__ void update(const Coefficients& k, float (&w)[8], const float (&g)[8], float (&m)[8],
                                       float (&v)[8], float (&root)[8]) {
  uint32_t least = 0xffffffffu;  // the smallest v that is not 0, by its bits less 1
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float gq = g[q] * k.scale;
    if constexpr (BITS == 32) {
      m[q] = fmaf(k.a1, gq, k.b1 * m[q]);
      v[q] = fmaf(k.a2 * gq, gq, k.b2 * v[q]);
    } else {
#pragma clang fp contract(off)
      m[q] = k.b1 * m[q] + k.a1 * gq;
      v[q] = k.b2 * v[q] + k.a2 * gq * gq;
    }
    least = min(least, __float_as_uint(v[q]) - 1u);
    root[q] = __builtin_amdgcn_sqrtf(v[q]);  // to 1 ulp, but 0 for subnormals
  }
  // Gradients under 1e-17: a root of 0 would leave eps alone, however small.
  if (__builtin_expect(least < 0x0d800000u - 1u, 0)) {  // 2^-100
#pragma unroll
    for (int q = 0; q < 8; ++q) root[q] = sqrtf(v[q]);
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float ratio = m[q] * __builtin_amdgcn_rcpf(fmaf(root[q], k.root_scale, k.eps));
    w[q] = fmaf(-k.size, ratio, w[q] * k.keep);
  }
}

// The 8-bit states of a lane's 8 values from i on: codes, and the half wave's
// scales. The rule's divisions and square roots would take longer than the rest of
// the step (636 us for 200M values with no masters, 430 this way), so a code comes
// from an approximation, and by the rule where that lies too near a border to
// tell (one value in 4000, so one wave in 50 at each). All 16 of a lane by the
// rule where one of them is near a border: 463 us, and 112 registers against 94.
__device__ __forceinline__ void encode(const Coefficients& k, const Entry& e, int64_t i, const float (&m)[8],
                                       const float (&v)[8], const float (&root)[8], uint32_t (&mc)[8],
                                       uint32_t (&vc)[8], float* m_scale, float* v_scale) {
  uint32_t m_max = 0, v_max = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    m_max = max(m_max, __float_as_uint(m[q]) & 0x7fffffffu);
    v_max = max(v_max, __float_as_uint(v[q]) & 0x7fffffffu);
  }
  const float ms = half_wave_max(m_max) * (1.0f / 16129.0f), vs = sqrtf(half_wave_max(v_max)) * (1.0f / 65025.0f);
  const float m_inv = ms > 0.0f ? __builtin_amdgcn_rcpf(ms) * 0x1p32f : 0.0f;
  const float v_inv = vs > 0.0f ? __builtin_amdgcn_rcpf(vs) * 0x1p32f : 0.0f;
  // Small scales' reciprocals overflow. (Without a scale both ways give code 0.)
  const bool by_rule = !(ms == 0.0f || ms > 0x1p-90f) || !(vs == 0.0f || vs > 0x1p-90f);
  const uint32_t key = mix(k.step_key ^ static_cast<uint32_t>(e.index)) + static_cast<uint32_t>(i >> 32);
  const uint32_t base = static_cast<uint32_t>(i) * 0x9E3779B9u + key;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const uint32_t bits = mix(base + q * 0x9E3779B9u);
    const uint32_t cm = near_code(fabsf(m[q]), m_inv, bits & 0xffffu), cv = near_code(root[q], v_inv, bits >> 16);
    mc[q] = min(cm >> 16, 127u);
    vc[q] = min(cv >> 16, 255u);
    if (__builtin_expect(near_border(cm, kFirstOff) || by_rule, 0))
      mc[q] = code_of(fabsf(m[q]), ms, bits & 0xffffu, 127.0f);
    if (__builtin_expect(near_border(cv, kSecondOff) || by_rule, 0))
      vc[q] = code_of(sqrtf(v[q]), vs, bits >> 16, 255.0f);
    const uint32_t sign = static_cast<uint32_t>(__float_as_int(m[q]) >> 31);
    mc[q] = (mc[q] ^ sign) - sign;
    vc[q] = max(vc[q], v[q] > 0.0f ? 1u : 0u);
  }
  *m_scale = ms;
  *v_scale = vs;
}

// A lane's 8 values from i on where some of them, or of another lane's, are
// past the tensor's end, or its arrays are not aligned: any types.
template <int BITS>
__device__ __forceinline__ void step_edge(const Coefficients& k, const Entry& e, int64_t i) {
  const int64_t n = e.numel;
  const bool whole = e.aligned && i + kValues <= n;
  float w[8], g[8], m[8], v[8], root[8];
  if (e.master) load8(e.master, SB_DTYPE_F32, i, n, whole, w);
  else load8(e.param, e.param_dtype, i, n, whole, w);
  load8(e.grad, e.grad_dtype, i, n, whole, g);
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
  update<BITS>(k, w, g, m, v, root);
  if (e.master) store8(e.master, SB_DTYPE_F32, i, n, whole, w);
  store8(e.param, e.param_dtype, i, n, whole, w);
  if constexpr (BITS == 32) {
    store8(e.m, SB_DTYPE_F32, i, n, whole, m);
    store8(e.v, SB_DTYPE_F32, i, n, whole, v);
  } else {
    // Values past the tensor's end were loaded as zeros and so add nothing.
    uint32_t mc[8], vc[8];
    float ms, vs;
    encode(k, e, i, m, v, root, mc, vc, &ms, &vs);
    store_codes(e.m, i, n, whole, mc);
    store_codes(e.v, i, n, whole, vc);
    if ((threadIdx.x & 31) == 0 && i < n) {
      e.m_scale[i / kQuantBlock] = ms;
      e.v_scale[i / kQuantBlock] = vs;
    }
  }
}

// N aligned values of dtype D (8, or 4 of 16 or 32 bits), as loaded and as floats.
// Runs of up to 16 bytes a lane, which whole instructions join to whole cache
// lines, go past the caches: nothing is read again (200M values with masters:
// 1262 us with plain accesses, 1190 this way; halves of lines so: 1700).
template <int D, int N>
struct Raw {
  static constexpr int kBytes = N * (D == SB_DTYPE_F32 ? 4 : 2);
  uint32_t a[kBytes / 4];
  __device__ __forceinline__ explicit Raw(const void* p, int64_t i) {
    const uint8_t* at = static_cast<const uint8_t*>(p) + i * (kBytes / N);
    if constexpr (kBytes == 8) {
      const u32x2_t q = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(at));
      a[0] = q[0], a[1] = q[1];
    } else {
#pragma unroll
      for (int b = 0; b < kBytes / 16; ++b) {
        const auto* from = reinterpret_cast<const u32x4_t*>(at) + b;
        const u32x4_t q = kBytes == 16 ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
        for (int e = 0; e < 4; ++e) a[4 * b + e] = q[e];
      }
    }
  }
  __device__ __forceinline__ void get(float* out) const {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if constexpr (D == SB_DTYPE_F32) {
        out[e] = __uint_as_float(a[e]);
      } else if constexpr (D == SB_DTYPE_BF16) {
        out[e] = __uint_as_float(e & 1 ? a[e / 2] & 0xffff0000u : a[e / 2] << 16);
      } else {
        out[e] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(a[e / 2] >> (16 * (e & 1)))));
      }
    }
  }
};

template <int D, int N>
__device__ __forceinline__ void put(void* p, int64_t i, const float* v) {
  constexpr int kBytes = N * (D == SB_DTYPE_F32 ? 4 : 2);
  uint32_t a[kBytes / 4];
#pragma unroll
  for (int e = 0; e < kBytes / 4; ++e) {
    if constexpr (D == SB_DTYPE_F32) {
      a[e] = __float_as_uint(v[e]);
    } else if constexpr (D == SB_DTYPE_BF16) {
      a[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
    } else {
      a[e] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(v[2 * e])) |
             static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(v[2 * e + 1]))) << 16;
    }
  }
  uint8_t* at = static_cast<uint8_t*>(p) + i * (kBytes / N);
  if constexpr (kBytes == 8) {
    __builtin_nontemporal_store(u32x2_t{a[0], a[1]}, reinterpret_cast<u32x2_t*>(at));
  } else {
#pragma unroll
    for (int b = 0; b < kBytes / 16; ++b) {
      const u32x4_t q = {a[4 * b], a[4 * b + 1], a[4 * b + 2], a[4 * b + 3]};
      if constexpr (kBytes == 16) __builtin_nontemporal_store(q, reinterpret_cast<u32x4_t*>(at));
      else reinterpret_cast<u32x4_t*>(at)[b] = q;
    }
  }
}

// A chunk of aligned values that are all there: types known, so that every
// load is under way before the first is waited for. `start` is the chunk's
// first value. fp32 states: a lane's 8 values are two runs of 4, a wave's 256
// values apart, so that each instruction's lanes cover whole cache lines.
template <int P, int G, bool MASTER>
__device__ __forceinline__ void step_whole32(const Coefficients& k, const Entry& e, int64_t start) {
  constexpr int W = MASTER ? SB_DTYPE_F32 : P;
  const void* from = MASTER ? static_cast<const void*>(e.master) : e.param;
  const int64_t i = start + (threadIdx.x >> 6) * 512 + (threadIdx.x & 63) * 4, j = i + 256;
  const Raw<W, 4> w0(from, i), w1(from, j);
  const Raw<G, 4> g0(e.grad, i), g1(e.grad, j);
  const Raw<SB_DTYPE_F32, 4> m0(e.m, i), m1(e.m, j), v0(e.v, i), v1(e.v, j);
  float w[8], g[8], m[8], v[8], root[8];
  w0.get(w), w1.get(w + 4);
  g0.get(g), g1.get(g + 4);
  m0.get(m), m1.get(m + 4);
  v0.get(v), v1.get(v + 4);
  update<32>(k, w, g, m, v, root);
  put<SB_DTYPE_F32, 4>(e.m, i, m), put<SB_DTYPE_F32, 4>(e.m, j, m + 4);
  put<SB_DTYPE_F32, 4>(e.v, i, v), put<SB_DTYPE_F32, 4>(e.v, j, v + 4);
  if constexpr (MASTER) put<SB_DTYPE_F32, 4>(e.master, i, w), put<SB_DTYPE_F32, 4>(e.master, j, w + 4);
  put<P, 4>(e.param, i, w), put<P, 4>(e.param, j, w + 4);
}

template <int P, int G, bool MASTER>
__device__ __forceinline__ void step_whole8(const Coefficients& k, const Entry& e, int64_t start) {
  const int64_t i = start + static_cast<int64_t>(threadIdx.x) * kValues;
  const Raw<MASTER ? SB_DTYPE_F32 : P, 8> rw(MASTER ? static_cast<const void*>(e.master) : e.param, i);
  const Raw<G, 8> rg(e.grad, i);
  auto* m_at = reinterpret_cast<u32x2_t*>(static_cast<uint8_t*>(e.m) + i);
  auto* v_at = reinterpret_cast<u32x2_t*>(static_cast<uint8_t*>(e.v) + i);
  const u32x2_t cm = *m_at, cv = *v_at;
  float ms = e.m_scale[i / kQuantBlock], vs = e.v_scale[i / kQuantBlock];
  float w[8], g[8], m[8], v[8], root[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    m[q] = signed_value(static_cast<uint8_t>(cm[q / 4] >> (8 * (q & 3))), ms);
    const float r = root_value(static_cast<uint8_t>(cv[q / 4] >> (8 * (q & 3))), vs);
    v[q] = r * r;
  }
  rw.get(w);
  rg.get(g);
  update<8>(k, w, g, m, v, root);
  uint32_t mc[8], vc[8];
  encode(k, e, i, m, v, root, mc, vc, &ms, &vs);
  u32x2_t om, ov;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    om[h] = __builtin_amdgcn_perm(mc[4 * h + 3], mc[4 * h + 2], 0x0c0c0400) << 16 |
            __builtin_amdgcn_perm(mc[4 * h + 1], mc[4 * h], 0x0c0c0400);
    ov[h] = vc[4 * h] | vc[4 * h + 1] << 8 | vc[4 * h + 2] << 16 | vc[4 * h + 3] << 24;
  }
  *m_at = om;
  *v_at = ov;
  if ((threadIdx.x & 31) == 0) {
    e.m_scale[i / kQuantBlock] = ms;
    e.v_scale[i / kQuantBlock] = vs;
  }
  if constexpr (MASTER) put<SB_DTYPE_F32, 8>(e.master, i, w);
  put<P, 8>(e.param, i, w);
}

template <int BITS>
__global__ void __launch_bounds__(kThreads) adamw_kernel(Table t, Hyper h) {
  const int lane = threadIdx.x & 63;
  const int64_t first = lane < t.count ? t.first_chunk[min(lane, kTensorsPerLaunch - 1)] : INT64_MAX;
  const uint32_t step = static_cast<uint32_t>(h.step[0]) + 1;
  const float lr = h.lr_ptr ? *h.lr_ptr : h.lr;
  Coefficients k;
  k.scale = h.grad_scale ? *h.grad_scale : 1.0f;
  k.b1 = static_cast<float>(h.beta1), k.a1 = static_cast<float>(1.0 - h.beta1);
  k.b2 = static_cast<float>(h.beta2), k.a2 = static_cast<float>(1.0 - h.beta2);
  k.size = static_cast<float>(lr / (1.0 - power(h.beta1, step)));
  k.root_scale = static_cast<float>(1.0 / sqrt(1.0 - power(h.beta2, step)));
  k.eps = h.eps;
  k.keep = 1.0f - lr * h.weight_decay;
  k.step_key = mix(step * 0x9E3779B9u + h.seed);

  for (int64_t c = blockIdx.x; c < t.chunks;) {
    const int at = __builtin_popcountll(__ballot(first <= c)) - 1;  // the last entry that starts at or before c
    const Entry e = t.e[at];
    // This workgroup's chunks c .. of the entry: the whole ones, then its last one.
    const int64_t base = t.first_chunk[at];
    const int64_t whole = base + (e.aligned ? e.numel / kChunk : 0), end = base + chunks_of(e.numel);
    auto run = [&](auto p, auto g, auto master) {
      for (; c < whole; c += gridDim.x) {
        if constexpr (BITS == 32)
          step_whole32<decltype(p)::value, decltype(g)::value, decltype(master)::value>(k, e, (c - base) * kChunk);
        else
          step_whole8<decltype(p)::value, decltype(g)::value, decltype(master)::value>(k, e, (c - base) * kChunk);
      }
    };
    auto by_master = [&](auto p, auto g) {
      if (e.master) run(p, g, std::true_type{});
      else run(p, g, std::false_type{});
    };
    auto by_grad = [&](auto p) {
      if (e.grad_dtype == SB_DTYPE_F32) by_master(p, std::integral_constant<int, SB_DTYPE_F32>{});
      else if (e.grad_dtype == SB_DTYPE_BF16) by_master(p, std::integral_constant<int, SB_DTYPE_BF16>{});
      else by_master(p, std::integral_constant<int, SB_DTYPE_F16>{});
    };
    if (c < whole) {
      if (e.param_dtype == SB_DTYPE_F32) by_grad(std::integral_constant<int, SB_DTYPE_F32>{});
      else if (e.param_dtype == SB_DTYPE_BF16) by_grad(std::integral_constant<int, SB_DTYPE_BF16>{});
      else by_grad(std::integral_constant<int, SB_DTYPE_F16>{});
    }
    for (; c < end; c += gridDim.x)
      step_edge<BITS>(k, e, (c - base) * kChunk + static_cast<int64_t>(threadIdx.x) * kValues);
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
  int64_t numel;
  int32_t is_signed, aligned;
};
constexpr int kValuesPerLaunch = 64;
struct ValueTable {
  int64_t first_chunk[kValuesPerLaunch];
  ValueEntry e[kValuesPerLaunch];
  int64_t chunks;
  int32_t count, dtype;
};
static_assert(sizeof(ValueTable) <= 3600, "under 4 KB of kernel arguments");

__global__ void __launch_bounds__(kThreads) dequantize_kernel(ValueTable t) {
  const int lane = threadIdx.x & 63;
  const int64_t first = lane < t.count ? t.first_chunk[lane] : INT64_MAX;
  for (int64_t c = blockIdx.x; c < t.chunks;) {
    const int at = __builtin_popcountll(__ballot(first <= c)) - 1;
    const ValueEntry e = t.e[at];
    const int64_t base = t.first_chunk[at], end = base + chunks_of(e.numel);
    for (; c < end; c += gridDim.x) {
      const int64_t i = (c - base) * kChunk + static_cast<int64_t>(threadIdx.x) * kValues;
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
}

bool known_dtype(int32_t d) { return d == SB_DTYPE_BF16 || d == SB_DTYPE_F16 || d == SB_DTYPE_F32; }

bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

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
      t.first_chunk[t.count] = t.chunks;
      t.e[t.count++] = Entry{a.param, a.grad, a.master, a.exp_avg, a.exp_avg_sq, a.exp_avg_scale, a.exp_avg_sq_scale,
                             a.numel, static_cast<int32_t>(i), static_cast<uint8_t>(a.param_dtype),
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
      t.first_chunk[t.count] = t.chunks;
      t.e[t.count++] = ValueEntry{a.codes, a.scales, a.out, a.numel, static_cast<int32_t>(a.is_signed != 0),
                                  aligned_to(a.codes, 8) && aligned16(a.out)};
      t.chunks += chunks_of(a.numel);
    }
    if (t.count == 0) continue;
    dequantize_kernel<<<grid_for(t.chunks, cus), kThreads, 0, as_stream(stream)>>>(t);
    if (const int rc = check_launch("dequantize")) return rc;
  }
  return clear_ok();
}
