// Orthogonalised updates: momentum, Newton-Schulz products, step.
//
//   m = b m + (1 - b) g,  u = (1 - b) g + b m  (nesterov; else m),  g = grad * grad_scale
//   X = u / (|u|_F + eps), the smaller side as rows
//   steps times:  A = X X^T,  B = b5 A + c5 A A,  X = a5 X + B X
//   w = w (1 - lr wd) - lr update_rms sqrt(max(rows, columns)) X
//
// (a5, b5, c5) = (3.4445, -4.7750, 2.0315): singular values in (0, 1] go to
// about [0.68, 1.2] in five steps, and none ever passes 1.21, whatever the
// input. So |X| < 1.21, |A| < 1.47 and |B| < 2.81, entry by entry, and all are
// held in fp16 times 2^14: no entry overflows, and those down to 2^-28 are normal.
// bf16 would lose what matters: a small singular value grows 3.44-fold each
// step while the rounding errors of the large ones grow along with it (a
// gradient with a few strong directions, 768 x 1024: 3.2% off in bf16, 0.4% in fp16).
// Most of that comes from rounding X itself, so what the rounding leaves goes
// into a second fp16 matrix, added in a5 X, which costs no product; most of the
// rest from the diagonals of A and B, which are kept in fp32 beside matrices with
// zeros there: (D + O)^2 = D^2 + D O + O D + O O, and B's diagonal joins a5 X.
// Where few rows or many steps make it count, B is multiplied with X's remainder too
// (run_batch), and up to 64 rows A's and B's are kept as well (chain_kernel). In up to five
// steps the result is then within 0.5% in the matrix's norm wherever its singular values
// lie: at worst 0.35% over spectra of decades, of two sizes and of nearly low rank, 0.49%
// over matrices of few equal values, whose entries round alike, 0.03 to 0.06% for noise
// with some strong directions; in eight steps within 1%.
//
// A and B are symmetric: only tiles on and above the diagonal are computed, and
// written twice. The products run on the LDS-DMA main loop (gemm_dma.hpp), X X^T
// with B's columns as rows. Matrices are padded with zeros to whole tiles, which
// the products leave zero. All matrices of one size go together, whichever side is the
// smaller, those of up to 16 tensors (kEntries: the table is a kernel's argument).
//
// Bound by the matrix cores where matrices are large, and there by the clock that the chip
// holds under them: 128 of 1024 x 4096 (bf16, fp32 masters) take X X^T 628 us (1094 TFLOP/s
// of its tiles), a product of m^3 229 (750), an update 1580 (695: its epilogue moves 4
// bytes in and 4 out a value while no product runs), the last one 2316 with the weights'
// step, momentum 1112 and X 1087 (both at 4.8 TB/s). Small lists are bound by their 17
// launches of 4 to 10 us: 24 of 256 x 512 take 114.

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "gemm_dma.hpp"
#include "workspace.hpp"

namespace sb {
namespace {

constexpr float kA5 = 3.4445f, kB5 = -4.7750f, kC5 = 2.0315f;
constexpr float kScale = 16384.0f, kUnscale = 1.0f / 16384.0f;
constexpr float kNormEps = 1e-7f;
constexpr int kThreads = 256;
constexpr int kMaxSteps = 32;
constexpr int64_t kMostPadded = kI32Limit / 2;  // values of a padded matrix: their offsets in bytes take 31 bits
constexpr int64_t kBatchBytes = int64_t{6} << 30;  // of a batch's workspace, where that holds a matrix

// ------------------------------------------------------------ the list ---

struct Entry {
  void* param;
  const void* grad;
  float *momentum, *master;
  int64_t param_matrix, param_row, grad_matrix, grad_row, momentum_matrix, momentum_row, master_matrix, master_row;
  int32_t first;  // its first matrix in the batch
  int32_t rows, columns;
  uint8_t param_dtype, grad_dtype, wide, tall;  // wide: vectors of 8 may be used; tall: rows > columns
};
constexpr int kEntries = 16;

struct Table {
  Entry e[kEntries];
  int32_t count;
};

struct Hyper {
  const float *lr_ptr, *grad_scale;
  float lr, momentum, weight_decay, update_rms;
  int32_t nesterov;
};

// The batch's entry of a matrix, and the matrix's place in it.
__device__ __forceinline__ const Entry& entry_of(const Table& t, int matrix, int64_t* at) {
  int i = 0;
  while (i + 1 < t.count && t.e[i + 1].first <= matrix) ++i;
  i = uniform(i);
  *at = matrix - t.e[i].first;
  return t.e[i];
}

__device__ __forceinline__ float value_of(uint16_t bits, int dtype) {
  return dtype == SB_DTYPE_BF16 ? bf16_to_f32(bits) : static_cast<float>(__builtin_bit_cast(_Float16, bits));
}

// Values i .. i + 7 of p (n of them there).
__device__ __forceinline__ void load8(const void* p, int dtype, int64_t i, int n, bool wide, float (&v)[8]) {
  if (dtype == SB_DTYPE_F32) {
    const float* f = static_cast<const float*>(p) + i;
    if (wide && n >= 8) {
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(f), b = *reinterpret_cast<const f32x4_t*>(f + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? f[e] : 0.0f;
    }
    return;
  }
  const uint16_t* h = static_cast<const uint16_t*>(p) + i;
  if (wide && n >= 8) {
    const u32x4_t a = *reinterpret_cast<const u32x4_t*>(h);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = value_of(static_cast<uint16_t>(a[e / 2] >> (16 * (e & 1))), dtype);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? value_of(h[e], dtype) : 0.0f;
  }
}

__device__ __forceinline__ uint16_t half_bits(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }

__device__ __forceinline__ u32x4_t pack8(const uint16_t (&bits)[8]) {
  u32x4_t a;
#pragma unroll
  for (int q = 0; q < 4; ++q) a[q] = bits[2 * q] | static_cast<uint32_t>(bits[2 * q + 1]) << 16;
  return a;
}

__device__ __forceinline__ void store8(void* p, int dtype, int64_t i, int n, bool wide, const float (&v)[8]) {
  if (dtype == SB_DTYPE_F32) {
    float* f = static_cast<float*>(p) + i;
    if (wide && n >= 8) {
      *reinterpret_cast<f32x4_t*>(f) = f32x4_t{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4_t*>(f + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) f[e] = v[e];
    }
    return;
  }
  uint16_t bits[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) bits[e] = dtype == SB_DTYPE_BF16 ? f32_to_bf16(v[e]) : half_bits(v[e]);
  uint16_t* h = static_cast<uint16_t*>(p) + i;
  if (wide && n >= 8) {
    *reinterpret_cast<u32x4_t*>(h) = pack8(bits);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) h[e] = bits[e];
  }
}

// What is orthogonalised, at eight values: of the momentum as it is after this
// step, or the gradient alone where there is none.
__device__ __forceinline__ void update_values(const Entry& e, const Hyper& h, float (&g)[8], const float (&m)[8]) {
  if (!e.momentum || !h.nesterov) {
    if (e.momentum)
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = m[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = (1.0f - h.momentum) * g[i] + h.momentum * m[i];
}

__device__ __forceinline__ void load_grad(const Entry& e, const Hyper& h, int64_t matrix, int row, int col, int n,
                                          float (&g)[8]) {
  load8(e.grad, e.grad_dtype, matrix * e.grad_matrix + row * e.grad_row + col, n, e.wide, g);
  if (h.grad_scale) {
    const float s = *h.grad_scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] *= s;
  }
}

// ------------------------------------------------- momentum and its size ---

constexpr int kVectors = 8;  // of 8 values, a lane's of a chunk, at most

int64_t chunks_of(int64_t rows, int64_t columns, int64_t vectors) {
  return (rows * ((columns + 7) / 8) + kThreads * vectors - 1) / (kThreads * vectors);
}

// m after this step, and the sum of u^2 over the chunk: in fp64, so that no
// gradient is too small or too large for its square.
__global__ void __launch_bounds__(kThreads) momentum_kernel(Table t, Hyper h, double* __restrict__ partial, int32_t vectors) {
  __shared__ double sums[kThreads / 64];
  int64_t matrix;
  const Entry& e = entry_of(t, static_cast<int>(blockIdx.y), &matrix);
  const uint32_t per_row = static_cast<uint32_t>((e.columns + 7) / 8), all = per_row * static_cast<uint32_t>(e.rows);
  double ss = 0.0;
#pragma unroll 2
  for (int i = 0; i < vectors; ++i) {
    const uint32_t at = (blockIdx.x * static_cast<uint32_t>(vectors) + i) * kThreads + threadIdx.x;
    if (at >= all) break;
    const int row = static_cast<int>(at / per_row), col = static_cast<int>(at % per_row) * 8, n = e.columns - col;
    float g[8], m[8] = {};
    load_grad(e, h, matrix, row, col, n, g);
    if (e.momentum) {
      const int64_t place = matrix * e.momentum_matrix + row * e.momentum_row + col;
      load8(e.momentum, SB_DTYPE_F32, place, n, e.wide, m);
#pragma unroll
      for (int q = 0; q < 8; ++q) m[q] = h.momentum * m[q] + (1.0f - h.momentum) * g[q];
      store8(e.momentum, SB_DTYPE_F32, place, n, e.wide, m);
    }
    update_values(e, h, g, m);
#pragma unroll
    for (int q = 0; q < 8; ++q) ss = fma(static_cast<double>(g[q]), static_cast<double>(g[q]), ss);
  }
  for (int s = 32; s > 0; s >>= 1) ss += __shfl_xor(ss, s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = ss;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 64; ++w) ss += sums[w];
    partial[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = ss;
  }
}

__device__ __forceinline__ float factor_of(double sum_of_squares) {
  return static_cast<float>(static_cast<double>(kScale) / (sqrt(sum_of_squares) + static_cast<double>(kNormEps)));
}

// factor[matrix] = 2^14 / (|u| + eps), the chunks' sums in a fixed order. Up to
// kFewChunks of them each wave of the next kernel adds up by itself (a launch less:
// 3.8 of 110 us for 24 of 256 x 512).
constexpr int kFewChunks = 64;

__global__ void __launch_bounds__(kThreads)
    norm_kernel(const double* __restrict__ partial, int32_t chunks, float* __restrict__ factor) {
  __shared__ double sums[kThreads / 64];
  double ss = 0.0;
  for (int i = threadIdx.x; i < chunks; i += kThreads) ss += partial[static_cast<int64_t>(blockIdx.x) * chunks + i];
  for (int s = 32; s > 0; s >>= 1) ss += __shfl_xor(ss, s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = ss;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 64; ++w) ss += sums[w];
    factor[blockIdx.x] = factor_of(ss);
  }
}

__device__ __forceinline__ float factor_of_few(const double* partial, int32_t chunks, int matrix) {
  const int lane = threadIdx.x & 63;
  double ss = lane < chunks ? partial[static_cast<int64_t>(matrix) * chunks + lane] : 0.0;
  for (int s = 32; s > 0; s >>= 1) ss += __shfl_xor(ss, s);
  return factor_of(ss);
}

// ---------------------------------------------------------------- X ---

// X [mp, np] of each matrix: hi, and lo = what hi's rounding left.
struct Padded {
  uint16_t *hi, *lo;
  int32_t mp, np;
};

constexpr int kTile = 64;

// A tile of 64 x 64 of the tensor, and its place in X: for a tall tensor the
// transposed one, through LDS (a row of 65 values: no two of a column in one bank).
struct TilePlace {
  int row, col;  // in the tensor
};

__device__ __forceinline__ TilePlace tile_place(const Entry& e, const Padded& x) {
  const int across = (e.tall ? x.mp : x.np) / kTile;
  return {static_cast<int>(blockIdx.x) / across * kTile, static_cast<int>(blockIdx.x) % across * kTile};
}

__global__ void __launch_bounds__(kThreads)
    fill_kernel(Table t, Hyper h, const double* __restrict__ partial, int32_t chunks, const float* __restrict__ factor,
                Padded x) {
  __shared__ float lds[kTile][kTile + 1];
  int64_t matrix;
  const Entry& e = entry_of(t, static_cast<int>(blockIdx.y), &matrix);
  const TilePlace tp = tile_place(e, x);
  const int y = static_cast<int>(blockIdx.y);
  const float f = chunks <= kFewChunks ? factor_of_few(partial, chunks, y) : factor[y];
  const int64_t base = static_cast<int64_t>(blockIdx.y) * x.mp * x.np;
  auto put = [&](int row, int col, const float (&v)[8]) {  // in X
    uint16_t hi[8], lo[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      hi[q] = half_bits(v[q]);
      lo[q] = half_bits(v[q] - value_of(hi[q], SB_DTYPE_F16));
    }
    const int64_t at = base + static_cast<int64_t>(row) * x.np + col;
    *reinterpret_cast<u32x4_t*>(x.hi + at) = pack8(hi);
    *reinterpret_cast<u32x4_t*>(x.lo + at) = pack8(lo);
  };
#pragma unroll
  for (int i = 0; i < kTile * kTile / 8 / kThreads; ++i) {
    const int item = i * kThreads + static_cast<int>(threadIdx.x), r = item / 8, c = item % 8 * 8;
    const int row = tp.row + r, col = tp.col + c, n = e.columns - col;
    float g[8] = {}, m[8] = {};
    if (row < e.rows && n > 0) {
      load_grad(e, h, matrix, row, col, n, g);
      if (e.momentum)
        load8(e.momentum, SB_DTYPE_F32, matrix * e.momentum_matrix + row * e.momentum_row + col, n, e.wide, m);
      update_values(e, h, g, m);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) g[q] *= f;
    if (!e.tall) {
      put(row, col, g);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) lds[r][c + q] = g[q];
    }
  }
  if (!e.tall) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kTile * kTile / 8 / kThreads; ++i) {
    const int item = i * kThreads + static_cast<int>(threadIdx.x), r = item / 8, c = item % 8 * 8;
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = lds[c + q][r];
    put(tp.col + r, tp.row + c, v);
  }
}

// ------------------------------------------------------------- products ---

// A symmetric matrix: the entries beside the diagonal in fp16 times `scale`, with
// zeros on it, and the diagonal in fp32. Each [M][mp][mp] and [M][mp]. rest: what off's
// rounding left, times `scale` (chain_kernel's factors alone).
struct Symmetric {
  uint16_t* off;
  float* diag;
  float scale;
  uint16_t* rest;
};

struct ProductArgs {
  const uint16_t *x, *lo;     // [M][mp][np]
  uint16_t *next, *next_lo;   // of the next X; next_lo may be lo where products do not read that
  Symmetric left, right, out;
  float of_left, of_right, of_product;  // out = of_left L + of_right R + of_product L R
  int32_t mp, np, matrices;
};

// Up to PARTS products one after another into one sum: a b, then a times what b's rounding
// left, then what a's left times b.
template <class Cfg, int PARTS>
struct Operands {
  __amdgpu_buffer_rsrc_t ra, rb, ra_rest, rb_rest;
  uint32_t a_off[Cfg::kAInstr], b_off[Cfg::kBInstr];
  uint32_t a_step, b_step;
  int steps;  // of a part
  __device__ __forceinline__ uint32_t a_voff(int q) const { return a_off[q]; }
  __device__ __forceinline__ uint32_t b_voff(int q) const { return b_off[q]; }
  __device__ __forceinline__ uint32_t step_of(int t) const {
    return static_cast<uint32_t>(PARTS > 2 && t >= 2 * steps ? t - 2 * steps : PARTS > 1 && t >= steps ? t - steps : t);
  }
  __device__ __forceinline__ void a_src(int t, __amdgpu_buffer_rsrc_t* r, uint32_t* s) const {
    *r = PARTS > 2 && t >= 2 * steps ? ra_rest : ra;
    *s = step_of(t) * a_step;
  }
  __device__ __forceinline__ void b_src(int t, __amdgpu_buffer_rsrc_t* r, uint32_t* s) const {
    *r = PARTS > 1 && t >= steps && !(PARTS > 2 && t >= 2 * steps) ? rb_rest : rb;
    *s = step_of(t) * b_step;
  }
};

// C rows i0 .., columns j0 .. of a [mp, k] times b: [k, columns], or with BT the rows of b
// [columns, k]. The remainders are not looked at where `parts` does not reach them.
template <class Cfg, int PARTS = 1>
__device__ __forceinline__ void product(uint8_t* __restrict__ lds, const uint16_t* a, const uint16_t* a_rest,
                                        const uint16_t* b, const uint16_t* b_rest, int mp, int k, int columns, int i0,
                                        int j0, typename DmaMainloop<Cfg>::Acc& acc, int parts = PARTS) {
  Operands<Cfg, PARTS> src;
  src.ra = make_rsrc(a, static_cast<uint32_t>(mp) * static_cast<uint32_t>(k) * 2u);
  src.rb = make_rsrc(b, static_cast<uint32_t>(columns) * static_cast<uint32_t>(k) * 2u);
  if constexpr (PARTS > 1) src.rb_rest = make_rsrc(b_rest, static_cast<uint32_t>(columns) * static_cast<uint32_t>(k) * 2u);
  if constexpr (PARTS > 2) src.ra_rest = make_rsrc(a_rest, static_cast<uint32_t>(mp) * static_cast<uint32_t>(k) * 2u);
  src.steps = k / Cfg::BK;
  const ADmaPos<Cfg> ap;
#pragma unroll
  for (int q = 0; q < Cfg::kAInstr; ++q)
    src.a_off[q] = (static_cast<uint32_t>(i0 + ap.row[q]) * static_cast<uint32_t>(k) + ap.chunk[q] * 8u) * 2u;
  src.a_step = Cfg::BK * 2;
  if constexpr (Cfg::BT) {
    const BtDmaPos<Cfg> bp;
#pragma unroll
    for (int q = 0; q < Cfg::kBInstr; ++q)
      src.b_off[q] = (static_cast<uint32_t>(j0 + bp.row[q]) * static_cast<uint32_t>(k) + bp.chunk[q] * 8u) * 2u;
    src.b_step = Cfg::BK * 2;
  } else {
    const BDmaPos<Cfg> bp;
#pragma unroll
    for (int q = 0; q < Cfg::kBInstr; ++q)
      src.b_off[q] = (static_cast<uint32_t>(bp.row[q]) * static_cast<uint32_t>(columns) + j0 + bp.col[q]) * 2u;
    src.b_step = Cfg::BK * static_cast<uint32_t>(columns) * 2u;
  }
  DmaMainloop<Cfg>::run(lds, src, parts * src.steps, acc);
}

// The accumulators in fp32 through LDS, kGroups groups of 32 rows of each row of
// waves at a time (a part): rows(part, fn) calls fn(row, col, 8 values) with rows
// and columns in the tile, neighbouring lanes on neighbouring columns. What fn
// leaves may be kept in the values' place, as 8 halves or as the values: mirror and
// columns then give it by columns, fn(col, row, of rows row ..), neighbouring lanes
// on the rows of a column that lie together.
template <class Cfg, int kGroups_ = (Cfg::TM >= 2 && 64 * Cfg::WM * Cfg::BN * 4 <= Cfg::kLdsAlloc ? 2 : 1)>
struct Epilogue {
  using ML = DmaMainloop<Cfg>;
  static constexpr int kGroups = kGroups_;
  static constexpr int kParts = Cfg::TM / kGroups;
  static constexpr int kRun = 32 * kGroups, kRows = kRun * Cfg::WM;  // rows that lie together, rows of a part
  static_assert(kRows * Cfg::BN * 4 <= Cfg::kLdsAlloc && Cfg::TM % kGroups == 0, "a part fits the ring");
  __device__ __forceinline__ static int place(int r, int col) {  // of the 16 bytes that hold (r, col)
    return r * (Cfg::BN * 4) + (((col >> 2) ^ (r & 15)) << 4);
  }
  __device__ __forceinline__ static int tile_row(int part, int r) { return r / kRun * Cfg::WTM + kRun * part + r % kRun; }

  template <int PART>
  __device__ __forceinline__ static void put(uint8_t* __restrict__ lds, const typename ML::Acc& acc) {
    const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) / Cfg::WN;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int r = kRun * wm + 32 * i + (lane & 31);
#pragma unroll
      for (int jn = 0; jn < Cfg::TN; ++jn)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16_t& v = acc[jn][PART * kGroups + i];
          *reinterpret_cast<f32x4_t*>(lds + place(r, ML::out_col(jn, g))) =
              f32x4_t{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
        }
    }
    __syncthreads();
  }

  // A thread's i-th eight values of a part: row r of the part, columns c ..
  static constexpr int kItems = kRows * Cfg::BN / 8 / Cfg::kThreads;
  __device__ __forceinline__ static int item_row(int i) { return (i * Cfg::kThreads + static_cast<int>(threadIdx.x)) / (Cfg::BN / 8); }
  __device__ __forceinline__ static int item_col(int i) { return (i * Cfg::kThreads + static_cast<int>(threadIdx.x)) % (Cfg::BN / 8) * 8; }

  // all[i] = the eight halves of `from` [.., stride] at item i of a part: asked for
  // before the part's barriers, since one by one each would wait for memory.
  __device__ __forceinline__ static void fetch(const uint16_t* from, int64_t stride, int part, u32x4_t (&all)[kItems]) {
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      all[i] = *reinterpret_cast<const u32x4_t*>(from + tile_row(part, item_row(i)) * stride + item_col(i));
  }

  // fn(i, row, col, values). KEEP 1: its result, 8 halves, is kept in the values'
  // place; 2: the values, as it leaves them.
  template <int KEEP, class Fn>
  __device__ __forceinline__ static void rows(uint8_t* __restrict__ lds, int part, Fn fn) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int r = item_row(i), c = item_col(i);
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(lds + place(r, c));
      const f32x4_t b = *reinterpret_cast<const f32x4_t*>(lds + place(r, c + 4));
      float v[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = a[q], v[4 + q] = b[q];
      const u32x4_t out = fn(i, tile_row(part, r), c, v);
      if constexpr (KEEP == 1) *reinterpret_cast<u32x4_t*>(lds + place(r, c)) = out;
      if constexpr (KEEP == 2) {
        *reinterpret_cast<f32x4_t*>(lds + place(r, c)) = f32x4_t{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_t*>(lds + place(r, c + 4)) = f32x4_t{v[4], v[5], v[6], v[7]};
      }
    }
  }

  // A thread turns blocks of 8 x 8 halves around in registers.
  template <class Fn>
  __device__ __forceinline__ static void mirror(const uint8_t* __restrict__ lds, int part, Fn fn) {
    constexpr int kTurns = kRows * Cfg::BN / 64, kBlocks = kRun / 8;
    __syncthreads();
#pragma unroll
    for (int i = 0; i * Cfg::kThreads < kTurns; ++i) {
      const int item = i * Cfg::kThreads + static_cast<int>(threadIdx.x);
      if (item >= kTurns) break;
      const int r = (item % kBlocks + item / (kBlocks * (Cfg::BN / 8)) * kBlocks) * 8, c = item / kBlocks % (Cfg::BN / 8) * 8;
      u32x4_t in[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) in[q] = *reinterpret_cast<const u32x4_t*>(lds + place(r + q, c));
#pragma unroll
      for (int q = 0; q < 8; ++q) {  // column c + q: half q of each row
        u32x4_t out;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          out[w] = q & 1 ? __builtin_amdgcn_perm(in[2 * w + 1][q / 2], in[2 * w][q / 2], 0x07060302u)
                         : __builtin_amdgcn_perm(in[2 * w + 1][q / 2], in[2 * w][q / 2], 0x05040100u);
        fn(c + q, tile_row(part, r), out);
      }
    }
  }

  // A thread's i-th eight values of a column: rows turn_row(i) .. of the part.
  static constexpr int kRunItems = kRun / 8;
  __device__ __forceinline__ static int turn_col(int i) {
    return (i * Cfg::kThreads + static_cast<int>(threadIdx.x)) / kRunItems % Cfg::BN;
  }
  __device__ __forceinline__ static int turn_row(int i) {
    const int item = i * Cfg::kThreads + static_cast<int>(threadIdx.x);
    return (item % kRunItems + item / (kRunItems * Cfg::BN) * kRunItems) * 8;
  }
  template <class Fn>
  __device__ __forceinline__ static void columns(const uint8_t* __restrict__ lds, int part, Fn fn) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int c = turn_col(i), r = turn_row(i);
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = *reinterpret_cast<const float*>(lds + place(r + q, c) + (c & 3) * 4);
      fn(i, c, tile_row(part, r), v);
    }
  }
};

// Tile `at` of the tiles on and above the diagonal of n x n.
__host__ __device__ __forceinline__ void upper_tile(int at, int n, int* i, int* j) {
  int row = 0;
  while (at >= n - row) at -= n - row, ++row;
  *i = row;
  *j = row + at;
}

// GRAM: out = X X^T. Otherwise out = of_left L + of_right R + of_product L R of
// symmetric matrices that commute, so that the result is symmetric too. With
// L = l + O, R = r + S: L R = l r + l S + O r + O S.
template <class Cfg, bool GRAM>
__global__ void __launch_bounds__(Cfg::kThreads, 1) symmetric_kernel(ProductArgs p) {
  using ML = DmaMainloop<Cfg>;
  using Ep = Epilogue<Cfg>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsAlloc];
  const int n = p.mp / Cfg::BM, per = n * (n + 1) / 2;
  const int at = xcd_remap(static_cast<int>(blockIdx.x), per * p.matrices);
  int i, j;
  upper_tile(uniform(at % per), n, &i, &j);
  const int64_t matrix = uniform(at / per);
  const int i0 = i * Cfg::BM, j0 = j * Cfg::BN;
  const int64_t square = matrix * p.mp * p.mp, line = matrix * p.mp;
  typename ML::Acc acc;
  float unit;  // of the accumulators
  if constexpr (GRAM) {
    const uint16_t* x = p.x + matrix * p.mp * p.np;
    product<Cfg>(lds, x, nullptr, x, nullptr, p.mp, p.np, p.mp, i0, j0, acc);
    unit = kUnscale * kUnscale;
  } else {
    product<Cfg>(lds, p.left.off + square, nullptr, p.right.off + square, nullptr, p.mp, p.mp, p.mp, i0, j0, acc);
    unit = p.of_product / (p.left.scale * p.right.scale);
  }
  const float scale = p.out.scale;
  uint16_t* out = p.out.off + square;
  static_for<0, Ep::kParts>([&](auto part) {
    constexpr int P = decltype(part)::value;
    u32x4_t ls[GRAM ? 1 : Ep::kItems], rs[GRAM ? 1 : Ep::kItems];
    if constexpr (!GRAM) {
      const int64_t tile = square + static_cast<int64_t>(i0) * p.mp + j0;
      Ep::fetch(p.left.off + tile, p.mp, P, ls);
      Ep::fetch(p.right.off + tile, p.mp, P, rs);
    }
    Ep::template put<P>(lds, acc);
    Ep::template rows<1>(lds, P, [&](int item, int r, int c, float (&v)[8]) {
      const int row = i0 + r, col = j0 + c;
      float w[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) w[q] = v[q] * unit;
      float l = 0.0f, rd = 0.0f;
      if constexpr (!GRAM) {
        const f32x4_t d0 = *reinterpret_cast<const f32x4_t*>(p.right.diag + line + col);
        const f32x4_t d1 = *reinterpret_cast<const f32x4_t*>(p.right.diag + line + col + 4);
        l = p.left.diag[line + row];
        rd = p.right.diag[line + row];
        const float of_s = (p.of_right + p.of_product * l) / p.right.scale, of_o = 1.0f / p.left.scale;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float o = value_of(static_cast<uint16_t>(ls[item][q / 2] >> (16 * (q & 1))), SB_DTYPE_F16);
          const float s = value_of(static_cast<uint16_t>(rs[item][q / 2] >> (16 * (q & 1))), SB_DTYPE_F16);
          w[q] += of_s * s + (p.of_left + p.of_product * (q < 4 ? d0[q] : d1[q - 4])) * (of_o * o);
        }
      }
      uint16_t bits[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) bits[q] = half_bits(w[q] * scale);
      if (i == j && row - col >= 0 && row - col < 8) {
        const int q = row - col;
        float self = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          self = q == e ? v[e] * unit : self;
          bits[e] = q == e ? 0 : bits[e];
        }
        p.out.diag[line + row] = GRAM ? self : self + p.of_left * l + p.of_right * rd + p.of_product * (l * rd);
      }
      const u32x4_t all = pack8(bits);
      *reinterpret_cast<u32x4_t*>(out + static_cast<int64_t>(row) * p.mp + col) = all;
      return all;
    });
    if (i != j)
      Ep::mirror(lds, P, [&](int c, int r, u32x4_t v) {
        *reinterpret_cast<u32x4_t*>(out + static_cast<int64_t>(j0 + c) * p.mp + i0 + r) = v;
      });
  });
}

// A and what follows from it for matrices of one tile, a workgroup each: the squares
// stay in LDS. out = B of one step, or the factor of X in two (run_steps), in place of 2 or
// 6 launches. So few rows do not average their roundings (nearly low rank, 2 x 3 7% off, 7 x 128
// 2%, 64 x 128 0.8%), and products are short here: each square keeps what its rounding to
// fp16 left beside it, products are L R with both remainders' cross terms, and the factor's
// remainder goes into X as well. X X^T takes X rounded to fp16 where n > 64, whose roundings
// average over n (0.14% for 2 rows of 65, 0.03% of 1000), and for n <= 64, one K step, its
// remainder too (5e-5). Three of 40 x 1001 76 us, one of 64 x 4096 108, 1000 of 64 x 256 222;
// without remainders 66, 96 and 182, and as launches of symmetric_kernel 78, 106 and 217.
// One LDS array: with a second one the compiler lets every read in the main loop wait for
// all loads (one of 64 x 4096: 177 without remainders). Matrices of 128 lose: a workgroup's
// product of 128^3 takes 3 us.
template <class Cfg>
__device__ __forceinline__ void chain(uint8_t* __restrict__ lds, const typename DmaMainloop<Cfg>::Acc& gram,
                                      const Symmetric& result, int64_t matrix, int32_t two) {
  using ML = DmaMainloop<Cfg>;
  constexpr int N = Cfg::BM, kBytes = N * N * 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row0 = wave / Cfg::WN * Cfg::WTM + (lane & 31), col0 = wave % Cfg::WN * Cfg::WTN + (lane & 31);
  auto scale_of = [](int of) { return of == 2 ? kScale / 4 : kScale; };
  auto diag = [&](int of, int r) -> float& { return reinterpret_cast<float*>(lds + 8 * kBytes)[of * N + r]; };
  // Where columns c .. of row r of square `of` are, or of its remainder: chunks of 8
  // halves, turned by the row.
  auto at = [&](int of, int rest, int r, int c) {
    return lds + (2 * of + rest) * kBytes + r * (2 * N) + (((c >> 3) ^ ((r ^ (r >> 3)) & 7)) << 4) + (c & 7) * 2;
  };
  // Square `to`, from fn(row, first of four columns, the accumulators' values).
  auto store = [&](int to, const typename ML::Acc& acc, auto fn) {
    const float scale = scale_of(to);
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i)
#pragma unroll
      for (int j = 0; j < Cfg::TN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int row = row0 + 32 * i, col = ML::out_col(j, g);
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[j][i][4 * g + e];
          fn(row, col, v);
          uint16_t bits[2][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = v[e] * scale;
            bits[0][e] = half_bits(x);
            bits[1][e] = half_bits(x - value_of(bits[0][e], SB_DTYPE_F16));
            if (row == col + e) diag(to, row) = v[e], bits[0][e] = bits[1][e] = 0;
          }
#pragma unroll
          for (int rest = 0; rest < 2; ++rest)
            *reinterpret_cast<u32x2_t*>(at(to, rest, row, col)) =
                u32x2_t{bits[rest][0] | static_cast<uint32_t>(bits[rest][1]) << 16,
                        bits[rest][2] | static_cast<uint32_t>(bits[rest][3]) << 16};
        }
    __syncthreads();
  };
  // to = of_l L + of_r R + of_lr L R, as symmetric_kernel; `to` is another square than both.
  auto multiply = [&](int l, int r, int to, float of_l, float of_r, float of_lr) {
    typename ML::Acc acc = {};
#pragma unroll
    for (int k0 = 0; k0 < N; k0 += 16) {
      const int k = k0 + 8 * (lane >> 5);
      bf16x8_t a[2][Cfg::TM], b[2][Cfg::TN];
#pragma unroll
      for (int rest = 0; rest < 2; ++rest) {
#pragma unroll
        for (int i = 0; i < Cfg::TM; ++i) a[rest][i] = *reinterpret_cast<const bf16x8_t*>(at(l, rest, row0 + 32 * i, k));
#pragma unroll
        for (int j = 0; j < Cfg::TN; ++j) b[rest][j] = *reinterpret_cast<const bf16x8_t*>(at(r, rest, col0 + 32 * j, k));
      }
#pragma unroll
      for (int part = 0; part < 3; ++part)  // hi hi, hi lo, lo hi
#pragma unroll
        for (int j = 0; j < Cfg::TN; ++j)
#pragma unroll
          for (int i = 0; i < Cfg::TM; ++i) acc[j][i] = ML::mfma(b[part == 1][j], a[part == 2][i], acc[j][i]);
    }
    const float ls = 1.0f / scale_of(l), rs = 1.0f / scale_of(r), unit = of_lr * ls * rs;
    store(to, acc, [&](int row, int col, float (&v)[4]) {
      auto entry = [&](int of, int rest) { return *reinterpret_cast<const u32x2_t*>(at(of, rest, row, col)); };
      const u32x2_t o[2] = {entry(l, 0), entry(l, 1)}, s[2] = {entry(r, 0), entry(r, 1)};
      auto value = [](const u32x2_t(&parts)[2], int e) {
        return value_of(static_cast<uint16_t>(parts[0][e / 2] >> (16 * (e & 1))), SB_DTYPE_F16) +
               value_of(static_cast<uint16_t>(parts[1][e / 2] >> (16 * (e & 1))), SB_DTYPE_F16);
      };
      const float ld = diag(l, row), rd = diag(r, row);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float oe = value(o, e) * ls, se = value(s, e) * rs;
        v[e] *= unit;
        if (row == col + e) v[e] += of_l * ld + of_r * rd + of_lr * (ld * rd);
        else v[e] += (of_r + of_lr * ld) * se + (of_l + of_lr * diag(r, col + e)) * oe;
      }
    });
  };
  __syncthreads();
  store(0, gram, [&](int, int, float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= kUnscale * kUnscale;
  });
  // B; then 2 a5 B + B^2, the next A and its B, and the factor of both steps. One copy
  // of the product's code, since a launch fetches every line of it anew.
#pragma unroll 1
  for (int i = 0; i < (two ? 5 : 1); ++i) {
    const int l = i == 4 ? 0 : i, r = i == 2 ? 0 : i == 4 ? 1 : i, to = i == 4 ? 2 : (i + 1) & 3;
    const bool poly = i == 0 || i == 3;
    multiply(l, r, to, poly ? kB5 : i == 1 ? 2.0f * kA5 : i == 2 ? 0.0f : kA5, i == 2 ? kA5 * kA5 : i == 4 ? kA5 : 0.0f,
             poly ? kC5 : 1.0f);
  }
  const int out = two ? 2 : 1;
  for (int i = threadIdx.x; i < N * N / 8; i += Cfg::kThreads) {
    const int r = i / (N / 8), c = i % (N / 8) * 8;
    *reinterpret_cast<u32x4_t*>(result.off + matrix * N * N + r * N + c) = *reinterpret_cast<const u32x4_t*>(at(out, 0, r, c));
    *reinterpret_cast<u32x4_t*>(result.rest + matrix * N * N + r * N + c) = *reinterpret_cast<const u32x4_t*>(at(out, 1, r, c));
  }
  for (int i = threadIdx.x; i < N; i += Cfg::kThreads) result.diag[matrix * N + i] = diag(out, i);
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, 1) chain_kernel(ProductArgs p, int32_t two) {
  static_assert(Cfg::BN == Cfg::BM && Cfg::F16);
  constexpr int kSquares = 4 * Cfg::BM * (Cfg::BM * 4 + 4);  // with remainders, and diagonals
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsAlloc > kSquares ? Cfg::kLdsAlloc : kSquares];
  const int64_t matrix = blockIdx.x;
  typename DmaMainloop<Cfg>::Acc acc;
  const uint16_t *x = p.x + matrix * p.mp * p.np, *lo = p.lo + matrix * p.mp * p.np;
  product<Cfg, 3>(lds, x, lo, x, lo, p.mp, p.np, p.mp, 0, 0, acc, p.np <= Cfg::BK ? 3 : 1);
  chain<Cfg>(lds, acc, p.out, matrix, two);
}

// next, next_lo = of_right X + L X: of X's own rows of_right and L's diagonal. PARTS 2:
// L times X's remainder too (run_batch says where). 3: and L's remainder times X.
template <class Cfg, int PARTS>
__global__ void __launch_bounds__(Cfg::kThreads, 1) update_kernel(ProductArgs p) {
  using ML = DmaMainloop<Cfg>;
  using Ep = Epilogue<Cfg>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsAlloc];
  const int mt = p.mp / Cfg::BM, per = mt * (p.np / Cfg::BN);
  const int at = xcd_remap(static_cast<int>(blockIdx.x), per * p.matrices);
  const int64_t matrix = uniform(at / per);
  const int i0 = uniform(at % per % mt) * Cfg::BM, j0 = uniform(at % per / mt) * Cfg::BN;
  const int64_t whole = matrix * p.mp * p.np, tile = whole + static_cast<int64_t>(i0) * p.np + j0;
  typename ML::Acc acc;
  const int64_t square = matrix * p.mp * p.mp;
  product<Cfg, PARTS>(lds, p.left.off + square, PARTS > 2 ? p.left.rest + square : nullptr, p.x + whole, p.lo + whole, p.mp,
                      p.mp, p.np, i0, j0, acc);
  const float unit = 1.0f / p.left.scale;
  static_for<0, Ep::kParts>([&](auto part) {
    constexpr int P = decltype(part)::value;
    u32x4_t his[Ep::kItems], los[Ep::kItems];
    Ep::fetch(p.x + tile, p.np, P, his);
    Ep::fetch(p.lo + tile, p.np, P, los);
    Ep::template put<P>(lds, acc);
    Ep::template rows<0>(lds, P, [&](int item, int r, int c, float (&v)[8]) {
      const int64_t place = tile + static_cast<int64_t>(r) * p.np + c;
      const float self = p.of_right + p.left.diag[matrix * p.mp + i0 + r];
      uint16_t hi[8], lo[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float x = value_of(static_cast<uint16_t>(his[item][q / 2] >> (16 * (q & 1))), SB_DTYPE_F16) +
                        value_of(static_cast<uint16_t>(los[item][q / 2] >> (16 * (q & 1))), SB_DTYPE_F16);
        const float y = fmaf(unit, v[q], self * x);
        hi[q] = half_bits(y);
        lo[q] = half_bits(y - value_of(hi[q], SB_DTYPE_F16));
      }
      *reinterpret_cast<u32x4_t*>(p.next + place) = pack8(hi);
      *reinterpret_cast<u32x4_t*>(p.next_lo + place) = pack8(lo);
      return u32x4_t{};
    });
  });
}

// The last step, with the weights' step in its place (apply): w = keep w - size X;
// without a momentum X itself.
template <class Cfg, int PARTS>
__global__ void __launch_bounds__(Cfg::kThreads, 1) last_kernel(ProductArgs p, Table t, Hyper h) {
  using ML = DmaMainloop<Cfg>;
  using Ep = Epilogue<Cfg, 1>;  // the weights take the registers of the other rows
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Cfg::kLdsAlloc];
  const int mt = p.mp / Cfg::BM, per = mt * (p.np / Cfg::BN);
  const int at = xcd_remap(static_cast<int>(blockIdx.x), per * p.matrices);
  const int matrix = uniform(at / per);
  const int i0 = uniform(at % per % mt) * Cfg::BM, j0 = uniform(at % per / mt) * Cfg::BN;
  const int64_t whole = static_cast<int64_t>(matrix) * p.mp * p.np, tile = whole + static_cast<int64_t>(i0) * p.np + j0;
  int64_t place;
  const Entry e = entry_of(t, matrix, &place);
  typename ML::Acc acc;
  const int64_t square = static_cast<int64_t>(matrix) * p.mp * p.mp;
  product<Cfg, PARTS>(lds, p.left.off + square, PARTS > 2 ? p.left.rest + square : nullptr, p.x + whole, p.lo + whole, p.mp,
                      p.mp, p.np, i0, j0, acc);
  const float unit = 1.0f / p.left.scale;
  const float lr = h.lr_ptr ? *h.lr_ptr : h.lr;
  const float keep = 1.0f - lr * h.weight_decay;
  const float size = lr * h.update_rms * sqrtf(static_cast<float>(max(e.rows, e.columns)));
  void* const weights = e.master ? e.master : e.param;
  const int weights_dtype = e.master ? SB_DTYPE_F32 : e.param_dtype;
  const int64_t weights_at = place * (e.master ? e.master_matrix : e.param_matrix);
  const int64_t weights_row = e.master ? e.master_row : e.param_row;
  // Weights at row, col .. of the tensor: `there` of them (none outside).
  auto there = [&](int row, int col) { return row < e.rows ? e.columns - col : 0; };
  auto fetch = [&](int row, int col, float (&w)[8]) {
    if (e.momentum && there(row, col) > 0)
      load8(weights, weights_dtype, weights_at + row * weights_row + col, there(row, col), e.wide, w);
  };
  auto step = [&](int row, int col, const float (&w)[8], const float (&x)[8]) {
    const int n = there(row, col);
    if (n <= 0) return;
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = e.momentum ? w[q] * keep - size * x[q] : x[q];
    if (e.master) store8(e.master, SB_DTYPE_F32, weights_at + row * weights_row + col, n, e.wide, v);
    store8(e.param, e.param_dtype, place * e.param_matrix + row * e.param_row + col, n, e.wide, v);
  };
  static_for<0, Ep::kParts>([&](auto part) {
    constexpr int P = decltype(part)::value;
    u32x4_t his[Ep::kItems], los[Ep::kItems];
    float w[Ep::kItems][8];
    Ep::fetch(p.x + tile, p.np, P, his);
    Ep::fetch(p.lo + tile, p.np, P, los);
#pragma unroll
    for (int i = 0; i < Ep::kItems; ++i) {
      if (e.tall) fetch(j0 + Ep::turn_col(i), i0 + Ep::tile_row(P, Ep::turn_row(i)), w[i]);
      else fetch(i0 + Ep::tile_row(P, Ep::item_row(i)), j0 + Ep::item_col(i), w[i]);
    }
    Ep::template put<P>(lds, acc);
    Ep::template rows<2>(lds, P, [&](int item, int r, int c, float (&v)[8]) {
      const float self = p.of_right + p.left.diag[static_cast<int64_t>(matrix) * p.mp + i0 + r];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float x = value_of(static_cast<uint16_t>(his[item][q / 2] >> (16 * (q & 1))), SB_DTYPE_F16) +
                        value_of(static_cast<uint16_t>(los[item][q / 2] >> (16 * (q & 1))), SB_DTYPE_F16);
        v[q] = fmaf(unit, v[q], self * x) * kUnscale;
      }
      if (!e.tall) step(i0 + r, j0 + c, w[item], v);
      return u32x4_t{};
    });
    if (e.tall) Ep::columns(lds, P, [&](int item, int c, int r, const float (&v)[8]) { step(j0 + c, i0 + r, w[item], v); });
  });
}

// 256 x 256 tiles of 8 waves (X X^T in K steps of 64, two stages of A and three
// of B; the others in steps of 32, A two at a time), 128 x 128 of 4 (64 KB of LDS, so
// that two workgroups share a CU: against three stages of 64, one a CU, 100 of 256 x 256
// take 228 us for 287, 20 of 1024 x 1024 737 for 893), or 64 x 64 of 4 (X X^T, whose
// reductions are long, with a stage more; six stages each: 141 us for 111 at 24 of
// 256 x 512).
using WideGram = DmaCfg<256, 256, 64, 2, 2, 4, 0, 0, 5, 1, 0, 3, 0, 0, 1, 0, 1>;
using WideRows = DmaCfg<256, 256, 32, 4, 2, 4, 0, 0, 5, 1, 1, 0, 0, 0, 0, 0, 1>;
using WideSquare = DmaCfg<128, 128, 32, 4, 2, 2, 0, 0, 5, 1, 1, 0, 0, 0, 0, 0, 1>;
using NarrowGram = DmaCfg<128, 128, 32, 4, 2, 2, 0, 0, 5, 1, 0, 0, 0, 0, 1, 0, 1>;
using NarrowRows = DmaCfg<128, 128, 32, 4, 2, 2, 0, 0, 5, 1, 0, 0, 0, 0, 0, 0, 1>;
using SmallGram = DmaCfg<64, 64, 64, 4, 2, 2, 0, 0, 5, 1, 0, 0, 0, 0, 1, 0, 1>;
using SmallRows = DmaCfg<64, 64, 64, 3, 2, 2, 0, 0, 5, 1, 0, 0, 0, 0, 0, 0, 1>;

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// A batch: matrices of one size.
struct Shape {
  int64_t m, n;
  int64_t mp, np;
  int tile;  // 256, 128 or 64
  bool chain;  // chain_kernel
  int32_t vectors;  // a lane's of a chunk
  bool pairs;
};

Shape shape_of(int64_t rows, int64_t columns, int64_t matrices, int cus) {
  Shape s;
  s.m = std::min(rows, columns);
  s.n = std::max(rows, columns);
  auto steps_of_a = [&](int64_t tile) {  // A's tiles on and above the diagonal, times their K steps in A A
    const int64_t t = round_up(s.m, tile) / tile;
    return matrices * t * (t + 1) / 2 * t;
  };
  auto padded = [&](int64_t tile) {  // m^2 n
    const double m = static_cast<double>(round_up(s.m, tile));
    return m * m * static_cast<double>(round_up(s.n, tile));
  };
  // Wide tiles (one workgroup a CU) where matrices are large and padding to them costs
  // little, small ones where the work is little or padding to 128 would add a third.
  // us for five steps of bf16 stacks, wide, narrow, small:
  //   128 of 768 x 2048  4223  4804  5761     24 of 256 x 512       257  161   114
  //   20 of 2048 x 2048  4183  5061  7275     200 of 256 x 256      421  396   337
  //   64 of 768 x 2048   2239  2466  2963     3 of 1024 x 1024      405  249   210
  //   26 of 1024 x 4096  2724  2774  3427     7 of 1024 x 1024      437  334   384
  //   400 of 512 x 512   2900  2902  3444     90 of 512 x 1024     1151 1077  1203
  //   100 of 512 x 2048  2052  1948  2250     100 of 320 x 1024    1170  749   592
  //   300 of 256 x 256    653   520   478     1000 of 192 x 192    1783 1694  1017
  auto fits = [&](int64_t tile) { return round_up(s.m, tile) * round_up(s.n, tile) < kMostPadded; };
  if (fits(256) && s.m > 512 && 2 * padded(256) <= 3 * padded(64) && 2 * steps_of_a(256) >= int64_t{9} * cus) s.tile = 256;
  else if (!fits(128) || steps_of_a(64) <= int64_t{32} * cus || 4 * padded(64) <= 3 * padded(128)) s.tile = 64;
  else s.tile = 128;
  // The first two steps at a time (run_steps) where X is long, and not so little that
  // launches count: 16 of 512 x 2048 take 410 us for 455, 1 of 128 x 4096 136 for 146, 100 of
  // 512 x 1024 1152 for 1231; 24 of 256 x 512 would take 115.5 for 113.7.
  s.chain = s.tile == 64 && s.m <= 64;
  s.pairs = s.n >= 2 * s.m &&
            (s.chain || s.n >= 2048 || matrices * (round_up(s.m, 64) / 64) * (round_up(s.n, 64) / 64) >= int64_t{4} * cus);
  s.mp = round_up(s.m, s.tile);
  s.np = round_up(s.n, s.tile);
  // Shorter chunks where they are few (24 of 256 x 512, 192 chunks of 8 vectors: 13.5 us).
  s.vectors = kVectors;
  while (s.vectors > 1 && matrices * chunks_of(s.m, s.n, s.vectors) < int64_t{4} * cus) s.vectors /= 2;
  return s;
}

struct Buffers {
  uint16_t *hi[2], *lo[2];
  Symmetric square[4];
  double* partial;
  float* factor;
  int64_t used;
};

Buffers carve(void* workspace, const Shape& s, int64_t matrices) {
  Carver ws{static_cast<uint8_t*>(workspace)};
  Buffers b;
  b.hi[0] = ws.take<uint16_t>(matrices * s.mp * s.np);
  b.hi[1] = ws.take<uint16_t>(matrices * s.mp * s.np);
  b.lo[0] = ws.take<uint16_t>(matrices * s.mp * s.np);
  b.lo[1] = ws.take<uint16_t>(matrices * s.mp * s.np);  // sizes do not know whether steps will need it
  for (int i = 0; i < (s.pairs && !s.chain ? 4 : 2); ++i) {
    b.square[i].off = ws.take<uint16_t>(matrices * s.mp * s.mp);
    b.square[i].diag = ws.take<float>(matrices * s.mp);
    b.square[i].rest = ws.take<uint16_t>(s.chain && i == 0 ? matrices * s.mp * s.mp : 0);
  }
  b.partial = ws.take<double>(matrices * std::max(chunks_of(s.m, s.n, s.vectors), chunks_of(s.n, s.m, s.vectors)));
  b.factor = ws.take<float>(matrices);
  b.used = ws.used;
  return b;
}

int64_t batch_bytes(const Shape& s, int64_t matrices) { return carve(nullptr, s, matrices).used; }

// Matrices of a batch.
int64_t most_of(const Shape& s) {
  int64_t most = 1;
  while (most < 65535 && batch_bytes(s, most * 2) <= kBatchBytes) most *= 2;
  return std::min<int64_t>(most, 65535);
}

// The steps, one or two at a time. Two: with P = a5 + B of A = X X^T, the next
// step's A is P A P = a5^2 A + (2 a5 B + B^2) A, and both steps' factor of X is
// P' P = a5^2 + (a5 B + a5 B' + B' B): five products of m^3 (half of each) for two, in
// place of one X X^T and one B X of m^2 n and of X's passage through memory. Worth it
// where n is 2 m or more, and only for the first two steps: the factor's entries beside
// the diagonal are those of P' P, up to 11.9 in size where B's are 2.8, and so is their
// rounding. While the singular values' squares add up to 1, few are large enough for
// that to count (256 x 512, over spectra of decades and steps: 0.27% of the result, as
// with single steps). In the next two it does (0.74%; 0.69% measured for 300 x 700, a
// quarter of the singular values ten times the others). chain_kernel's factors keep what their
// rounding leaves, and take every pair.
template <class Gram, class Square, class Rows, int PARTS, bool CHAIN = false>
int run_steps(const Table& table, const Hyper& h, const Shape& s, const Buffers& b, int64_t matrices, int32_t steps,
              hipStream_t stream) {
  if (!reduction_fits<Gram>(s.np) || !reduction_fits<Square>(s.mp) || !reduction_fits<Rows>(s.mp))
    return fail(SB_ERR_INVALID, "orthogonalise: problem too large");
  auto upper = [&](int64_t tile) { return matrices * (s.mp / tile) * (s.mp / tile + 1) / 2; };
  const int64_t all = matrices * (s.mp / Rows::BM) * (s.np / Rows::BN);
  if (all > 2147483647LL || upper(Square::BM) > 2147483647LL) return fail(SB_ERR_INVALID, "orthogonalise: problem too large");
  ProductArgs p{};
  p.mp = static_cast<int32_t>(s.mp);
  p.np = static_cast<int32_t>(s.np);
  p.matrices = static_cast<int32_t>(matrices);
  auto scaled = [&](int i, float scale) { return Symmetric{b.square[i].off, b.square[i].diag, scale, b.square[i].rest}; };
  auto multiply = [&](const Symmetric& l, const Symmetric& r, const Symmetric& out, float of_l, float of_r, float of_lr) {
    p.left = l, p.right = r, p.out = out;
    p.of_left = of_l, p.of_right = of_r, p.of_product = of_lr;
    symmetric_kernel<Square, false><<<static_cast<uint32_t>(upper(Square::BM)), Square::kThreads, 0, stream>>>(p);
    return check_launch("orthogonalise: A A");
  };
  int at = 0;
  for (int32_t done = 0; done < steps;) {
    const bool two = s.pairs && (CHAIN || done == 0) && steps - done >= 3;
    p.x = b.hi[at];
    p.next = b.hi[at ^ 1];
    p.lo = b.lo[PARTS > 1 ? at : 0];
    p.next_lo = b.lo[PARTS > 1 ? at ^ 1 : 0];
    const Symmetric a = scaled(0, kScale), poly = scaled(1, kScale);
    Symmetric factor = poly;
    if constexpr (CHAIN) {
      factor = scaled(0, two ? kScale / 4 : kScale);
      p.out = factor;
      chain_kernel<Gram><<<static_cast<uint32_t>(matrices), Gram::kThreads, 0, stream>>>(p, two);
      if (const int rc = check_launch("orthogonalise: A")) return rc;
    } else {
      p.out = a;
      symmetric_kernel<Gram, true><<<static_cast<uint32_t>(upper(Gram::BM)), Gram::kThreads, 0, stream>>>(p);
      if (const int rc = check_launch("orthogonalise: X X^T")) return rc;
      if (const int rc = multiply(a, a, poly, kB5, 0.0f, kC5)) return rc;
      if (two) {
        // |2 a5 B + B^2| and |P' P - a5^2| stay under 11.9.
        const Symmetric wide = scaled(2, kScale / 4), next_a = scaled(3, kScale), next_poly = scaled(0, kScale);
        if (const int rc = multiply(poly, poly, wide, 2.0f * kA5, 0.0f, 1.0f)) return rc;
        if (const int rc = multiply(wide, a, next_a, 0.0f, kA5 * kA5, 1.0f)) return rc;
        if (const int rc = multiply(next_a, next_a, next_poly, kB5, 0.0f, kC5)) return rc;
        if (const int rc = multiply(next_poly, poly, wide, kA5, kA5, 1.0f)) return rc;
        factor = wide;
      }
    }
    p.left = factor;
    p.of_right = two ? kA5 * kA5 : kA5;
    at ^= 1;
    done += two ? 2 : 1;
    if (done < steps) update_kernel<Rows, PARTS><<<static_cast<uint32_t>(all), Rows::kThreads, 0, stream>>>(p);
    else last_kernel<Rows, PARTS><<<static_cast<uint32_t>(all), Rows::kThreads, 0, stream>>>(p, table, h);
    if (const int rc = check_launch("orthogonalise: B X")) return rc;
  }
  return SB_OK;
}

constexpr int64_t kRemainderRows = 192;
constexpr int32_t kFewSteps = 5;

template <class T>
struct Tag {
  using type = T;
};

int run_batch(const Table& t, const Hyper& h, const Shape& s, int64_t matrices, int32_t steps, void* workspace,
              hipStream_t stream) {
  const Buffers b = carve(workspace, s, matrices);
  const uint32_t y = static_cast<uint32_t>(matrices);
  const int64_t chunks = std::max(chunks_of(s.m, s.n, s.vectors), chunks_of(s.n, s.m, s.vectors));
  const int64_t tiles = (s.mp / kTile) * (s.np / kTile);
  if (chunks > 2147483647LL || tiles > 2147483647LL) return fail(SB_ERR_INVALID, "orthogonalise: problem too large");
  momentum_kernel<<<dim3(static_cast<uint32_t>(chunks), y), kThreads, 0, stream>>>(t, h, b.partial, s.vectors);
  if (const int rc = check_launch("orthogonalise: momentum")) return rc;
  if (chunks > kFewChunks) {
    norm_kernel<<<y, kThreads, 0, stream>>>(b.partial, static_cast<int32_t>(chunks), b.factor);
    if (const int rc = check_launch("orthogonalise: norm")) return rc;
  }
  const Padded first{b.hi[0], b.lo[0], static_cast<int32_t>(s.mp), static_cast<int32_t>(s.np)};
  fill_kernel<<<dim3(static_cast<uint32_t>(tiles), y), kThreads, 0, stream>>>(t, h, b.partial, static_cast<int32_t>(chunks),
                                                                            b.factor, first);
  if (const int rc = check_launch("orthogonalise: fill")) return rc;
  if (s.chain) return run_steps<SmallGram, SmallRows, SmallRows, 3, true>(t, h, s, b, matrices, steps, stream);
  // B X takes X rounded to fp16, a5 X all of it. What B X lacks is noise in the rows of the
  // large singular values, whose product with the noise in A falls on the small ones'.
  // Beyond 192 rows and in up to five steps the result stays within 0.35% whatever the
  // singular values; with 65 rows it is up to 0.8% off, and in eight steps up to 17% (half
  // of the singular values 1e-4 of the others). There B is multiplied with X's remainder
  // too: 0.2% in five steps, 0.6% in eight. That takes 3 to 13% longer for few rows (3 of
  // 77 x 1001 93 us for 90, 100 of 128 x 4096 751 for 668), more for many (eight steps of
  // 128 of 768 x 2048: 8300 for 6700).
  const bool remainder = s.m <= kRemainderRows || steps > kFewSteps;
  auto run = [&](auto gram, auto square, auto rows) {
    using G = typename decltype(gram)::type;
    using S = typename decltype(square)::type;
    using R = typename decltype(rows)::type;
    return remainder ? run_steps<G, S, R, 2>(t, h, s, b, matrices, steps, stream)
                     : run_steps<G, S, R, 1>(t, h, s, b, matrices, steps, stream);
  };
  if (s.tile == 64) return run(Tag<SmallGram>{}, Tag<SmallRows>{}, Tag<SmallRows>{});
  if (s.tile == 128) return run(Tag<NarrowGram>{}, Tag<NarrowRows>{}, Tag<NarrowRows>{});
  // The squares of wide matrices in the tiles whose rounds are shorter: 128 x 128, two
  // a CU, take 1.15 times as long for their area (128 of 1024 x 1024 237 us for 227 in
  // 9 rounds of half a wide one's for 5 of those; 64 of them 117 for 129, 5 for 3).
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  auto rounds = [&](int64_t tile, int64_t at_once) {
    const int64_t n = s.mp / tile;
    return (matrices * n * (n + 1) / 2 + at_once - 1) / at_once;
  };
  if (23 * rounds(128, int64_t{2} * cus) < 40 * rounds(256, cus)) return run(Tag<WideGram>{}, Tag<WideSquare>{}, Tag<WideRows>{});
  return run(Tag<WideGram>{}, Tag<WideRows>{}, Tag<WideRows>{});
}

bool known_dtype(int64_t d) { return d == SB_DTYPE_BF16 || d == SB_DTYPE_F16 || d == SB_DTYPE_F32; }

int check_list(const SbMuonTensor* tensors, int64_t count) {
  if (count < 0 || (count > 0 && !tensors)) return fail(SB_ERR_INVALID, "muon: null buffer");
  for (int64_t i = 0; i < count; ++i) {
    const SbMuonTensor& a = tensors[i];
    if (a.matrices < 0 || a.rows < 0 || a.columns < 0) return fail(SB_ERR_INVALID, "muon: negative size");
    if (a.matrices == 0 || a.rows == 0 || a.columns == 0) continue;
    if (a.rows >= kI32Limit || a.columns >= kI32Limit || a.matrices >= kI32Limit ||
        round_up(a.rows, 64) * round_up(a.columns, 64) >= kMostPadded)
      return fail(SB_ERR_INVALID, "muon: under 2^31 matrices of under 2^30 values, sides padded to 64, got %lld of %lld x %lld",
                  static_cast<long long>(a.matrices), static_cast<long long>(a.rows), static_cast<long long>(a.columns));
    if (!a.param || !a.grad) return fail(SB_ERR_INVALID, "muon: null buffer");
    if (!known_dtype(a.param_dtype) || !known_dtype(a.grad_dtype))
      return fail(SB_ERR_INVALID, "muon: unsupported dtype code");
    for (const int64_t stride : {a.param_matrix, a.param_row, a.grad_matrix, a.grad_row, a.momentum_matrix,
                                 a.momentum_row, a.master_matrix, a.master_row})
      if (stride < 0) return fail(SB_ERR_INVALID, "muon: negative stride");
  }
  return SB_OK;
}

bool empty(const SbMuonTensor& a) { return a.matrices == 0 || a.rows == 0 || a.columns == 0; }

// Where a stack's values lie: rows of `width` bytes, and two counts with their strides, the
// larger stride first.
struct Place {
  int64_t first, last;  // its bytes are in [first, last)
  int64_t width, n[2], stride[2];
  int64_t tensor;
  int kind;  // 0 parameter, 1 master, 2 momentum, 3 gradient
};

Place place_of(const SbMuonTensor& a, int64_t tensor, int kind, const void* p, int64_t bytes, int64_t matrix, int64_t row) {
  Place q{};
  q.width = a.columns * bytes;
  q.n[0] = matrix > 0 ? a.matrices : 1, q.stride[0] = matrix * bytes;
  q.n[1] = row > 0 ? a.rows : 1, q.stride[1] = row * bytes;
  if (q.n[1] == 1 || (q.n[0] > 1 && q.stride[1] > q.stride[0])) std::swap(q.n[0], q.n[1]), std::swap(q.stride[0], q.stride[1]);
  q.first = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p));
  q.last = q.first + (q.n[0] - 1) * q.stride[0] + (q.n[1] - 1) * q.stride[1] + q.width;
  q.tensor = tensor;
  q.kind = kind;
  return q;
}

bool same_place(const Place& a, const Place& b) {
  return a.first == b.first && a.last == b.last && a.width == b.width && a.n[0] == b.n[0] && a.n[1] == b.n[1] &&
         a.stride[0] == b.stride[0];
}

// f(i) for the i of low .. high with after < at + i step < before, until it is true.
template <class F>
bool any_between(int64_t at, int64_t step, int64_t low, int64_t high, int64_t after, int64_t before, F&& f) {
  if (step == 0) return after < at && at < before && f(int64_t{0});
  auto floor_of = [&](int64_t v) { return v / step - (v % step < 0); };
  for (int64_t i = std::max(low, floor_of(after - at) + 1), last = std::min(high, -floor_of(at - before) - 1); i <= last; ++i)
    if (f(i)) return true;
  return false;
}

// Whether two stacks have a byte in common. Where their strides differ that is left open: false.
bool share_bytes(const Place& a, const Place& b) {
  int64_t stride[2];
  for (int d = 0; d < 2; ++d) {
    if (a.n[d] > 1 && b.n[d] > 1 && a.stride[d] != b.stride[d]) return false;
    stride[d] = a.n[d] > 1 ? a.stride[d] : b.n[d] > 1 ? b.stride[d] : 0;
  }
  // Row j of matrix i of b lies at + i stride[0] + j stride[1] from a's first one: of both
  // rows' and matrices' numbers the differences count.
  const int64_t at = b.first - a.first;
  return any_between(at, stride[0], 1 - a.n[0], b.n[0] - 1, -b.width - (b.n[1] - 1) * stride[1],
                     a.width + (a.n[1] - 1) * stride[1], [&](int64_t i) {
                       return any_between(at + i * stride[0], stride[1], 1 - a.n[1], b.n[1] - 1, -b.width, a.width,
                                          [](int64_t) { return true; });
                     });
}

// No values that are written lie where others do: workgroups would race for them. A
// parameter may be its own fp32 master, and its own gradient (or the master may): gradients
// are read for the last time before weights are written.
int check_apart(const SbMuonTensor* tensors, int64_t count) try {
  std::vector<Place> places;
  for (int64_t i = 0; i < count; ++i) {
    const SbMuonTensor& a = tensors[i];
    if (empty(a)) continue;
    auto bytes = [](int32_t dtype) -> int64_t { return dtype == SB_DTYPE_F32 ? 4 : 2; };
    places.push_back(place_of(a, i, 0, a.param, bytes(a.param_dtype), a.param_matrix, a.param_row));
    if (a.master) places.push_back(place_of(a, i, 1, a.master, 4, a.master_matrix, a.master_row));
    if (a.momentum) places.push_back(place_of(a, i, 2, a.momentum, 4, a.momentum_matrix, a.momentum_row));
    places.push_back(place_of(a, i, 3, a.grad, bytes(a.grad_dtype), a.grad_matrix, a.grad_row));
  }
  std::sort(places.begin(), places.end(), [](const Place& a, const Place& b) { return a.first < b.first; });
  std::vector<Place> reach;  // those before that end behind this one's start
  for (const Place& p : places) {
    reach.erase(std::remove_if(reach.begin(), reach.end(), [&](const Place& q) { return q.last <= p.first; }), reach.end());
    for (const Place& q : reach) {
      if (p.kind == 3 && q.kind == 3) continue;
      if (p.tensor == q.tensor && p.kind != 2 && q.kind != 2 && same_place(p, q)) continue;
      if (share_bytes(q, p)) return fail(SB_ERR_INVALID, "muon: parameters, momenta, masters and gradients must not overlap");
    }
    reach.push_back(p);
  }
  return SB_OK;
} catch (const std::bad_alloc&) {
  return fail(SB_ERR_INVALID, "muon: no memory for a list of %lld tensors", static_cast<long long>(count));
}

bool wide_values(const SbMuonTensor& a) {
  auto ok = [](const void* p, int64_t dtype, int64_t matrix, int64_t row) {
    const int64_t bytes = dtype == SB_DTYPE_F32 ? 4 : 2;
    return !p || (aligned16(p) && matrix * bytes % 16 == 0 && row * bytes % 16 == 0);
  };
  return ok(a.param, a.param_dtype, a.param_matrix, a.param_row) && ok(a.grad, a.grad_dtype, a.grad_matrix, a.grad_row) &&
         ok(a.momentum, SB_DTYPE_F32, a.momentum_matrix, a.momentum_row) &&
         ok(a.master, SB_DTYPE_F32, a.master_matrix, a.master_row);
}

// f(table, shape, matrices) for each batch: matrices of one size, of up to kEntries tensors,
// as many as their workspace's bound lets in. Their own number chooses their shape.
template <class F>
int for_each_batch(const SbMuonTensor* tensors, int64_t count, int cus, F&& f) {
  auto same = [&](int64_t i, int64_t q) {
    return !empty(tensors[q]) && std::minmax(tensors[i].rows, tensors[i].columns) == std::minmax(tensors[q].rows, tensors[q].columns);
  };
  for (int64_t i = 0; i < count; ++i) {
    if (empty(tensors[i])) continue;
    bool first = true;
    for (int64_t q = 0; q < i && first; ++q) first = !same(i, q);
    if (!first) continue;
    int64_t total = 0;
    for (int64_t q = i; q < count; ++q)
      if (same(i, q)) total += tensors[q].matrices;
    const int64_t most = most_of(shape_of(tensors[i].rows, tensors[i].columns, total, cus));
    Table t{};
    int64_t matrices = 0;
    auto flush = [&]() -> int {
      const int rc = matrices ? f(t, shape_of(tensors[i].rows, tensors[i].columns, matrices, cus), matrices) : SB_OK;
      t = Table{};
      matrices = 0;
      return rc;
    };
    for (int64_t q = i; q < count; ++q) {
      if (!same(i, q)) continue;
      const SbMuonTensor& a = tensors[q];
      for (int64_t at = 0; at < a.matrices;) {
        if (t.count == kEntries || matrices == most)
          if (const int rc = flush()) return rc;
        const int64_t take = std::min(a.matrices - at, most - matrices);
        const int64_t pe = a.param_dtype == SB_DTYPE_F32 ? 4 : 2, ge = a.grad_dtype == SB_DTYPE_F32 ? 4 : 2;
        t.e[t.count++] = Entry{static_cast<uint8_t*>(a.param) + at * a.param_matrix * pe,
                               static_cast<const uint8_t*>(a.grad) + at * a.grad_matrix * ge,
                               a.momentum ? a.momentum + at * a.momentum_matrix : nullptr,
                               a.master ? a.master + at * a.master_matrix : nullptr,
                               a.param_matrix, a.param_row, a.grad_matrix, a.grad_row, a.momentum_matrix,
                               a.momentum_row, a.master_matrix, a.master_row, static_cast<int32_t>(matrices),
                               static_cast<int32_t>(a.rows), static_cast<int32_t>(a.columns),
                               static_cast<uint8_t>(a.param_dtype), static_cast<uint8_t>(a.grad_dtype),
                               static_cast<uint8_t>(wide_values(a)), static_cast<uint8_t>(a.rows > a.columns)};
        matrices += take;
        at += take;
      }
    }
    if (const int rc = flush()) return rc;
  }
  return SB_OK;
}

int run_list(const SbMuonTensor* tensors, int64_t count, const Hyper& h, int32_t steps, void* workspace,
             int64_t workspace_bytes, hipStream_t stream) {
  if (steps < 1 || steps > kMaxSteps) return fail(SB_ERR_INVALID, "muon: 1 to %d steps, got %d", kMaxSteps, steps);
  if (const int rc = check_apart(tensors, count)) return rc;
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  // All of them before the first is launched: a list that is refused is left as it was.
  const int rc = for_each_batch(tensors, count, cus, [&](const Table&, const Shape& s, int64_t matrices) {
    return check_workspace(workspace, workspace_bytes, batch_bytes(s, matrices));
  });
  if (rc) return rc;
  return for_each_batch(tensors, count, cus, [&](const Table& t, const Shape& s, int64_t matrices) {
    return run_batch(t, h, s, matrices, steps, workspace, stream);
  });
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_muon_sizes(const SbMuonTensor* tensors, int64_t count, int64_t* workspace_bytes) {
  if (const int rc = check_list(tensors, count)) return rc;
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  int64_t most = 256;
  if (const int rc = for_each_batch(tensors, count, cus, [&](const Table&, const Shape& s, int64_t matrices) {
        most = std::max(most, batch_bytes(s, matrices));
        return SB_OK;
      }))
    return rc;
  if (workspace_bytes) *workspace_bytes = most;
  return clear_ok();
}

extern "C" int sb_muon(const SbMuonTensor* tensors, int64_t count, float lr, const float* lr_ptr, float momentum,
                       int32_t nesterov, float weight_decay, float update_rms, int32_t steps, const float* grad_scale,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check_list(tensors, count)) return rc;
  for (int64_t i = 0; i < count; ++i)
    if (!empty(tensors[i]) && !tensors[i].momentum) return fail(SB_ERR_INVALID, "muon: null buffer");
  if (!(momentum >= 0.0f && momentum < 1.0f)) return fail(SB_ERR_INVALID, "muon: momentum must be in [0, 1)");
  const Hyper h{lr_ptr, grad_scale, lr, momentum, weight_decay, update_rms, nesterov != 0};
  if (const int rc = run_list(tensors, count, h, steps, workspace, workspace_bytes, as_stream(stream))) return rc;
  return clear_ok();
}

extern "C" int sb_orthogonalize(const SbMuonTensor* tensors, int64_t count, int32_t steps, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if (const int rc = check_list(tensors, count)) return rc;
  for (int64_t i = 0; i < count; ++i)
    if (tensors[i].momentum || tensors[i].master)
      return fail(SB_ERR_INVALID, "orthogonalise: neither momentum nor master");
  const Hyper h{};
  if (const int rc = run_list(tensors, count, h, steps, workspace, workspace_bytes, as_stream(stream))) return rc;
  return clear_ok();
}
