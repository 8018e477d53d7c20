// The weight gradients of the gated experts, dW1[e] = xg^T [dG | dU] and
// dW2[e] = wh^T gog over the expert's rows: for each expert a product whose
// reduction is short (its rows, often 100 or so) and whose output is long (all
// of its weights), so a tile is a few K steps and 128 KB of output.
//
// One workgroup per CU walks its tiles of both products, and the K steps of
// all its tiles form one stream through the ring: the loads run three steps
// ahead of the products, across tile borders, so a tile's first data arrives
// while the one before it is computed and written. The finished tile leaves
// through LDS of its own (the ring stays in use). D = 1024, F = 4096, E = 64, 128
// rows an expert, both products: 567 us as workgroups of their own, whatever the
// tile (each took 11 us, most of it its start and its first loads), 451 this way;
// 240 is the write alone (1.6 GB at 6.9 TB/s), 284 all but the output. D = 4096,
// F = 14336, E = 8, 512 rows an expert 1662 us, 868 TFLOP/s: there a K step takes 1.0
// us, twice its MFMAs. Both operands are read transposed (ds_read_b64_tr), 98
// KB of LDS a step, and these reads run at half the rate of the others.
//
// Tile 256 x 256, 8 waves (2 x 4, 128 x 64 each), K steps of 32 through a
// 4-stage ring (128 KB), the output in four parts of 64 rows through 32 KB. A
// side that 256 do not divide ends in half a tile: what its loads find past the
// edge are other columns' values (or zeros, past the last row), and meets only
// results that are not written.
// Each expert's tiles go over all XCDs, a contiguous part of them each, and the
// experts with most rows come first, runs of a tile a CU in alternate
// directions, so that whatever the routing every CU gets its share of the K
// steps (E = 128, D = 2048, F = 768, one expert with 3000 of 16380 rows: in the
// experts' order 443 us, 377 this way).

#include "gated.hpp"

namespace sb {
namespace {

using Cfg = DmaCfg<256, 256, 32, 4, 2, 4, 0, 0, 5, 1, 0, 0, 0, 1>;
using ML = DmaMainloop<Cfg>;
constexpr int kRing = Cfg::STAGES * Cfg::kStageBytes;
constexpr int kPartRows = 64, kPartBytes = kPartRows * Cfg::BN * 2;
constexpr int kStores = kPartBytes / 16 / Cfg::kThreads;  // a lane's, per part
static_assert(kRing + kPartBytes <= 160 * 1024 && Cfg::TM == 4, "LDS; a part is a row group of each wave row");

struct Product {
  const uint16_t *a, *b;  // [P, m], [P, n]
  uint16_t* out;          // [E, m, n]
  int32_t m, n;
};

struct OuterArgs {
  Product p[2];
  GatedLayout layout;
  const int32_t* expert_order;
  int32_t tiles[2];  // of an expert
  int32_t total;     // of all experts
};

// A tile: its operands from the expert's first row and the tile's first
// column, its rows (K), and where it goes.
struct Tile {
  const uint16_t *a, *b;
  uint16_t* out;
  int32_t m, n, rows;
  int32_t height, width;  // up to 256
};

// The K steps of a tile; one, of rows past the expert's last (zeros), for an
// expert without rows.
__device__ __forceinline__ int steps_of(const Tile& t) { return max(1, (t.rows + Cfg::BK - 1) / Cfg::BK); }

__host__ __device__ __forceinline__ int tiles_over(int64_t length, int tile) {
  return static_cast<int>((length + tile - 1) / tile);
}

// 64 tiles of the workgroup's list, one a lane: worked out together (the
// divisions and the loads of an expert's rows take microseconds one by one),
// read by v_readlane.
struct Batch {
  int32_t rows, row0, place, expert;  // place: tile row | tile column << 16; expert: | product << 31, -1 past the list
  // The workgroup's tiles from number `first` on: one in each run of
  // gridDim.x tiles, whose odd runs are taken in the other direction.
  __device__ __forceinline__ Batch(const OuterArgs& args, int first) {
    const int i = first + static_cast<int>(threadIdx.x & 63), stride = static_cast<int>(gridDim.x);
    const int t = i * stride + (i & 1 ? stride - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x));
    rows = row0 = place = 0;
    expert = -1;
    if (t >= args.total) return;
    const int both = args.tiles[0] + args.tiles[1], at = t / both;
    const int e = min(max(args.expert_order[at], 0), args.layout.num_experts - 1);
    const int which = t - at * both >= args.tiles[0] ? 1 : 0;
    const int per = which ? args.tiles[1] : args.tiles[0];
    // Workgroups keep to an XCD, so a tile's place in its expert's order modulo
    // 8 says which: each XCD gets a contiguous part of the expert's tiles.
    const int j = t - at * both - (which ? args.tiles[0] : 0);
    const int part = per / kNumXcd, rem = per % kNumXcd, x = j % kNumXcd;
    const int tile = (x < rem ? x * (part + 1) : rem * (part + 1) + (x - rem) * part) + j / kNumXcd;
    // Groups of kTileGroup tile rows, walked down one column at a time.
    const int row_tiles = tiles_over(which ? args.p[1].m : args.p[0].m, Cfg::BM);
    const int slices = tiles_over(which ? args.p[1].n : args.p[0].n, Cfg::BN);
    const int group = tile / (kTileGroup * slices);
    const int height = min(kTileGroup, row_tiles - group * kTileGroup);
    const int in = tile - group * kTileGroup * slices;
    place = (group * kTileGroup + in % height) | in / height << 16;
    expert = e | which << 31;
    rows = args.layout.tokens_per_expert[e];
    row0 = args.layout.padded_offsets[e];
    if (rows < 0 || row0 < 0 || row0 + rows > args.layout.max_row_blocks * kBS) rows = row0 = 0;  // not a routing layout
  }
  __device__ __forceinline__ Tile get(const OuterArgs& args, int lane) const {
    const int32_t code = __builtin_amdgcn_readlane(expert, lane), at = __builtin_amdgcn_readlane(place, lane);
    const int64_t first_row = __builtin_amdgcn_readlane(row0, lane);
    const bool second = code < 0;
    const int64_t e = code & 0x7fffffff, m0 = (at & 0xffff) * Cfg::BM, n0 = (at >> 16) * Cfg::BN;
    Tile t;
    t.m = second ? args.p[1].m : args.p[0].m;
    t.n = second ? args.p[1].n : args.p[0].n;
    t.rows = code == -1 ? -1 : __builtin_amdgcn_readlane(rows, lane);
    t.a = (second ? args.p[1].a : args.p[0].a) + first_row * t.m + m0;
    t.b = (second ? args.p[1].b : args.p[0].b) + first_row * t.n + n0;
    t.out = (second ? args.p[1].out : args.p[0].out) + (e * t.m + m0) * t.n + n0;
    t.height = min(t.m - static_cast<int32_t>(m0), static_cast<int32_t>(Cfg::BM));
    t.width = min(t.n - static_cast<int32_t>(n0), static_cast<int32_t>(Cfg::BN));
    return t;
  }
};

// This wave's loads of one step into a slot: operator()(q), q < kCount, issues
// one (A's, then B's). The buffers start at the step's first row and end at the
// tile's last column in the expert's last one: rows past it read as zeros. Issued from within
// ML::compute, through a __restrict__ pointer to another slot than the one
// that is read there: otherwise the compiler waits for them before each read.
struct StepLoads {
  static constexpr int kCount = Cfg::kLoadsPerStep;
  uint8_t* __restrict__ slot;
  __amdgpu_buffer_rsrc_t ra, rb;
  int32_t m, n;
  const AtDmaPos<Cfg>& ap;
  const BDmaPos<Cfg>& bp;
  __device__ __forceinline__ StepLoads(const Tile& t, int step, uint8_t* __restrict__ slot_, const AtDmaPos<Cfg>& ap_,
                                       const BDmaPos<Cfg>& bp_)
      : slot(slot_ + (threadIdx.x >> 6) * (Cfg::kAInstr * 1024)), m(t.m), n(t.n), ap(ap_), bp(bp_) {
    static_assert(Cfg::kAInstr == Cfg::kBInstr, "one wave offset for both");
    const int left = min(t.rows - step * Cfg::BK, static_cast<int>(Cfg::BK));
    const bool some = left > 0;  // past the last tile: empty buffers, no read of memory
    ra = make_rsrc(t.a + static_cast<int64_t>(step) * Cfg::BK * m,
                   some ? static_cast<uint32_t>((left - 1) * m + t.height) * 2u : 0u);
    rb = make_rsrc(t.b + static_cast<int64_t>(step) * Cfg::BK * n,
                   some ? static_cast<uint32_t>((left - 1) * n + t.width) * 2u : 0u);
  }
  __device__ __forceinline__ void operator()(int q) const {
    if (q < Cfg::kAInstr)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void_t*)(slot + q * 1024), 16,
                                               static_cast<uint32_t>(ap.row[q] * m + ap.col[q]) * 2u, 0, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rb, (lds_void_t*)(slot + Cfg::kABytes + (q - Cfg::kAInstr) * 1024), 16,
          static_cast<uint32_t>(bp.row[q - Cfg::kAInstr] * n + bp.col[q - Cfg::kAInstr]) * 2u, 0, 0, 0);
  }
};

// Every wave's LDS accesses before it are done, its loads under way stay so
// (__syncthreads would wait for them too).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Part P of the finished tile: row group P of each row of waves.
template <int P>
__device__ __forceinline__ void write_part(uint8_t* __restrict__ stage, const Tile& t, const ML::Acc& acc) {
  const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) / Cfg::WN;
  lds_barrier();  // the part before has been read
#pragma unroll
  for (int jn = 0; jn < Cfg::TN; ++jn)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int n = ML::out_col(jn, g);
      *reinterpret_cast<u32x2_t*>(stage + staged_at<Cfg::BN * 2>(32 * wm + (lane & 31), n >> 3) + (n & 7) * 2) =
          u32x2_t{pack_bf16x2(acc[jn][P][4 * g], acc[jn][P][4 * g + 1]),
                  pack_bf16x2(acc[jn][P][4 * g + 2], acc[jn][P][4 * g + 3])};
    }
  lds_barrier();
  // Places past the tile's edges are out of the buffer, so every lane's stores
  // are issued, whatever the tile: the loop's waits count them.
  const auto out = make_rsrc(t.out, static_cast<uint32_t>((t.height - 1) * t.n + t.width) * 2u);
#pragma unroll
  for (int s = 0; s < kStores; ++s) {
    const int q = s * Cfg::kThreads + static_cast<int>(threadIdx.x);
    const int r = q / (Cfg::BN / 8), c = q % (Cfg::BN / 8);
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(stage + staged_at<Cfg::BN * 2>(r, c));
    const uint32_t at = static_cast<uint32_t>((r / 32 * Cfg::WTM + 32 * P + r % 32) * t.n + c * 8) * 2u;
    // Past the caches: the gradients are read next by another call, and what
    // they would displace is read by this one.
    __builtin_amdgcn_raw_buffer_store_b128(v, out, c * 8 < t.width ? at : kOutOfRange, 0, 2);  // nt
  }
}

__device__ __forceinline__ void outer_stream(uint8_t* __restrict__ ring, uint8_t* __restrict__ stage,
                                             const OuterArgs& args) {
  const AtDmaPos<Cfg> ap;
  const BDmaPos<Cfg> bp;
  constexpr int S = Cfg::STAGES, kL = Cfg::kLoadsPerStep;

  // Tile i of the workgroup is lane i % 64 of batch i / 64; `near` is the batch
  // of the tile being computed, and the loads are at most S - 1 tiles ahead.
  Batch near(args, 0), far(args, 64);
  int base = 0;  // near's first tile
  auto tile_at = [&](int i) { return i - base < 64 ? near.get(args, i - base) : far.get(args, i - base - 64); };

  Tile in = tile_at(0);
  int in_at = 0, in_step = 0;  // the next step to load
  auto next_loads = [&](int to) {
    if (in.rows >= 0 && in_step >= steps_of(in)) {
      in = tile_at(++in_at);
      in_step = 0;
    }
    return StepLoads(in, in_step++, ring + to * Cfg::kStageBytes, ap, bp);
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) ML::issue_all(next_loads(s));

  const typename ML::Frags fr;
  typename ML::FragA fa;
  typename ML::FragB fb;
  wait_vmcnt<(S - 2) * kL>();
  __builtin_amdgcn_s_barrier();
  fr.read_a(ring, 0, 0, fa[0]);
  fr.read_b(ring + Cfg::kABytes, 0, fb[0]);

  int slot = 0;
  int since = S;  // steps since the last tile was written
  for (int i = 0;; ++i) {
    if (i - base == 64) {
      near = far;
      base += 64;
      far = Batch(args, base + 64);
    }
    const Tile t = near.get(args, i - base);
    if (t.rows < 0) break;
    ML::Acc acc;
#pragma unroll
    for (int jn = 0; jn < Cfg::TN; ++jn)
#pragma unroll
      for (int im = 0; im < Cfg::TM; ++im)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[jn][im][v] = 0.0f;
    const int steps = steps_of(t);
    for (int k = 0; k < steps; ++k) {
      // A step's loads go to the slot that was read before it (every wave has
      // passed the barrier of that step's end). Its end waits for the next
      // step's loads: at most the operations after them are outstanding then,
      // the loads of S - 2 steps, and a tile's stores if they came in between
      // (the loads were issued S - 2 steps ago).
      const bool stores = since < S - 2;
      auto wait = [&] {
        if (stores) wait_vmcnt<(S - 2) * kL + Cfg::TM * kStores>();
        else wait_vmcnt<(S - 2) * kL>();
      };
      ++since;
      const uint8_t* from = ring + slot * Cfg::kStageBytes;
      const uint8_t* next = ring + (slot + 1) % S * Cfg::kStageBytes;
      ML::template compute_xs<true>(from, from + Cfg::kABytes, 0, acc, next_loads((slot + S - 1) % S), fr, fa, fb, next,
                                    next + Cfg::kABytes, 0, wait);
      slot = (slot + 1) % S;
    }
    static_for<0, Cfg::TM>([&](auto pc) { write_part<decltype(pc)::value>(stage, t, acc); });
    since = 0;
  }
  wait_vmcnt<0>();  // no load may write LDS that is no longer this workgroup's
}

__global__ void __launch_bounds__(Cfg::kThreads) expert_outer_stream_kernel(OuterArgs args) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kRing + kPartBytes];
  outer_stream(lds, lds + kRing, args);
}

}  // namespace

int launch_expert_outers(const void* a1, const void* b1, void* out1, int64_t m1, int64_t n1, const void* a2,
                         const void* b2, void* out2, int64_t m2, int64_t n2, const GatedLayout& layout,
                         const int32_t* expert_order, hipStream_t stream) {
  int cus = 0;
  if (const int rc = device_cus(&cus)) return rc;
  OuterArgs args{};
  auto product = [&](int i, const void* a, const void* b, void* out, int64_t m, int64_t n) {
    args.p[i] = Product{static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(b), static_cast<uint16_t*>(out),
                        static_cast<int32_t>(m), static_cast<int32_t>(n)};
    const int64_t tiles = static_cast<int64_t>(tiles_over(m, Cfg::BM)) * tiles_over(n, Cfg::BN);
    args.tiles[i] = static_cast<int32_t>(tiles);
    return tiles * layout.num_experts;
  };
  args.layout = layout;
  const int64_t total = product(0, a1, b1, out1, m1, n1) + product(1, a2, b2, out2, m2, n2);
  args.expert_order = expert_order;
  // Whole eighths of workgroups, so that each keeps to its XCD's tiles.
  const int64_t grid = std::max<int64_t>(kNumXcd, std::min<int64_t>(total, cus) / kNumXcd * kNumXcd);
  if (total + 192 * grid > 2147483647LL || tiles_over(std::max(m1, m2), Cfg::BM) > 65535 ||
      tiles_over(std::max(n1, n2), Cfg::BN) > 32767)
    return fail(SB_ERR_INVALID, "problem too large");
  args.total = static_cast<int32_t>(total);
  expert_outer_stream_kernel<<<static_cast<uint32_t>(grid), Cfg::kThreads, 0, stream>>>(args);
  return check_launch("gated backward: weight gradients");
}

}  // namespace sb
