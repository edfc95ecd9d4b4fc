// Products of ragged row groups, each with a weight of its own, in bf16 or block-scaled e4m3:
//
//   D[m,:] = A[m,:] * B[g],   group_offsets[g] <= m < group_offsets[g + 1]
//
// One group without offsets is the plain product.  With e4m3 operands every 128 elements of a row of A
// and every 128 x 128 block of B carry an fp32 scale:
//
//   D[m,n] = sum_b sa[m,b] * sb[b,n/128] * sum_{k in block b} A[m,k] * B[k,n]
//
// The inner sums are tensor-core work (tcgen05.mma, fp32 in TMEM), the outer one is a multiply-add per
// output element and block on the CUDA cores: the accumulator of each K block is read out of TMEM, scaled
// (one factor per thread: a thread owns a row, and 128 columns share a scale of B) and added to fp32 sums
// in registers, while the tensor core fills another TMEM buffer with the next block.
//
// Roles inside a 384-thread CTA: warp 0 TMA producer, warp 1 MMA issuer, warp 2 TMEM allocator, warps 4-11
// promotion and epilogue (warp % 4 names the TMEM lane quadrant = 32 rows, the half of the eight warps the
// columns).  The grid is persistent; every role walks the same list of work items, which each CTA derives
// from the group offsets in device memory: a tile never holds rows of two groups.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "xf_act.cuh"
#include "xf_params.h"
#include "xf_ptx.cuh"

namespace xf {
namespace grouped {

static const int kMaxGroups = 1024;
static const int kMaxExtent = 0x7FFFFF00;   // an extent rounded up to a tile's edge stays within 32 bits
static const int kTileList = 128;   // tiles of a unit that are looked up once, when the kernel starts
enum : int { KIND_BF16 = 0, KIND_E4M3 = 2 };   // the KIND of ptx::umma
// What a kernel instance writes.  One instance for each: the code of another form, never run, takes registers
// that the loop over K blocks needs (spills there cost a sixth of the throughput).
enum : int { OUT_BF16 = 0, OUT_PAIR_BF16 = 1, OUT_F32 = 2, OUT_PAIR_F32 = 3, OUT_COUNT = 4 };

struct alignas(64) Params {
  CUtensorMap tm_a;      // [M][K], box {128 bytes of K, 128 rows}
  CUtensorMap tm_a32;    // the same with boxes of 32 rows, for tiles with few rows
  CUtensorMap tm_b;      // [G][K][N], box {128 bytes of N, K rows of one stage}; or [G][N][K], box {128 bytes of K, 128 rows}
  CUtensorMap tm_d;      // [M][columns of D], box {64 bytes, 32 rows}, 64-byte swizzle; unused where vec_d == 0
  int M, N, K, G;
  int tiles_n, num_kb;
  int group_m;           // rasterisation: row tiles per column sweep
  int b_nk, b_grouped;   // b_grouped 0: all groups share one weight
  const int* offsets;    // [G + 1], null: one group of all M rows
  const float* sa;
  const float* sb;
  long long sa_row, sa_blk, sb_k, sb_n, sb_group;
  void* D;
  long long ldd;
  int pair;
  int vec_d;             // rows of D start on 16-byte boundaries: TMA may write them
  int* status;
  long long wait_budget;
  // Tiles whose K range several units share (split_kb > 0: see Split): one flag per epilogue warp and one
  // slot of partial sums per CTA.
  int split_kb;          // what sharing a tile between two units costs, in K blocks of one unit
  int split_max;         // most units that share a tile: they are summed one by one
  int* flags;            // [grid][8], zero between launches, raised by one
  float4* partials;      // [grid][8 warps][columns of a warp / 4][32 lanes]
};

template <int KIND_, int BN_, int CTAS_>
struct Cfg {
  static constexpr int KIND = KIND_, BN = BN_, CTAS = CTAS_;
  static constexpr int TM = 128 * CTAS;                 // rows of a tile
  static constexpr int ES = KIND == KIND_BF16 ? 2 : 1;
  static constexpr int KBLK = 128 / ES;                 // K elements of a stage: one 128-byte slab
  // K blocks summed in TMEM before the sum moves to registers: one where each has its scales; with bf16 four (256
  // elements), because the tensor core truncates as it adds: in one piece, K = 4236 to 7572 is 8e-6 of the
  // result off, in pieces 2e-7 to 5e-7, like a sum of rounded products.  4096 x 4096 x 4096 takes 1 % longer.
  static constexpr int SEG = KIND == KIND_E4M3 ? 1 : 4;
  static constexpr int UK = 32 / ES;                    // K elements of one MMA
  static constexpr int BN_CTA = BN / CTAS;              // columns of B one CTA loads
  static constexpr int GRP_COLS = 128 / ES;             // columns of a 128-byte column group ([K][N] weights)
  static constexpr int GRP_BYTES = KBLK * 128;
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BN_CTA * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = CTAS == 2 ? 4 : BN == 256 ? 3 : 5;
  static constexpr int NBUF = 512 / BN;                 // accumulators in TMEM
  static constexpr int NC = BN / 2;                     // columns per epilogue warp
  static constexpr bool SPLIT_REGS = NC == 128;
  static constexpr int STG_BUFS = NC / 32;        // staging buffers per epilogue warp: 32 rows x 64 bytes
  static constexpr int STG_BYTES = STG_BUFS * 2048;
  static constexpr int BAR_BYTES = 256;
  static constexpr int TAB_BYTES = (kMaxGroups + 1 + 2 * kMaxGroups) * 4;   // first tile, {first row, rows} of a group
  static constexpr int LIST_BYTES = kTileList * 16;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + 8 * STG_BYTES + BAR_BYTES + LIST_BYTES + TAB_BYTES;
  static_assert(BN_CTA % 128 == 0, "B is loaded in boxes of 128 columns");
  static_assert(NC == 64 || NC == 128, "an epilogue warp's columns share one scale of B");
  static_assert(SMEM_BYTES + 1024 <= 227 * 1024, "shared memory, with what is static in front of it");
};

// The tile of index t: group, first row of A and D, rows of the group from there on, first column.
struct Tile {
  int g, row0, rows, n0;
};

template <class C>
__device__ __forceinline__ Tile decode(const Params& p, const int* first, const int* row0, int t) {
  int lo = 0, hi = p.G;                      // last group whose first tile is not behind t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= t) lo = mid; else hi = mid;
  }
  Tile x;
  x.g = lo;
  const int r = t - first[lo];
  const int tiles_m = (first[lo + 1] - first[lo]) / p.tiles_n;
  const int sweep = p.group_m * p.tiles_n;
  const int s = r / sweep, rr = r - s * sweep;
  const int h = min(p.group_m, tiles_m - s * p.group_m);
  const int tn = rr / h, tm = s * p.group_m + rr - tn * h;
  x.row0 = row0[2 * lo] + tm * C::TM;
  x.rows = row0[2 * lo + 1] - tm * C::TM;
  x.n0 = tn * C::BN;
  return x;
}

// One work item: K blocks [kb0, kb1) of a tile.
struct Item {
  int tile, kb0, kb1;
};

// The work items of one unit (a CTA, or a pair of them).  Unit u takes the whole tiles u, u + U, ... of the full
// waves.  The R tiles of the last, partly filled wave are laid end to end, R * num_kb blocks, and cut into
// equal ranges, one for each of `sharers` units, if that saves more than the exchange of partial sums
// costs (split_kb).  A unit walks its range backwards and before its whole tiles: the piece at the
// range's end, which may lack the tile's last blocks, is published at once; the piece at its start, which
// then has the tile's last block, collects what the units below it published.  So a unit only ever waits for
// units of lower index, which never wait before they publish: the wait ends whatever else runs on the GPU.
struct Split {
  int whole;        // tiles of full waves
  int sharers;      // units that share the others
  int lo, hi;       // this unit's range
  // Start of unit u's range: blocks * u / sharers, in 32 bits (a 64-bit division is a call, and what lives in
  // registers around it is spilled).  The host keeps num_kb below 2^20.
  __device__ __forceinline__ static int bound(unsigned blocks, unsigned sharers, unsigned u) {
    const unsigned q = blocks / sharers;
    return static_cast<int>(q * u + (blocks - q * sharers) * u / sharers);
  }
  __device__ __forceinline__ void set(const Params& p, int tiles, int unit, int units) {
    const int rest = tiles % units;
    whole = tiles;
    sharers = lo = hi = 0;
    if (p.split_kb == 0 || rest == 0) return;
    // At least 4 blocks for each unit, and where two or more units go to a tile the same number to each: a
    // range that touches two tiles adds a sharer.
    int n = min(min(units, p.split_max * rest), rest * p.num_kb / 4);
    if (n >= 2 * rest) n -= n % rest;
    if (n <= rest || (n - rest) * static_cast<long long>(p.num_kb) <= static_cast<long long>(p.split_kb) * n) return;
    sharers = n;
    whole = tiles - rest;
    if (unit >= n) return;
    lo = bound(rest * p.num_kb, n, unit);
    hi = bound(rest * p.num_kb, n, unit + 1);
  }
};
// What the roles of a CTA have begun, for its end where a wait has run out.
struct Begun {
  int gave_up;          // a role of this CTA, or of the other one of a pair, did
  int sent, sent_other; // K blocks copied here, and by the other CTA (known to the leader)
  int issued, filled;   // K blocks multiplied, accumulators handed over (known to both)
};
// Waits until the last of `uses` completions of a ring of N barriers, one after another, has arrived at each of them.
template <int N>
__device__ __forceinline__ void wait_ring(uint64_t* ring, int uses, long long budget) {
#pragma unroll 1
  for (int s = 0; s < N && s < uses; ++s)
    ptx::mbar_wait(ptx::smem_u32(&ring[s]), static_cast<uint32_t>((uses - 1 - s) / N) & 1u, budget);
}
// A role's walk over them; the split stays in shared memory, out of the role's registers.
struct Walk {
  int next_tile, pos, count;   // count: items taken, the place of the next one's tile in the list
  __device__ __forceinline__ bool next(const Params& p, const Split& s, int units, Item& it) {
    ++count;
    if (pos > s.lo) {
      const int t = (pos - 1) / p.num_kb, start = t * p.num_kb;
      it.tile = ptx::uniform(s.whole + t);
      it.kb1 = ptx::uniform(pos - start);
      it.kb0 = ptx::uniform(max(s.lo - start, 0));
      pos = max(s.lo, start);
      return true;
    }
    if (next_tile >= ptx::uniform(s.whole)) return false;
    it.tile = next_tile;
    it.kb0 = 0;
    it.kb1 = p.num_kb;
    next_tile += units;
    return true;
  }
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two fp32 values in one 64-bit register pair.
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  return v;
}
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t x, uint64_t f) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(x), "l"(f));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, float lo, float hi) {
  return pair_of(__float_as_uint(lo_of(a) + lo), __float_as_uint(hi_of(a) + hi));
}
// acc += r * f for the 16 words r of a TMEM slice, two columns per instruction; f holds the factor twice.
__device__ __forceinline__ void scale_add(uint64_t* acc, const uint4 (&r)[4], uint64_t f) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    fma2(acc[2 * j], pair_of(r[j].x, r[j].y), f);
    fma2(acc[2 * j + 1], pair_of(r[j].z, r[j].w), f);
  }
}

// Puts 64 bytes of a row per lane into one of the warp's staging buffers, in the 64-byte swizzle of the
// store's tensor map (16-byte chunk j of row r at j ^ (r / 2 % 4)), which also keeps the banks apart.
__device__ __forceinline__ void stage_row64(uint8_t* buf, int lane, const uint32_t (&w)[16]) {
  uint8_t* mine = buf + lane * 64;
  const int sw = (lane >> 1) & 3;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(mine + ((j ^ sw) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}

// Writes the first `rows` of the 32 staged rows to row-major global memory: for row blocks that end inside a
// group's last tile, and for rows that a tensor map cannot address.  Four lanes per row with 16 bytes each
// where rows allow it, else neighbouring lanes write neighbouring elements.  ES: bytes per element.
template <int ES>
__device__ __forceinline__ void copy_rows64(const uint8_t* buf, int lane, char* d, long long pitch, int rows, int col,
                                            int ncols, int vec) {
  rows = min(rows, 32);
  if (vec && col + 64 / ES <= ncols) {
    const int ch = lane & 3;
#pragma unroll 1
    for (int r = lane >> 2; r < rows; r += 8)
      *reinterpret_cast<uint4*>(d + r * pitch + static_cast<long long>(col) * ES + ch * 16) =
          *reinterpret_cast<const uint4*>(buf + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4));
    return;
  }
  constexpr int PER_ROW = 64 / ES, STEP = 32 / PER_ROW;   // elements of a row; rows a warp writes at a time
  const int e = lane % PER_ROW;
  if (col + e >= ncols) return;
  char* q = d + static_cast<long long>(col + e) * ES;
#pragma unroll 4
  for (int r = lane / PER_ROW; r < rows; r += STEP) {
    const uint8_t* s = buf + r * 64 + ((((e * ES) >> 4) ^ ((r >> 1) & 3)) << 4) + ((e * ES) & 15);
    if (ES == 4) *reinterpret_cast<uint32_t*>(q + r * pitch) = *reinterpret_cast<const uint32_t*>(s);
    else *reinterpret_cast<uint16_t*>(q + r * pitch) = *reinterpret_cast<const uint16_t*>(s);
  }
}

template <int KIND, int BN, int CTAS, int OUT>
__global__ void __launch_bounds__(384, 1) grouped_gemm_kernel(const __grid_constant__ Params p) {
  using C = Cfg<KIND, BN, CTAS>;
  constexpr int STAGES = C::STAGES, NBUF = C::NBUF, NC = C::NC;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ Begun begun;
  const uint32_t raw = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* staging = smem + STAGES * C::STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + 8 * C::STG_BYTES);
  uint64_t* full_bar = bars;                     // [STAGES] operands landed (the leader CTA's is used; each CTA of a pair
                                                 //          announces and counts its own copies there)
  uint64_t* empty_bar = bars + STAGES;           // [STAGES] MMAs have read the stage
  uint64_t* tfull_bar = bars + 2 * STAGES;       // [NBUF]   accumulator complete
  uint64_t* tempty_bar = tfull_bar + NBUF;       // [NBUF]   accumulator read out (the leader CTA's is used)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + NBUF);
  Tile* list = reinterpret_cast<Tile*>(staging + 8 * C::STG_BYTES + C::BAR_BYTES);  // [kTileList] this unit's tiles
  int* first = reinterpret_cast<int*>(list + kTileList);   // [G + 1] first tile of a group
  Split* split = reinterpret_cast<Split*>(tmem_slot + 1);
  int* grow = first + kMaxGroups + 1;            // [G][2] first row, rows

  const int warp = ptx::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = CTAS > 1 ? ptx::cluster_ctarank() : 0u;
  const int unit = CTAS > 1 ? static_cast<int>(ptx::cluster_id_x()) : blockIdx.x;
  const int units = CTAS > 1 ? static_cast<int>(ptx::num_clusters_x()) : gridDim.x;

  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&p.tm_a);
    ptx::prefetch_tmap(&p.tm_a32);
    ptx::prefetch_tmap(&p.tm_b);
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[s]), CTAS);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1);
    }
    for (int b = 0; b < NBUF; ++b) {
      ptx::mbar_init(ptx::smem_u32(&tfull_bar[b]), 1);
      ptx::mbar_init(ptx::smem_u32(&tempty_bar[b]), 8 * CTAS);
    }
    ptx::fence_mbar_init();
    begun.gave_up = 0;
  }
  if (warp == 2) {
    ptx::tmem_alloc<CTAS>(ptx::smem_u32(tmem_slot), 512);
    ptx::tmem_relinquish<CTAS>();
  }
  // Everything above touched neither global memory nor what the previous kernel of the stream writes.
  ptx::griddep_launch_dependents();
  if (p.offsets) ptx::griddep_wait();

  // Rows of each group, clamped to the rows there are: whatever the offsets hold, no tile leaves A and D.
  for (int g = threadIdx.x; g < p.G; g += 384) {
    int lo = 0, hi = p.M;
    if (p.offsets) {
      lo = min(max(p.offsets[g], 0), p.M);
      hi = min(max(p.offsets[g + 1], lo), p.M);
    }
    grow[2 * g] = lo;
    grow[2 * g + 1] = hi - lo;
  }
  __syncthreads();
  if (warp == 3) {                               // first tile of each group: a running sum, 32 groups at a time
    int base = 0;
    for (int g0 = 0; g0 < p.G; g0 += 32) {
      const int g = g0 + lane;
      int n = g < p.G ? (grow[2 * g + 1] + C::TM - 1) / C::TM * p.tiles_n : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += up;
      }
      if (g < p.G) first[g + 1] = base + n;
      base += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) {
      first[0] = 0;
      split->set(p, base, unit, units);
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CTAS > 1) {
    ptx::cluster_arrive_relaxed();
    ptx::cluster_wait();
  }
  ptx::tc_fence_after();
  // Where a unit takes several tiles, one thread looks up each of them now: every role would do it in turn,
  // between tiles (64 groups, 16384 x 4096 x 2048: 275 -> 250 us; a single tile starts 1 us sooner without).
  const int listed = ptx::uniform(first[p.G]) > 2 * units ? kTileList : 0;
  if (listed) {
    const int shared_tiles = split->hi > split->lo ? (split->hi - 1) / p.num_kb - split->lo / p.num_kb + 1 : 0;
    for (int i = threadIdx.x; i < kTileList; i += 384) {
      const int tile = i < shared_tiles ? split->whole + (split->hi - 1) / p.num_kb - i : unit + (i - shared_tiles) * units;
      if (i < shared_tiles || tile < split->whole) list[i] = decode<C>(p, first, grow, tile);
    }
    __syncthreads();
  }
  if (!p.offsets) ptx::griddep_wait();
  const uint32_t tmem = ptx::uniform(*reinterpret_cast<volatile uint32_t*>(tmem_slot));
  Walk sched = {unit, ptx::uniform(split->hi), 0};
  Item it;
  ptx::Waiter<Params> w = {p, &begun.gave_up, false};

  // 128 sums and two slices of 16 columns per thread do not fit the 168 registers that 384 threads can have
  // each: the first four warps hand theirs over (72 + 2 x 216 = 3 x 168).
  if constexpr (C::SPLIT_REGS) {
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  }
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    int stage = 0, sent = 0;
    uint32_t phase = 0;
    while (sched.next(p, *split, units, it)) {
      const Tile x = sched.count <= listed ? list[sched.count - 1] : decode<C>(p, first, grow, it.tile);
      // rows of A that this CTA needs, in boxes of 32 (4: one box of 128), and the bytes that it loads
      const int boxes = min(max((x.rows - static_cast<int>(rank) * 128 + 31) / 32, 0), 4);
      const uint32_t bytes = boxes * 4096 + C::B_BYTES;
      const int row = x.row0 + static_cast<int>(rank) * 128;
      const int col = x.n0 + static_cast<int>(rank) * C::BN_CTA;
      const int bg = p.b_grouped ? x.g : 0;
      for (int kb = it.kb0; kb < it.kb1; ++kb) {
        w.wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1u, DEV_TIMEOUT_PRODUCER_EMPTY);
        // once a wait has run out nothing more is loaded: a stage's barrier may still be in its last phase
        const bool go = !w.any_lost();
        if (go && ptx::elect_one()) {
          const uint32_t own = ptx::smem_u32(&full_bar[stage]);
          const uint32_t bar = CTAS == 2 ? ptx::mapa(own, 0) : own;
          if constexpr (CTAS == 2) ptx::mbar_arrive_expect_tx_cluster(bar, bytes);
          else ptx::mbar_arrive_expect_tx(own, bytes);
          const uint32_t sa = ptx::smem_u32(smem + stage * C::STAGE_BYTES), sb = sa + C::A_BYTES;
          const int k = kb * C::KBLK;
          if (boxes == 4) {
            ptx::tma_load_3d<CTAS>(sa, &p.tm_a, bar, k, row, 0);
          } else {
            for (int b = 0; b < boxes; ++b) ptx::tma_load_3d<CTAS>(sa + b * 4096, &p.tm_a32, bar, k, row + b * 32, 0);
          }
          if (p.b_nk) {
#pragma unroll
            for (int c = 0; c < C::BN_CTA / 128; ++c)
              ptx::tma_load_3d<CTAS>(sb + c * 16384, &p.tm_b, bar, k, col + c * 128, bg);
          } else {
#pragma unroll
            for (int c = 0; c < C::BN_CTA / C::GRP_COLS; ++c)
              ptx::tma_load_3d<CTAS>(sb + c * C::GRP_BYTES, &p.tm_b, bar, col + c * C::GRP_COLS, k, bg);
          }
        }
        __syncwarp();
        sent += go;
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
    }
    // The last stages have been read, so their copies have landed, and the commits that say so have arrived here.
    // (Rolled up: code that runs once comes cold from memory; unrolled, the loops here took 0.5 us.)
#pragma unroll 1
    for (int s = 0; s < STAGES; ++s)
      w.wait(ptx::smem_u32(&empty_bar[s]), s < stage ? phase : phase ^ 1u, DEV_TIMEOUT_PRODUCER_EMPTY);
    if (lane == 0) begun.sent = sent;
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    // The whole warp walks the loop and one elected lane issues: addresses and descriptors then stay in
    // uniform registers (with one lane in the loop, an MMA took 110 clocks to issue).
    if (rank == 0) {
      // D fp32, A and B bf16 (1) or e4m3 (0), A K-major, B N-major unless the weights are [N][K]
      constexpr uint32_t fmt = KIND == KIND_BF16 ? 1u : 0u;
      const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((p.b_nk ? 0u : 1u) << 16) |
                             (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>(C::TM >> 4) << 24);
      const uint32_t b_lbo = p.b_nk ? 16u : static_cast<uint32_t>(C::GRP_BYTES);
      const uint64_t b_step = p.b_nk ? 2u : static_cast<uint64_t>(C::UK * 128) >> 4;   // per MMA, in 16 bytes
      const uint32_t smem0 = ptx::smem_u32(smem), full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
      const uint32_t tfull0 = ptx::smem_u32(tfull_bar), tempty0 = ptx::smem_u32(tempty_bar);
      int stage = 0, buf = 0, issued = 0, filled = 0;
      uint32_t phase = 0, tphase = 0;
      while (sched.next(p, *split, units, it)) {
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          const bool fresh = (kb - it.kb0) % C::SEG == 0;                            // starts an accumulator
          const bool done = (kb - it.kb0) % C::SEG == C::SEG - 1 || kb + 1 == it.kb1;   // and completes it
          w.wait(full0 + stage * 8, phase, DEV_TIMEOUT_MMA_FULL);
          const uint32_t sa = smem0 + stage * C::STAGE_BYTES;
          const uint64_t adesc = ptx::make_smem_desc_sw128(sa, 16, 1024);
          const uint64_t bdesc = ptx::make_smem_desc_sw128(sa + C::A_BYTES, b_lbo, 1024);
          const uint32_t d = tmem + static_cast<uint32_t>(buf * BN);
          // last of all, the wait that the promotion warps answer: what follows it is on their round trip
          if (fresh) w.wait(tempty0 + buf * 8, tphase ^ 1u, DEV_TIMEOUT_MMA_TMEM_EMPTY);
          const bool lost = w.any_lost();
          ptx::tc_fence_after();
          if (!lost && ptx::elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              ptx::umma<KIND, CTAS>(d, adesc + static_cast<uint64_t>(2 * k), bdesc + k * b_step, idesc,
                                    (!fresh || k > 0) ? 1u : 0u);
            if constexpr (CTAS == 2) {
              if (done) ptx::umma_commit_pair(tfull0 + buf * 8);
              ptx::umma_commit_pair(empty0 + stage * 8);
            } else {
              if (done) ptx::umma_commit<1>(tfull0 + buf * 8);
              ptx::umma_commit<1>(empty0 + stage * 8);
            }
          }
          __syncwarp();
          issued += !lost;
          filled += done && !lost;
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          if (done && ++buf == NBUF) { buf = 0; tphase ^= 1u; }
        }
      }
      // The last accumulators have been read, and the other CTA's arrivals that say so have come in.
#pragma unroll 1
      for (int b = 0; b < NBUF; ++b)
        w.wait(tempty0 + b * 8, b < buf ? tphase : tphase ^ 1u, DEV_TIMEOUT_MMA_TMEM_EMPTY);
      if (lane == 0) {
        begun.issued = issued;
        begun.filled = filled;
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ promotion and epilogue
    if constexpr (C::SPLIT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint8_t* stg = staging + (warp - 4) * C::STG_BYTES;
    const uint32_t lead = CTAS == 2 ? ptx::mapa(ptx::smem_u32(&tempty_bar[0]), 0) : ptx::smem_u32(&tempty_bar[0]);
    const uint32_t t_base = tmem + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(half * NC);
    const int ncols = OUT == OUT_PAIR_BF16 || OUT == OUT_PAIR_F32 ? p.N >> 1 : p.N;
    const uint32_t tfull0 = ptx::smem_u32(tfull_bar);
    int buf = 0;
    uint32_t tphase = 0;
    // A tile as this warp sees it: its place, and where its block scales are (the first two on their way).
    // (Entering the next tile before the results of the last one have left costs registers that the loop over
    // K blocks then lacks: 404 -> 482 us at 4096 x 28672 x 4096.)
    Tile x;
    int roff = static_cast<int>(rank) * 128 + q * 32, rows = 0, col = 0;   // rows: of the group, from the warp's first on
    bool live = false;                                                    // the warp has outputs here
    const float* sa = nullptr;
    const float* sb = nullptr;
    float a0 = 0.0f, b0 = 0.0f, a1 = 0.0f, b1 = 0.0f;
    auto enter = [&]() {
      x = sched.count <= listed ? list[sched.count - 1] : decode<C>(p, first, grow, it.tile);
      rows = x.rows - roff;
      col = x.n0 + half * NC;
      live = rows > 0 && col < p.N;
      if (KIND == KIND_E4M3 && live) {
        sa = p.sa + (static_cast<long long>(x.row0) + roff + min(lane, rows - 1)) * p.sa_row + it.kb0 * p.sa_blk;
        sb = p.sb + static_cast<long long>(x.g) * p.sb_group + static_cast<long long>(col >> 7) * p.sb_n + it.kb0 * p.sb_k;
        a0 = ptx::ld_early(sa);
        b0 = ptx::ld_early(sb);
        if (it.kb0 + 1 < it.kb1) {
          a1 = ptx::ld_early(sa + p.sa_blk);
          b1 = ptx::ld_early(sb + p.sb_k);
        }
      }
    };
    bool more = sched.next(p, *split, units, it);
    if (more) enter();
    while (more) {
      uint64_t sum[NC / 2];                    // columns 2 i and 2 i + 1
#pragma unroll
      for (int i = 0; i < NC / 2; ++i) sum[i] = 0;
      const int last = it.kb1 - 1, segs = (it.kb1 - it.kb0 + C::SEG - 1) / C::SEG;
      auto open = [&]() {
        w.wait(tfull0 + buf * 8, tphase, DEV_TIMEOUT_EPI_TMEM_FULL);
        __syncwarp();
        ptx::tc_fence_after();
      };
      auto release = [&]() {
        ptx::tc_fence_before();
        if (lane == 0) ptx::mbar_arrive_cluster_relaxed(lead + static_cast<uint32_t>(buf * 8));
        if (++buf == NBUF) { buf = 0; tphase ^= 1u; }
      };
      // The tile's accumulators one after another, in slices of 16 columns: while a slice is scaled and added,
      // the next one is on its way out of TMEM.  A buffer is free once its last slice has been read.
      auto take = [&](float factor) {
        uint4 r[2][4];
        const uint64_t f = pair_of(__float_as_uint(factor), __float_as_uint(factor));
        open();
        const uint32_t t0 = t_base + static_cast<uint32_t>(buf * BN);
        ptx::tmem_ld_32x16_async(t0, r[0]);
#pragma unroll
        for (int c = 0; c < NC / 16; ++c) {
          ptx::tmem_ld_wait_for(r[c & 1]);
          if (c + 1 < NC / 16) ptx::tmem_ld_32x16_async(t0 + static_cast<uint32_t>((c + 1) * 16), r[(c + 1) & 1]);
          else release();
          scale_add(&sum[c * 8], r[c & 1], f);
        }
      };
      if (!live) {                                // nothing to add, but every accumulator is released by all
        for (int s = 0; s < segs; ++s) {
          open();
          release();
        }
      } else if constexpr (KIND == KIND_BF16) {
#pragma unroll 1
        for (int s = 0; s < segs; ++s) take(1.0f);
      } else {
        // Block scales are asked for two blocks ahead of their use.
#pragma unroll 1
        for (int kb = it.kb0; kb <= last; kb += 2) {
          sa += 2 * p.sa_blk;
          sb += 2 * p.sb_k;
          const float f0 = a0 * b0;
          if (kb + 2 <= last) {
            a0 = ptx::ld_early(sa);
            b0 = ptx::ld_early(sb);
          }
          take(f0);
          if (kb == last) break;
          const float f1 = a1 * b1;
          if (kb + 3 <= last) {
            a1 = ptx::ld_early(sa + p.sa_blk);
            b1 = ptx::ld_early(sb + p.sb_k);
          }
          take(f1);
        }
      }
      if (it.kb1 < p.num_kb) {
        // Not the tile's last blocks: the sums go to this CTA's slot, in a layout in which a warp's lanes are side by side.
        float4* slot = p.partials + (static_cast<size_t>(blockIdx.x) * 8 + (warp - 4)) * (NC / 4) * 32 + lane;
        if (live && lane < rows) {
#pragma unroll
          for (int i = 0; i < NC / 4; ++i)
            slot[i * 32] = make_float4(lo_of(sum[2 * i]), hi_of(sum[2 * i]), lo_of(sum[2 * i + 1]), hi_of(sum[2 * i + 1]));
        }
        __syncwarp();
        if (live && lane == 0) ptx::add_release_gpu(p.flags + blockIdx.x * 8 + (warp - 4), 1);
        live = false;
      } else if (it.kb0 > 0 && live) {
        // The tile's last blocks: the units below hold the rest, nearest first, down to the one with block 0.
        const int blocks = (first[p.G] - split->whole) * p.num_kb, start = (it.tile - split->whole) * p.num_kb;
        int count = 1;
        while (Split::bound(blocks, split->sharers, unit - count) > start) ++count;
        // one lane for each of them, all flags at once; then their sums, nearest unit first
        int* flag = p.flags + ((unit - 1 - min(lane, count - 1)) * CTAS + static_cast<int>(rank)) * 8 + (warp - 4);
        w.wait_flags(flag, DEV_TIMEOUT_SPLIT_PARTIALS);
        __syncwarp();                            // what one lane's flag announces is read by all
#pragma unroll 1
        for (int u = 1; u <= count; ++u) {
          const int cta = (unit - u) * CTAS + static_cast<int>(rank);
          // lanes without a row add what the first lane's holds: no branch around 128 registers
          const float4* slot = p.partials + (static_cast<size_t>(cta) * 8 + (warp - 4)) * (NC / 4) * 32 + (lane < rows ? lane : 0);
#pragma unroll
          for (int i = 0; i < NC / 4; ++i) {
            const float4 f = __ldcg(slot + i * 32);
            sum[2 * i] = add2(sum[2 * i], f.x, f.y);
            sum[2 * i + 1] = add2(sum[2 * i + 1], f.z, f.w);
          }
        }
        __syncwarp();
        if (lane < count) *reinterpret_cast<volatile int*>(flag) = 0;   // for the next launch
      }
      const int wcol = OUT == OUT_PAIR_BF16 || OUT == OUT_PAIR_F32 ? col >> 1 : col, drow = x.row0 + roff;
      // 64 bytes of each row make a unit; as many as there are buffers are staged before one fence hands them to
      // the store engine
      constexpr bool F32 = OUT == OUT_F32 || OUT == OUT_PAIR_F32, PAIR = OUT == OUT_PAIR_BF16 || OUT == OUT_PAIR_F32;
      constexpr int UNIT = (F32 ? 16 : 32) * (PAIR ? 2 : 1);     // sums that make 64 bytes of D
      constexpr int COLS = F32 ? 16 : 32;
      constexpr int ROUND = NC / UNIT < C::STG_BUFS ? NC / UNIT : C::STG_BUFS;
      const bool tma = p.vec_d && rows >= 32;    // a tensor map's box has 32 rows, all of this group
#pragma unroll
      for (int u0 = 0; u0 < NC / UNIT; u0 += ROUND) {
        if (wcol + u0 * COLS >= ncols || !live) break;
        if (lane == 0) ptx::tma_store_wait_read<0>();   // the last round's stores have read the buffers
        __syncwarp();
#pragma unroll
        for (int u = u0; u < u0 + ROUND; ++u) {
          float v[COLS];
          const uint64_t* s = &sum[u * (UNIT / 2)];
          if constexpr (!PAIR) {
#pragma unroll
            for (int i = 0; i < UNIT / 2; ++i) {
              v[2 * i] = lo_of(s[i]);
              v[2 * i + 1] = hi_of(s[i]);
            }
          } else if (p.pair == PAIR_SWIGLU) {      // the choice outside the loops: their elements interleave
#pragma unroll
            for (int i = 0; i < UNIT / 2; ++i) v[i] = silu_fast(lo_of(s[i])) * hi_of(s[i]);
          } else {
#pragma unroll
            for (int i = 0; i < UNIT / 2; ++i) v[i] = gelu_rel(lo_of(s[i])) * hi_of(s[i]);
          }
          uint32_t words[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) words[i] = F32 ? __float_as_uint(v[i]) : pack_bf16(v[2 * i % COLS], v[(2 * i + 1) % COLS]);
          stage_row64(stg + (u - u0) * 2048, lane, words);
        }
        if (tma) ptx::fence_proxy_async_smem();
        __syncwarp();
#pragma unroll
        for (int u = u0; u < u0 + ROUND; ++u) {
          const int c = wcol + u * COLS;
          if (c >= ncols) break;
          if (!tma) {
            const long long pitch = p.ldd * (F32 ? 4 : 2);
            copy_rows64<F32 ? 4 : 2>(stg + (u - u0) * 2048, lane, static_cast<char*>(p.D) + drow * pitch, pitch, rows, c, ncols, p.vec_d);
          } else if (lane == 0) {
            ptx::tma_store_3d(&p.tm_d, ptx::smem_u32(stg + (u - u0) * 2048), c, drow, 0);
          }
        }
        if (lane == 0) ptx::tma_store_commit();
      }
      more = sched.next(p, *split, units, it);
      if (more) enter();
    }
    if (lane == 0) ptx::tma_store_wait_read<0>();   // the staging buffers have been read before the CTA goes
  }

  // ------------------------------------------------------------------ teardown
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  // No CTA leaves while its peer may still write its barriers or read the pair's TMEM.
  if constexpr (CTAS > 1) {
    if (threadIdx.x == 0 && begun.gave_up) {       // both learn of it
      ptx::st_shared_cluster(ptx::mapa(ptx::smem_u32(&begun.gave_up), rank ^ 1u), 1);
      ptx::fence_cluster();
    }
    __syncwarp();
    ptx::cluster_arrive_relaxed();
    ptx::cluster_wait();
  }
  if (begun.gave_up) {
    // Roles that gave up stopped at different blocks, so copies, MMAs and commits may be on their way that nobody
    // waited for.  What was begun says which of them have to arrive before the shared memory and TMEM may go.
    if constexpr (CTAS > 1) {
      if (warp == 0 && lane == 0) {
        if (rank != 0) {
          ptx::st_shared_cluster(ptx::mapa(ptx::smem_u32(&begun.sent_other), 0), begun.sent);
        } else {
          ptx::st_shared_cluster(ptx::mapa(ptx::smem_u32(&begun.issued), 1), begun.issued);
          ptx::st_shared_cluster(ptx::mapa(ptx::smem_u32(&begun.filled), 1), begun.filled);
        }
      }
      __syncwarp();
      ptx::cluster_arrive();
      ptx::cluster_wait();
    }
    if (warp == 0 && rank == 0) {
      int sent = begun.sent;
      if constexpr (CTAS > 1) {
        // A block that only one CTA copied lacks the other one's announcement.  (One CTA is at most STAGES blocks ahead:
        // a stage is filled again only after MMAs have read what both had put there.)
        const int from = min(sent, begun.sent_other);
        sent = max(sent, begun.sent_other);
        for (int b = from + lane; b < sent; b += 32) ptx::mbar_arrive(ptx::smem_u32(&full_bar[b % STAGES]));
        __syncwarp();
      }
      wait_ring<STAGES>(full_bar, sent, p.wait_budget);
    } else if (warp == 1) {
      wait_ring<STAGES>(empty_bar, begun.issued, p.wait_budget);
      wait_ring<NBUF>(tfull_bar, begun.filled, p.wait_budget);
    }
    __syncwarp();
    if constexpr (CTAS > 1) {
      ptx::cluster_arrive();
      ptx::cluster_wait();
    } else {
      __syncthreads();
    }
  }
  if (warp == 2) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<CTAS>(tmem, 512);
  }
}

// Kernel instances by output form, in the order of the tile variants below; defined in xf_grouped_gemm_bf16.cu
// and xf_grouped_gemm_e4m3.cu.
typedef void (*KernelFn)(const Params);
struct Variant {
  int kind, bn, ctas, smem;
  KernelFn fn[OUT_COUNT];
  const char* name;
};
#define XF_GROUPED_VARIANT(KIND, BN, CTAS, NAME)                                                          \
  {KIND, BN, CTAS, Cfg<KIND, BN, CTAS>::SMEM_BYTES,                                                      \
   {grouped_gemm_kernel<KIND, BN, CTAS, OUT_BF16>, grouped_gemm_kernel<KIND, BN, CTAS, OUT_PAIR_BF16>,   \
    grouped_gemm_kernel<KIND, BN, CTAS, OUT_F32>, grouped_gemm_kernel<KIND, BN, CTAS, OUT_PAIR_F32>},    \
   NAME}
static const int kTilesBf16 = 2, kTilesE4m3 = 3;
extern const Variant g_variants_bf16[kTilesBf16], g_variants_e4m3[kTilesE4m3];

}  // namespace grouped
}  // namespace xf
