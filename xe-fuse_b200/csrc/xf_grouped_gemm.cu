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
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>

#include "../../include/xefuse_b200.h"
#include "xf_act.cuh"
#include "xf_host_util.h"
#include "xf_params.h"
#include "xf_ptx.cuh"

namespace xf {
namespace grouped {

static const int kMaxGroups = 1024;
enum : int { KIND_BF16 = 0, KIND_E4M3 = 2 };   // the KIND of ptx::umma

struct alignas(64) Params {
  CUtensorMap tm_a;      // [M][K], box {128 bytes of K, 128 rows}
  CUtensorMap tm_a32;    // the same with boxes of 32 rows, for tiles with few rows
  CUtensorMap tm_b;      // [G][K][N], box {128 bytes of N, K rows of one stage}; or [G][N][K], box {128 bytes of K, 128 rows}
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
  int d_f32, pair, vec_d;
  int* status;
  long long wait_budget;
};

template <int KIND_, int BN_, int CTAS_>
struct Cfg {
  static constexpr int KIND = KIND_, BN = BN_, CTAS = CTAS_;
  static constexpr int TM = 128 * CTAS;                 // rows of a tile
  static constexpr int ES = KIND == KIND_BF16 ? 2 : 1;
  static constexpr int KBLK = 128 / ES;                 // K elements of a stage: one 128-byte slab
  static constexpr int UK = 32 / ES;                    // K elements of one MMA
  static constexpr int BN_CTA = BN / CTAS;              // columns of B one CTA loads
  static constexpr int GRP_COLS = 128 / ES;             // columns of a 128-byte column group ([K][N] weights)
  static constexpr int GRP_BYTES = KBLK * 128;
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BN_CTA * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 6;
  static constexpr int NBUF = 512 / BN;                 // accumulators in TMEM
  static constexpr int NC = BN / 2;                     // columns per epilogue warp
  static constexpr bool SPLIT_REGS = NC == 128;
  static constexpr int STG_BYTES = 2048;                // staging per epilogue warp: 32 rows x 64 bytes
  static constexpr int BAR_BYTES = 256;
  static constexpr int TAB_BYTES = (kMaxGroups + 1 + 2 * kMaxGroups) * 4;   // first tile, {first row, rows} of a group
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + 8 * STG_BYTES + BAR_BYTES + TAB_BYTES;
  static_assert(BN_CTA == 128, "a CTA loads 128 columns of B");
  static_assert(NC % 64 == 0 && NC <= 128, "an epilogue warp's columns share one scale of B");
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
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
struct Schedule {
  int next_tile, step, tiles, num_kb;
  __device__ __forceinline__ bool next(Item& it) {
    if (next_tile >= tiles) return false;
    it.tile = next_tile;
    it.kb0 = 0;
    it.kb1 = num_kb;
    next_tile += step;
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
// acc += r * f for the 16 words r of a TMEM slice, two columns per instruction; f holds the factor twice.
__device__ __forceinline__ void scale_add(uint64_t* acc, const uint4 (&r)[4], uint64_t f) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    fma2(acc[2 * j], pair_of(r[j].x, r[j].y), f);
    fma2(acc[2 * j + 1], pair_of(r[j].z, r[j].w), f);
  }
}

// Writes 64 bytes of each of 32 rows (w: this lane's row) to row-major global memory through the warp's
// staging buffer, so that four neighbouring lanes write one row's 64 bytes.  Chunks of 16 bytes are
// swizzled by the row: both directions are free of bank conflicts.  ES: bytes per element.
template <int ES>
__device__ __forceinline__ void store_rows64(uint8_t* stg, int lane, const uint32_t (&w)[16], char* d, long long pitch,
                                             int rows, int col, int ncols, int vec) {
  uint8_t* mine = stg + lane * 64;
  const int sw = (lane >> 1) & 3;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(mine + ((j ^ sw) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2), ch = lane & 3;
    const uint4 u = *reinterpret_cast<const uint4*>(stg + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4));
    const int c = col + ch * (16 / ES);
    if (r < rows && c < ncols) {
      char* q = d + r * pitch + static_cast<long long>(c) * ES;
      if (vec && c + 16 / ES <= ncols) {
        *reinterpret_cast<uint4*>(q) = u;
      } else {
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 16 / ES; ++e) {
          if (c + e >= ncols) break;
          if (ES == 4) reinterpret_cast<uint32_t*>(q)[e] = x[e];
          else reinterpret_cast<uint16_t*>(q)[e] = static_cast<uint16_t>(x[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  }
  __syncwarp();
}

template <int KIND, int BN, int CTAS>
__global__ void __launch_bounds__(384, 1) grouped_gemm_kernel(const __grid_constant__ Params p) {
  using C = Cfg<KIND, BN, CTAS>;
  constexpr int STAGES = C::STAGES, NBUF = C::NBUF, NC = C::NC;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* staging = smem + STAGES * C::STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + 8 * C::STG_BYTES);
  uint64_t* full_bar = bars;                     // [STAGES] operands landed (the leader CTA's is used)
  uint64_t* empty_bar = bars + STAGES;           // [STAGES] MMAs have read the stage
  uint64_t* tfull_bar = bars + 2 * STAGES;       // [NBUF]   accumulator complete
  uint64_t* tempty_bar = tfull_bar + NBUF;       // [NBUF]   accumulator read out (the leader CTA's is used)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + NBUF);
  int* first = reinterpret_cast<int*>(staging + 8 * C::STG_BYTES + C::BAR_BYTES);   // [G + 1] first tile of a group
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
      ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 1);
    }
    for (int b = 0; b < NBUF; ++b) {
      ptx::mbar_init(ptx::smem_u32(&tfull_bar[b]), 1);
      ptx::mbar_init(ptx::smem_u32(&tempty_bar[b]), 8 * CTAS);
    }
    ptx::fence_mbar_init();
  }
  if (warp == 2) {
    ptx::tmem_alloc<CTAS>(ptx::smem_u32(tmem_slot), 512);
    ptx::tmem_relinquish<CTAS>();
  }
  // Everything above touched neither global memory nor what the previous kernel of the stream writes.
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();

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
    if (lane == 0) first[0] = 0;
  }
  ptx::tc_fence_before();
  __syncthreads();
  if constexpr (CTAS > 1) {
    ptx::cluster_arrive_relaxed();
    ptx::cluster_wait();
  }
  ptx::tc_fence_after();
  const uint32_t tmem = ptx::uniform(*reinterpret_cast<volatile uint32_t*>(tmem_slot));
  Schedule sched = {unit, units, ptx::uniform(first[p.G]), p.num_kb};
  Item it;
  ptx::Waiter w = {p.status, p.wait_budget};

  // 128 sums and two slices of 16 columns per thread do not fit the 168 registers that 384 threads can have
  // each: the first four warps hand theirs over (72 + 2 x 216 = 3 x 168).
  if constexpr (C::SPLIT_REGS) {
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  }
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      while (sched.next(it)) {
        const Tile x = decode<C>(p, first, grow, it.tile);
        // rows of A that this CTA needs, and the bytes that both CTAs of a pair load
        uint32_t bytes = 0;
        int boxes = 0;                           // of 32 rows; 4: one box of 128
#pragma unroll
        for (int c = 0; c < CTAS; ++c) {
          const int need = min(max((x.rows - c * 128 + 31) / 32, 0), 4);
          bytes += need * 4096 + C::B_BYTES;
          if (c == static_cast<int>(rank)) boxes = need;
        }
        const int row = x.row0 + static_cast<int>(rank) * 128;
        const int col = x.n0 + static_cast<int>(rank) * C::BN_CTA;
        const int bg = p.b_grouped ? x.g : 0;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          w.wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1u, DEV_TIMEOUT_PRODUCER_EMPTY);
          const uint32_t own = ptx::smem_u32(&full_bar[stage]);
          const uint32_t bar = CTAS == 2 ? ptx::mapa(own, 0) : own;
          if (rank == 0) ptx::mbar_arrive_expect_tx(own, bytes);
          const uint32_t sa = ptx::smem_u32(smem + stage * C::STAGE_BYTES), sb = sa + C::A_BYTES;
          const int k = kb * C::KBLK;
          if (boxes == 4) {
            ptx::tma_load_3d<CTAS>(sa, &p.tm_a, bar, k, row, 0);
          } else {
            for (int b = 0; b < boxes; ++b) ptx::tma_load_3d<CTAS>(sa + b * 4096, &p.tm_a32, bar, k, row + b * 32, 0);
          }
          if (p.b_nk) {
            ptx::tma_load_3d<CTAS>(sb, &p.tm_b, bar, k, col, bg);
          } else {
#pragma unroll
            for (int c = 0; c < C::BN_CTA / C::GRP_COLS; ++c)
              ptx::tma_load_3d<CTAS>(sb + c * C::GRP_BYTES, &p.tm_b, bar, col + c * C::GRP_COLS, k, bg);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      // The CTA may not go before its last copies have landed, also where another role gave up and
      // nobody waited for them (the leader's barriers count both CTAs' bytes; the pair leaves together).
      if (rank == 0) {
        for (int s = 0; s < STAGES; ++s)
          w.wait(ptx::smem_u32(&full_bar[s]), s < stage ? phase : phase ^ 1u, DEV_TIMEOUT_MMA_FULL);
      }
    }
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
      int stage = 0, buf = 0;
      uint32_t phase = 0, tphase = 0;
      while (sched.next(it)) {
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          const bool fresh = KIND == KIND_E4M3 || kb == it.kb0;          // starts an accumulator
          const bool done = KIND == KIND_E4M3 || kb + 1 == it.kb1;       // and completes it
          w.wait(full0 + stage * 8, phase, DEV_TIMEOUT_MMA_FULL);
          const uint32_t sa = smem0 + stage * C::STAGE_BYTES;
          const uint64_t adesc = ptx::make_smem_desc_sw128(sa, 16, 1024);
          const uint64_t bdesc = ptx::make_smem_desc_sw128(sa + C::A_BYTES, b_lbo, 1024);
          const uint32_t d = tmem + static_cast<uint32_t>(buf * BN);
          // last of all, the wait that the promotion warps answer: what follows it is on their round trip
          if (fresh) w.wait(tempty0 + buf * 8, tphase ^ 1u, DEV_TIMEOUT_MMA_TMEM_EMPTY);
          __syncwarp();
          ptx::tc_fence_after();
          if (ptx::elect_one()) {
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
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          if (done && ++buf == NBUF) { buf = 0; tphase ^= 1u; }
        }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ promotion and epilogue
    if constexpr (C::SPLIT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int q = warp & 3, half = (warp - 4) >> 2;
    uint8_t* stg = staging + (warp - 4) * C::STG_BYTES;
    const uint32_t lead = CTAS == 2 ? ptx::mapa(ptx::smem_u32(&tempty_bar[0]), 0) : ptx::smem_u32(&tempty_bar[0]);
    const uint32_t t_base = tmem + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(half * NC);
    const int ncols = p.pair == PAIR_NONE ? p.N : p.N >> 1;
    const uint32_t tfull0 = ptx::smem_u32(tfull_bar);
    int buf = 0;
    uint32_t tphase = 0;
    while (sched.next(it)) {
      const Tile x = decode<C>(p, first, grow, it.tile);
      const int roff = static_cast<int>(rank) * 128 + q * 32;      // of this warp inside the tile
      const int rows = x.rows - roff;                              // of the group, from this warp's first on
      const int col = x.n0 + half * NC;
      const bool live = rows > 0 && col < p.N;                     // the warp has outputs here
      uint64_t sum[NC / 2];                    // columns 2 i and 2 i + 1
#pragma unroll
      for (int i = 0; i < NC / 2; ++i) sum[i] = 0;
      // The tile's accumulators one after another, in slices of 16 columns: while a slice is scaled and added,
      // the next one is on its way out of TMEM.  A buffer is free once its last slice has been read.
      const int last = KIND == KIND_E4M3 ? it.kb1 - 1 : it.kb0;
      uint4 r[2][4];
      auto open = [&](int b, uint32_t ph) {
        w.wait(tfull0 + b * 8, ph, DEV_TIMEOUT_EPI_TMEM_FULL);
        __syncwarp();
        ptx::tc_fence_after();
      };
      auto take = [&](float factor) {
        open(buf, tphase);
        const uint64_t f = pair_of(__float_as_uint(factor), __float_as_uint(factor));
        const uint32_t t0 = t_base + static_cast<uint32_t>(buf * BN);
        ptx::tmem_ld_32x16_async(t0, r[0]);
#pragma unroll
        for (int c = 0; c < NC / 16; ++c) {
          ptx::tmem_ld_wait_for(r[c & 1]);
          if (c + 1 < NC / 16) {
            ptx::tmem_ld_32x16_async(t0 + static_cast<uint32_t>((c + 1) * 16), r[(c + 1) & 1]);
          } else {
            ptx::tc_fence_before();
            if (lane == 0) ptx::mbar_arrive_cluster_relaxed(lead + static_cast<uint32_t>(buf * 8));
          }
          scale_add(&sum[c * 8], r[c & 1], f);
        }
        if (++buf == NBUF) { buf = 0; tphase ^= 1u; }
      };
      if (!live) {                                // nothing to add, but every accumulator is released by all
        for (int kb = it.kb0; kb <= last; ++kb) {
          open(buf, tphase);
          ptx::tc_fence_before();
          if (lane == 0) ptx::mbar_arrive_cluster_relaxed(lead + static_cast<uint32_t>(buf * 8));
          if (++buf == NBUF) { buf = 0; tphase ^= 1u; }
        }
        continue;
      }
      if constexpr (KIND == KIND_BF16) {
        take(1.0f);
      } else {
        // Block scales are asked for two blocks ahead of their use.
        const float* sa = p.sa + (static_cast<long long>(x.row0) + roff + min(lane, rows - 1)) * p.sa_row + it.kb0 * p.sa_blk;
        const float* sb = p.sb + static_cast<long long>(x.g) * p.sb_group + static_cast<long long>(col >> 7) * p.sb_n +
                          it.kb0 * p.sb_k;
        float a0 = ptx::ld_early(sa), b0 = ptx::ld_early(sb), a1 = 0.0f, b1 = 0.0f;
        if (it.kb0 < last) {
          a1 = ptx::ld_early(sa + p.sa_blk);
          b1 = ptx::ld_early(sb + p.sb_k);
        }
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
      float acc[NC];
#pragma unroll
      for (int i = 0; i < NC / 2; ++i) {
        acc[2 * i] = lo_of(sum[i]);
        acc[2 * i + 1] = hi_of(sum[i]);
      }
      if (p.pair != PAIR_NONE) {
#pragma unroll
        for (int i = 0; i < NC / 2; ++i)
          acc[i] = (p.pair == PAIR_SWIGLU ? silu_f(acc[2 * i]) : gelu_f(acc[2 * i])) * acc[2 * i + 1];
      }
      const int nc = p.pair == PAIR_NONE ? NC : NC / 2;
      const int ocol = p.pair == PAIR_NONE ? col : col >> 1;
      const long long drow = static_cast<long long>(x.row0) + roff;
      const long long pitch = p.ldd * (p.d_f32 ? 4 : 2);
      char* d = static_cast<char*>(p.D) + drow * pitch;
      if (p.d_f32) {
#pragma unroll
        for (int c = 0; c < NC; c += 16) {
          if (c >= nc) break;
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(acc[c + i]);
          store_rows64<4>(stg, lane, w, d, pitch, rows, ocol + c, ncols, p.vec_d);
        }
      } else {
#pragma unroll
        for (int c = 0; c < NC; c += 32) {
          if (c >= nc) break;
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = pack_bf16(acc[c + 2 * i], acc[c + 2 * i + 1]);
          store_rows64<2>(stg, lane, w, d, pitch, rows, ocol + c, ncols, p.vec_d);
        }
      }
    }
  }

  // ------------------------------------------------------------------ teardown
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  // No CTA leaves while its peer may still write its barriers or read the pair's TMEM.
  if constexpr (CTAS > 1) {
    ptx::cluster_arrive_relaxed();
    ptx::cluster_wait();
  }
  if (warp == 2) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<CTAS>(tmem, 512);
  }
}

// ---------------------------------------------------------------------------- host
typedef void (*KernelFn)(const Params);
struct Variant {
  int kind, bn, ctas, smem;
  KernelFn fn;
  const char* name;
};
#define XF_GG(KIND, BN, CTAS, NAME) {KIND, BN, CTAS, Cfg<KIND, BN, CTAS>::SMEM_BYTES, grouped_gemm_kernel<KIND, BN, CTAS>, NAME}
static const Variant g_variants[] = {
    XF_GG(KIND_E4M3, 256, 2, "e4m3_256x256_cta2"),
    XF_GG(KIND_BF16, 256, 2, "bf16_256x256_cta2"),
    XF_GG(KIND_E4M3, 128, 1, "e4m3_128x128_cta1"),
    XF_GG(KIND_BF16, 128, 1, "bf16_128x128_cta1"),
};
#undef XF_GG

static bool aligned(const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) % to) == 0; }

static xf_status validate(const xf_grouped_gemm_desc* d) {
  if (!d) {
    set_error("null descriptor");
    return XF_ERR_INVALID_PROBLEM;
  }
  if (d->dtype_ab != XF_DT_BF16 && d->dtype_ab != XF_DT_E4M3) {
    set_error("A/B dtype must be bf16 or e4m3 (got %d)", d->dtype_ab);
    return XF_ERR_INVALID_DATA_TYPE;
  }
  if (d->dtype_d != XF_DT_BF16 && d->dtype_d != XF_DT_F32) {
    set_error("D dtype must be bf16 or f32 (got %d)", d->dtype_d);
    return XF_ERR_INVALID_DATA_TYPE;
  }
  if (d->M < 0 || d->N <= 0 || d->K <= 0 || d->num_groups <= 0) {
    set_error("problem extents must be positive (M=%d N=%d K=%d groups=%d)", d->M, d->N, d->K, d->num_groups);
    return XF_ERR_INVALID_PROBLEM;
  }
  if (d->num_groups > kMaxGroups) {
    set_error("at most %d groups (got %d)", kMaxGroups, d->num_groups);
    return XF_ERR_NOT_SUPPORTED;
  }
  if (d->num_groups > 1 && !d->group_offsets) {
    set_error("%d groups need group_offsets", d->num_groups);
    return XF_ERR_INVALID_PROBLEM;
  }
  if (d->flags & ~(XF_FLAG_FORCE_1CTA | XF_FLAG_FORCE_2CTA | XF_FLAG_NO_SPLIT | XF_FLAG_NO_PDL | XF_FLAG_SHORT_WAITS)) {
    set_error("unsupported flags 0x%x", d->flags);
    return XF_ERR_NOT_SUPPORTED;
  }
  if (d->b_layout != XF_B_KN && d->b_layout != XF_B_NK) {
    set_error("unknown layout of B (%d)", d->b_layout);
    return XF_ERR_INVALID_LAYOUT;
  }
  if (d->pair != XF_PAIR_NONE && d->pair != XF_PAIR_SWIGLU && d->pair != XF_PAIR_GEGLU) {
    set_error("pair op %d: only SwiGLU and GeGLU, in the compact layout", d->pair);
    return XF_ERR_NOT_SUPPORTED;
  }
  if (d->pair != XF_PAIR_NONE && (d->N & 1)) {
    set_error("pair ops need an even N (N=%d)", d->N);
    return XF_ERR_INVALID_PROBLEM;
  }
  if ((static_cast<long long>(d->M) / 128 + d->num_groups) * ((d->N + 127) / 128) > 0x7FFFFFFFLL) {
    set_error("more than 2^31 tiles (M=%d N=%d groups=%d)", d->M, d->N, d->num_groups);
    return XF_ERR_NOT_SUPPORTED;
  }
  const int es = d->dtype_ab == XF_DT_BF16 ? 2 : 1, ds = d->dtype_d == XF_DT_BF16 ? 2 : 4;
  const int bcols = d->b_layout == XF_B_KN ? d->N : d->K, brows = d->b_layout == XF_B_KN ? d->K : d->N;
  const int ncols = d->pair == XF_PAIR_NONE ? d->N : d->N / 2;
  if (d->lda < d->K || d->ldb < bcols || d->ldd < ncols ||
      (d->num_groups > 1 && d->batch_b != 0 && d->batch_b < d->ldb * (brows - 1) + bcols)) {
    set_error("pitches too small (lda=%lld ldb=%lld batch_b=%lld ldd=%lld for M=%d N=%d K=%d)", (long long)d->lda,
              (long long)d->ldb, (long long)d->batch_b, (long long)d->ldd, d->M, d->N, d->K);
    return XF_ERR_INVALID_LAYOUT;
  }
  if (d->M > 0 && (!d->A || !d->D)) {
    set_error("A and D must be non-null");
    return XF_ERR_INVALID_PROBLEM;
  }
  if (!d->B) {
    set_error("B must be non-null");
    return XF_ERR_INVALID_PROBLEM;
  }
  if (!aligned(d->A, 16) || !aligned(d->B, 16) || (d->lda * es) % 16 != 0 || (d->ldb * es) % 16 != 0 ||
      (d->batch_b * es) % 16 != 0) {
    set_error("A/B base pointers, row pitches and group strides must be multiples of 16 bytes (lda=%lld ldb=%lld "
              "batch_b=%lld, %d-byte elements)", (long long)d->lda, (long long)d->ldb, (long long)d->batch_b, es);
    return XF_ERR_MISALIGNED_OPERAND;
  }
  if (!aligned(d->D, ds) || !aligned(d->group_offsets, 4) || !aligned(d->scale_a, 4) || !aligned(d->scale_b, 4)) {
    set_error("pointers must be aligned to their element size");
    return XF_ERR_MISALIGNED_OPERAND;
  }
  if (d->dtype_ab == XF_DT_E4M3) {
    if ((d->M > 0 && !d->scale_a) || !d->scale_b) {
      set_error("e4m3 operands need scale_a and scale_b");
      return XF_ERR_INVALID_PROBLEM;
    }
    if (d->scale_a_row_stride < 0 || d->scale_a_blk_stride < 0 || d->scale_b_k_stride < 0 || d->scale_b_n_stride < 0 ||
        d->scale_b_group_stride < 0) {
      set_error("scale strides must not be negative");
      return XF_ERR_INVALID_LAYOUT;
    }
  } else if (d->scale_a || d->scale_b) {
    set_error("bf16 operands take no scales");
    return XF_ERR_INVALID_PROBLEM;
  }
  return XF_SUCCESS;
}

// What a problem looks like on the current device.
struct Geometry {
  const Variant* v;
  int dev, units;
  size_t workspace_bytes;
};

static xf_status plan_geometry(const xf_grouped_gemm_desc* d, Geometry* g) {
  int dev = 0, major = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    set_error("no CUDA device: %s", cudaGetErrorString(cudaGetLastError()));
    return XF_ERR_ARCH_MISMATCH;
  }
  cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (major != 10) {
    set_error("this library holds sm_100a code only; device %d has compute capability %d.x", dev, major);
    return XF_ERR_ARCH_MISMATCH;
  }
  const int kind = d->dtype_ab == XF_DT_BF16 ? KIND_BF16 : KIND_E4M3;
  const Variant* v = nullptr;
  // Pairs of CTAs on 256 x 256 tiles need half the operand bytes per multiplication of single CTAs on
  // 128 x 128 tiles, which waste less on groups of few rows.
  int ctas = d->M / d->num_groups > 128 ? 2 : 1;
  if (d->flags & XF_FLAG_FORCE_1CTA) ctas = 1;
  else if (d->flags & XF_FLAG_FORCE_2CTA) ctas = 2;
  for (const Variant& c : g_variants)
    if (c.kind == kind && c.ctas == ctas) v = &c;
  const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(v->fn),
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, v->smem);
  if (e != cudaSuccess) {
    set_error("cudaFuncSetAttribute(smem=%d) failed: %s", v->smem, cudaGetErrorString(e));
    return XF_ERR_INTERNAL;
  }
  g->v = v;
  g->dev = dev;
  g->units = sms;
  if (v->ctas > 1) {   // pairs that can run at once: GPC boundaries may leave SMs without a partner
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms - sms % v->ctas, 1, 1);
    cfg.blockDim = dim3(384, 1, 1);
    cfg.dynamicSmemBytes = v->smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = v->ctas; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&g->units, reinterpret_cast<const void*>(v->fn), &cfg) != cudaSuccess || g->units < 1) {
      cudaGetLastError();
      g->units = sms / v->ctas;
    }
  }
  g->workspace_bytes = 256;
  return XF_SUCCESS;
}

}  // namespace grouped
}  // namespace xf

struct xf_grouped_plan {
  xf::grouped::Params params;
  const xf::grouped::Variant* variant;
  int grid, device, no_pdl;
  size_t clear_bytes;
  char name[64];
};

extern "C" {

xf_status xf_grouped_gemm_can_implement(const xf_grouped_gemm_desc* desc) { return xf::grouped::validate(desc); }

xf_status xf_grouped_gemm_workspace_size(const xf_grouped_gemm_desc* desc, size_t* bytes) {
  if (!bytes) {
    xf::set_error("null output pointer");
    return XF_ERR_INVALID_PROBLEM;
  }
  *bytes = 256;
  if (!desc || xf::grouped::validate(desc) != XF_SUCCESS) return XF_SUCCESS;   // can_implement reports why
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev == 0) {
    cudaGetLastError();
    return XF_SUCCESS;   // no GPU here: a plan cannot be created either
  }
  xf::grouped::Geometry g;
  const xf_status s = xf::grouped::plan_geometry(desc, &g);
  if (s == XF_SUCCESS) *bytes = g.workspace_bytes;
  return s;
}

xf_status xf_grouped_gemm_plan_create(const xf_grouped_gemm_desc* d, void* workspace, void* stream,
                                      xf_grouped_plan** out) {
  using namespace xf;
  using namespace xf::grouped;
  if (!out) {
    set_error("null plan output pointer");
    return XF_ERR_INVALID_PROBLEM;
  }
  *out = nullptr;
  xf_status s = grouped::validate(d);
  if (s != XF_SUCCESS) return s;
  if (!grouped::aligned(workspace, 16)) {
    set_error("the workspace must be 16-byte aligned");
    return XF_ERR_MISALIGNED_OPERAND;
  }
  Geometry g;
  s = grouped::plan_geometry(d, &g);
  if (s != XF_SUCCESS) return s;
  const Variant* v = g.v;
  xf_grouped_plan* plan = nullptr;
  if (posix_memalign(reinterpret_cast<void**>(&plan), 64, sizeof(xf_grouped_plan)) != 0) {
    set_error("out of host memory");
    return XF_ERR_MEMORY_ALLOCATION;
  }
  memset(plan, 0, sizeof(*plan));
  Params& p = plan->params;
  const int es = v->kind == KIND_BF16 ? 2 : 1, kblk = 128 / es;
  p.M = d->M; p.N = d->N; p.K = d->K; p.G = d->num_groups;
  p.tiles_n = (d->N + v->bn - 1) / v->bn;
  p.num_kb = (d->K + kblk - 1) / kblk;
  // row tiles run fastest inside sweeps of at most group_m of them, as many as fill 40 % of L2 with A
  int l2 = 0;
  cudaDeviceGetAttribute(&l2, cudaDevAttrL2CacheSize, g.dev);
  const double panel = 128.0 * v->ctas * d->K * es;
  p.group_m = static_cast<int>(0.40 * l2 / panel);
  if (p.group_m < 8) p.group_m = 8;
  if (p.group_m > (1 << 30) / p.tiles_n) p.group_m = (1 << 30) / p.tiles_n;
  p.b_nk = d->b_layout == XF_B_NK;
  p.b_grouped = d->batch_b != 0;
  p.offsets = d->group_offsets;
  p.sa = d->scale_a; p.sa_row = d->scale_a_row_stride; p.sa_blk = d->scale_a_blk_stride;
  p.sb = d->scale_b; p.sb_k = d->scale_b_k_stride; p.sb_n = d->scale_b_n_stride; p.sb_group = d->scale_b_group_stride;
  p.D = d->D; p.ldd = d->ldd;
  p.d_f32 = d->dtype_d == XF_DT_F32;
  p.pair = d->pair;
  p.vec_d = grouped::aligned(d->D, 16) && (d->ldd * (p.d_f32 ? 4 : 2)) % 16 == 0;
  p.wait_budget = (d->flags & XF_FLAG_SHORT_WAITS) ? 2000000LL : 4000000000LL;
  plan->variant = v;
  plan->device = g.dev;
  plan->no_pdl = (d->flags & XF_FLAG_NO_PDL) ? 1 : 0;
  if (d->M > 0) {
    const CUtensorMapDataType dt = v->kind == KIND_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const uint64_t pa = static_cast<uint64_t>(d->lda) * es, pb = static_cast<uint64_t>(d->ldb) * es;
    const int b0 = p.b_nk ? d->K : d->N, b1 = p.b_nk ? d->N : d->K;
    const uint64_t sb = d->batch_b ? static_cast<uint64_t>(d->batch_b) * es : pb * b1;
    const uint64_t ng = d->batch_b ? d->num_groups : 1;
    if (!encode_3d(&p.tm_a, dt, d->A, d->K, d->M, 1, pa, pa * d->M, kblk, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_3d(&p.tm_a32, dt, d->A, d->K, d->M, 1, pa, pa * d->M, kblk, 32, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_3d(&p.tm_b, dt, d->B, b0, b1, ng, pb, sb, 128 / es, p.b_nk ? 128 : kblk, CU_TENSOR_MAP_SWIZZLE_128B)) {
      free(plan);
      return XF_ERR_INTERNAL;
    }
    long long tiles = (static_cast<long long>(d->M) + 128 * v->ctas - 1) / (128 * v->ctas) + d->num_groups - 1;
    tiles *= p.tiles_n;
    plan->grid = static_cast<int>(tiles < g.units ? tiles : g.units) * v->ctas;
  }
  snprintf(plan->name, sizeof(plan->name), "%s", v->name);
  if (workspace && d->workspace_bytes >= 256) {
    p.status = static_cast<int*>(workspace);
    plan->clear_bytes = 256;
    const cudaError_t e = cudaMemsetAsync(workspace, 0, plan->clear_bytes, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) {
      free(plan);
      set_error("clearing the workspace failed: %s", cudaGetErrorString(e));
      return XF_ERR_INTERNAL;
    }
  }
  *out = plan;
  return XF_SUCCESS;
}

xf_status xf_grouped_gemm_run(xf_grouped_plan* plan, void* stream) {
  if (!plan) {
    xf::set_error("null plan");
    return XF_ERR_INVALID_PROBLEM;
  }
  int cur = -1;
  if (cudaGetDevice(&cur) != cudaSuccess || cur != plan->device) {
    xf::set_error("plan %s was created on device %d but device %d is current", plan->name, plan->device, cur);
    return XF_ERR_INVALID_PROBLEM;
  }
  if (plan->grid == 0) return XF_SUCCESS;   // no rows
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan->grid, 1, 1);
  cfg.blockDim = dim3(384, 1, 1);
  cfg.dynamicSmemBytes = plan->variant->smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = plan->variant->ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = plan->no_pdl ? 1 : 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, plan->variant->fn, plan->params);
  if (e != cudaSuccess) {
    xf::set_error("launch of %s failed: %s", plan->name, cudaGetErrorString(e));
    return XF_ERR_INTERNAL;
  }
  return XF_SUCCESS;
}

xf_status xf_grouped_gemm_plan_device_status(xf_grouped_plan* plan, int32_t* device_code) {
  if (!plan || !device_code) {
    xf::set_error("null argument");
    return XF_ERR_INVALID_PROBLEM;
  }
  *device_code = 0;
  if (!plan->params.status) return XF_SUCCESS;
  cudaError_t e = cudaMemcpy(device_code, plan->params.status, sizeof(int32_t), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) {
    xf::set_error("reading the status word failed: %s", cudaGetErrorString(e));
    return XF_ERR_INTERNAL;
  }
  if (*device_code != 0) {
    // reported once: the words a launch that gave up may have left part-way start over
    e = cudaMemset(plan->params.status, 0, plan->clear_bytes);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    xf::set_error("kernel %s gave up in a bounded wait (device code %d)", plan->name, *device_code);
    return XF_ERR_INTERNAL;
  }
  return XF_SUCCESS;
}

const char* xf_grouped_gemm_plan_kernel_name(const xf_grouped_plan* plan) { return plan ? plan->name : ""; }

xf_status xf_grouped_plan_destroy(xf_grouped_plan* plan) {
  free(plan);
  return XF_SUCCESS;
}

}  // extern "C"
