// Host side of the grouped products: argument checks, choice of the tile, tensor maps, launch.  Exposes the
// xf_grouped_gemm_* entry points declared in include/xefuse_b200.h.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "../../include/xefuse_b200.h"
#include "xf_grouped_gemm_kernel.cuh"
#include "xf_host_util.h"

namespace xf {
namespace grouped {

static bool aligned(const void* p, int to) { return (reinterpret_cast<uintptr_t>(p) % to) == 0; }

static const Variant* tiles_of(int dtype_ab, int* count) {
  *count = dtype_ab == XF_DT_BF16 ? kTilesBf16 : kTilesE4m3;
  return dtype_ab == XF_DT_BF16 ? g_variants_bf16 : g_variants_e4m3;
}
static bool allowed(const Variant& v, int flags) {
  return !((flags & XF_FLAG_FORCE_1CTA && v.ctas != 1) || (flags & XF_FLAG_FORCE_2CTA && v.ctas != 2) ||
           (flags & XF_FLAG_FORCE_BN128 && v.bn != 128) || (flags & XF_FLAG_FORCE_BN256 && v.bn != 256));
}

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
  if (d->M > kMaxExtent || d->N > kMaxExtent || d->K > kMaxExtent) {
    set_error("extents of at most %d (M=%d N=%d K=%d)", kMaxExtent, d->M, d->N, d->K);
    return XF_ERR_NOT_SUPPORTED;
  }
  if (d->num_groups > kMaxGroups) {
    set_error("at most %d groups (got %d)", kMaxGroups, d->num_groups);
    return XF_ERR_NOT_SUPPORTED;
  }
  if (d->num_groups > 1 && !d->group_offsets) {
    set_error("%d groups need group_offsets", d->num_groups);
    return XF_ERR_INVALID_PROBLEM;
  }
  if (d->flags & ~(XF_FLAG_FORCE_1CTA | XF_FLAG_FORCE_2CTA | XF_FLAG_FORCE_BN128 | XF_FLAG_FORCE_BN256 | XF_FLAG_NO_SPLIT | XF_FLAG_NO_PDL | XF_FLAG_SHORT_WAITS)) {
    set_error("unsupported flags 0x%x", d->flags);
    return XF_ERR_NOT_SUPPORTED;
  }
  int count = 0, left = 0;
  const Variant* all = tiles_of(d->dtype_ab, &count);
  for (int i = 0; i < count; ++i) left += allowed(all[i], d->flags);
  if (left == 0) {
    set_error("no tile of this type matches the flags 0x%x", d->flags);
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
  KernelFn fn;
  int dev, units;
  int split_kb, split_max;   // Params; split_kb 0: whole tiles only
  size_t partials_off, workspace_bytes;   // [0, 256) status, flags, partial sums
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
  // The tile: the lowest estimate of clocks for whole waves plus the last one, whose tiles may be shared.
  // Measured on long problems, in clocks for a K block, the end of a tile, publishing a share of one and
  // summing another unit's share:
  //   e4m3  256 x 256, CTA pair  720  3700  5000  1800     bf16  256 x 256, CTA pair  680  3700  5000  1800
  //         128 x 256, one CTA   870  3700  5000  1800           128 x 128, one CTA   490  2000  3000   900
  //         128 x 128, one CTA   600  2000  3000   900
  // Large tiles read fewer operand bytes per multiplication; tiles of 128 rows waste less on groups of few
  // rows, and small ones spread better.  Rows of a group are taken to fill half of its last tile.  e4m3, pair /
  // 128 x 256 / 128 x 128, in bursts of 30 launches: 4096 x 28672 x 4096 407 / 429 / 539 us, 777 x 5001 x 2000
  // 35 / 21 / 25 us, 64 experts 16384 x 4096 x 2048 268 / 216 / 242 us, 100 x 8192 x 8192 - / 23 / 16.5 us.  (Back to
  // back, under the power cap, the first takes 464 us and the third 243 us with the tiles chosen here.)
  const Variant* v = nullptr;
  int count = 0;
  const Variant* all = tiles_of(d->dtype_ab, &count);
  const int kblk = kind == KIND_BF16 ? 64 : 128;
  const double num_kb = (d->K + kblk - 1) / kblk;
  double best = 0.0;
  for (int i = 0; i < count; ++i) {
    const Variant& c = all[i];
    if (!allowed(c, d->flags)) continue;
    const bool wide = c.bn == 256;
    const double per_kb = kind == KIND_BF16 ? (wide ? 680 : 490) : (c.ctas == 2 ? 720 : wide ? 870 : 600);
    const double tile = num_kb * per_kb + (wide ? 3700 : 2000), publish = wide ? 5000 : 3000, sum = wide ? 1800 : 900;
    const int rows = 128 * c.ctas, units = sms / c.ctas;
    // sharing a tile's K range s ways takes tile / s + publish + (s - 1) * sum: least at s = sqrt(tile / sum)
    const int most = static_cast<int>(sqrt(num_kb * per_kb / sum) + 0.5);
    const int split_max = most < 2 ? 2 : most > 8 ? 8 : most;
    const double tiles_m = d->num_groups == 1 ? (d->M + rows - 1) / rows : static_cast<double>(d->M) / rows + 0.5 * d->num_groups;
    const double waves = tiles_m * ((d->N + c.bn - 1) / c.bn) / units, full = floor(waves), rest = waves - full;
    const double share = rest * split_max < 1.0 ? 1.0 / split_max : rest;
    const double last = rest == 0.0 ? 0.0 : share * tile + publish + (1.0 / share < 2.0 ? 1.0 : 1.0 / share - 1.0) * sum;
    const double cost = full * tile + (last < tile || rest == 0.0 ? last : tile);
    if (!v || cost < best) {
      v = &c;
      best = cost;
      g->split_kb = static_cast<int>((publish + sum) / per_kb + 0.5);
      g->split_max = split_max;
    }
  }
  const bool f32 = d->dtype_d == XF_DT_F32;
  g->fn = v->fn[d->pair == XF_PAIR_NONE ? (f32 ? OUT_F32 : OUT_BF16) : (f32 ? OUT_PAIR_F32 : OUT_PAIR_BF16)];
  const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(g->fn),
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
    if (cudaOccupancyMaxActiveClusters(&g->units, reinterpret_cast<const void*>(g->fn), &cfg) != cudaSuccess || g->units < 1) {
      cudaGetLastError();
      g->units = sms / v->ctas;
    }
  }
  if (d->flags & XF_FLAG_NO_SPLIT) g->split_kb = 0;
  if ((d->K + 63) / 64 > (1 << 20)) g->split_kb = 0;   // block numbers of a whole wave stay within 32 bits
  const size_t grid = static_cast<size_t>(g->units) * v->ctas;
  g->partials_off = 256 + (grid * 8 * sizeof(int) + 255) / 256 * 256;
  g->workspace_bytes = g->split_kb ? g->partials_off + grid * 128 * v->bn * sizeof(float) : 256;
  return XF_SUCCESS;
}

}  // namespace grouped
}  // namespace xf

struct xf_grouped_plan {
  xf::grouped::Params params;
  const xf::grouped::Variant* variant;
  xf::grouped::KernelFn fn;
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
  const int es = v->kind == KIND_BF16 ? 2 : 1, ds = d->dtype_d == XF_DT_F32 ? 4 : 2, kblk = 128 / es;
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
  p.pair = d->pair;
  p.vec_d = grouped::aligned(d->D, 16) && (d->ldd * ds) % 16 == 0;
  p.wait_budget = (d->flags & XF_FLAG_SHORT_WAITS) ? 2000000LL : 4000000000LL;
  plan->variant = v;
  plan->fn = g.fn;
  plan->device = g.dev;
  plan->no_pdl = (d->flags & XF_FLAG_NO_PDL) ? 1 : 0;
  if (d->M > 0) {
    const CUtensorMapDataType dt = v->kind == KIND_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const uint64_t pa = static_cast<uint64_t>(d->lda) * es, pb = static_cast<uint64_t>(d->ldb) * es;
    const int b0 = p.b_nk ? d->K : d->N, b1 = p.b_nk ? d->N : d->K;
    const uint64_t sb = d->batch_b ? static_cast<uint64_t>(d->batch_b) * es : pb * b1;
    const uint64_t pd = static_cast<uint64_t>(d->ldd) * ds;
    const uint64_t ng = d->batch_b ? d->num_groups : 1;
    if (!encode_3d(&p.tm_a, dt, d->A, d->K, d->M, 1, pa, pa * d->M, kblk, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_3d(&p.tm_a32, dt, d->A, d->K, d->M, 1, pa, pa * d->M, kblk, 32, CU_TENSOR_MAP_SWIZZLE_128B) ||
        (p.vec_d && !encode_3d(&p.tm_d, ds == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, d->D,
                               p.pair == XF_PAIR_NONE ? d->N : d->N / 2, d->M, 1, pd, pd * d->M, 64 / ds, 32,
                               CU_TENSOR_MAP_SWIZZLE_64B)) ||
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
    if (g.split_kb && d->workspace_bytes >= g.workspace_bytes) {
      p.split_kb = g.split_kb;
      p.split_max = g.split_max;
      p.flags = reinterpret_cast<int*>(static_cast<char*>(workspace) + 256);
      p.partials = reinterpret_cast<float4*>(static_cast<char*>(workspace) + g.partials_off);
      plan->clear_bytes = g.partials_off;
      plan->grid = plan->grid ? g.units * v->ctas : 0;
    }
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, plan->fn, plan->params);
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
