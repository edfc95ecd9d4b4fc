// Row passes with an 8-bit output: RMSNorm (optionally after a residual addition) and SwiGLU / GeGLU,
// written as int8 with one scale per row or as e4m3 with one scale per row and block of 128 columns.
//
// Mathematics.  With h the (summed) input row, w the norm weight and rstd = 1/sqrt(mean h^2 + eps), the
// normalised value is t * rstd, t = h * w.  A row's common factor cancels between a value and the
// largest value of its block, so the codes need the row's sum of squares not at all:
//     a     = max(max |t|, 2^-100)  over the block (e4m3) or the row (int8)
//     code  = round(t * L / a)      L = 448 (e4m3, ties to even), 127 (int8, ties away from zero)
//     scale = a * rstd / L
// t is exact: a product of two bf16 values has 16 significant bits, and so the norm's codes are those of the exact
// quotient t * L / a (int8 and e4m3 alike).  The gate's y is rounded itself, and its codes are those of y * (448 / a).
// The floor of 2^-100 gives a block of zeros zero codes and keeps L / a finite.  Maxima are taken over the bit
// patterns without the sign, so a NaN is the largest of all and reaches the scale of its block.
//
// Bound.  Each byte moves once, 7 bytes per element with a residual (x, r in; h, code out), 5 per output element of
// the gated form, except in int8 rows that shared memory does not hold (see kRowBytes), which are read twice.  e4m3
// (4096 x 8192 with residual 42.4 us, 4096 x 14336 SiLU 53.8 us) runs at 5.5 TB/s, 0.84 of the copy rate, with issue
// slots 54 % and 64 % busy and warps waiting for loads most: too few of them in flight.  GeLU (77.7 us) is bound by issue
// slots, 92 % busy at 45 instructions per column.  int8 rows run well below either bound (4096 x 8192 68 us,
// 4096 x 14336 SiLU 124 us): 84 registers in the norm, 2 blocks per SM, and a second pass over each row.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/xefuse_b200.h"
#include "xf_act.cuh"
#include "xf_host_util.h"
#include "xf_ptx.cuh"

namespace xf {
namespace quantize {

static const int kBlock = 128;        // columns that share a scale
static const int kChunk = 16;         // columns a thread handles at a time: 32 bytes of bf16, 16 bytes of codes
static const int kLanes = kBlock / kChunk;   // lanes that hold one block
static const int kAhead = 2;          // chunks whose loads a thread of the norm has in flight
static const float kFloor = 7.888609052210118e-31f;   // 2^-100

struct Params {
  const __nv_bfloat16* in;
  long long ld_in;
  const __nv_bfloat16* residual;      // null: none
  __nv_bfloat16* residual_out;        // the sum, where there is a residual
  long long ld_res, ld_res_out;
  const __nv_bfloat16* weight;        // null: ones
  uint8_t* out;
  long long ld_out;
  float* scale;
  long long scale_row, scale_blk;     // strides of the scales
  int M, N;
  float eps;
  int vec_in, vec_res, vec_out;       // 1: rows of that tensor start where 16-byte accesses may
  int vec_w;
  int row_bytes;                      // int8: bytes of shared memory that hold a row, 0: read it again
};

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

struct Chunk {
  uint4 v[2];
};
// Columns [c0, c0 + 16) of a bf16 row; columns from N on read as zero.
__device__ __forceinline__ Chunk load_chunk(const __nv_bfloat16* row, int c0, int N, int vec) {
  Chunk c;
  if (vec && c0 + kChunk <= N) {
    c.v[0] = *reinterpret_cast<const uint4*>(row + c0);
    c.v[1] = *reinterpret_cast<const uint4*>(row + c0 + 8);
    return c;
  }
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
  uint32_t w[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const uint32_t lo = c0 + 2 * t < N ? p[c0 + 2 * t] : 0;
    const uint32_t hi = c0 + 2 * t + 1 < N ? p[c0 + 2 * t + 1] : 0;
    w[t] = lo | (hi << 16);
  }
  c.v[0] = make_uint4(w[0], w[1], w[2], w[3]);
  c.v[1] = make_uint4(w[4], w[5], w[6], w[7]);
  return c;
}
__device__ __forceinline__ void store_chunk(__nv_bfloat16* row, int c0, int N, int vec, const Chunk& c) {
  if (vec && c0 + kChunk <= N) {
    *reinterpret_cast<uint4*>(row + c0) = c.v[0];
    *reinterpret_cast<uint4*>(row + c0 + 8) = c.v[1];
    return;
  }
  const uint32_t w[8] = {c.v[0].x, c.v[0].y, c.v[0].z, c.v[0].w, c.v[1].x, c.v[1].y, c.v[1].z, c.v[1].w};
#pragma unroll
  for (int i = 0; i < kChunk; ++i)
    if (c0 + i < N) reinterpret_cast<uint16_t*>(row)[c0 + i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
}
__device__ __forceinline__ void store_codes(uint8_t* row, int c0, int N, int vec, const uint32_t (&w)[4]) {
  if (vec && c0 + kChunk <= N) {
    *reinterpret_cast<uint4*>(row + c0) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < kChunk; ++i)
    if (c0 + i < N) row[c0 + i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
}

__device__ __forceinline__ void unpack(const Chunk& c, float (&v)[16]) {
  const uint32_t w[8] = {c.v[0].x, c.v[0].y, c.v[0].z, c.v[0].w, c.v[1].x, c.v[1].y, c.v[1].z, c.v[1].w};
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    v[2 * t] = bf_lo(w[t]);
    v[2 * t + 1] = bf_hi(w[t]);
  }
}
// Largest magnitude as a bit pattern; a NaN wins (its pattern is above infinity's).
__device__ __forceinline__ uint32_t absmax_bits(const float (&v)[16]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[i]), "f"(v[i + 1]));
  return __float_as_uint(m);
}

// Two values to e4m3, round to nearest even, values beyond 448 to 448, NaN kept.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two fp32 values in a register pair, and x * y and x * y + z on both at once.
__device__ __forceinline__ uint64_t both(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void apart(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
  uint64_t v;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
  return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(x), "l"(y), "l"(z));
  return v;
}
// The code of t * 448 / a as one product with 448 / a: for values that are themselves rounded.
__device__ __forceinline__ void codes_e4m3(const float (&t)[16], float a, uint32_t (&w)[4]) {
  const float inv = __fdiv_rn(448.0f, a);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = e4m3x2(t[4 * i] * inv, t[4 * i + 1] * inv) | (e4m3x2(t[4 * i + 2] * inv, t[4 * i + 3] * inv) << 16);
}
// The code of the exact quotient, for t and a of at most 16 significant bits (products of two bf16 values).  The
// product alone is rounded twice and misses a quotient that lies exactly between two codes in one case of seven.
// With s = 7/8 t, which is exact, the quotient is s / (a / 512): q = s * (512 / a) is next to it, the remainder
// q * a / 512 - s is exact in one multiply-add, and taking its 512 / a-th off q leaves the correctly rounded quotient.
// That hits every tie, and no other quotient is nearer to a tie than 2^-21 of it.  For an infinite a, q stays 0.
// Costs up to 1 us: 4096 x 8192 27.8 -> 28.9 us, with a residual 41.8 -> 42.2 us.
__device__ __forceinline__ void codes_e4m3_exact(const float (&t)[16], float a, uint32_t (&w)[4]) {
  const float inv = __fdiv_rn(512.0f, a), unit = __float_as_uint(a) == 0x7F800000u ? 0.0f : a * (1.0f / 512.0f);
  const uint64_t minus = both(-inv, -inv), unit2 = both(unit, unit), neg = both(-0.875f, -0.875f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t s = mul2(both(t[2 * i], t[2 * i + 1]), neg);     // -7/8 t
    uint64_t q = mul2(s, minus);
    q = fma2(fma2(q, unit2, s), minus, q);
    float lo, hi;
    apart(q, lo, hi);
    const uint32_t c = e4m3x2(lo, hi);
    if (i & 1) w[i >> 1] |= c << 16;
    else w[i >> 1] = c;
  }
}
// round(t * 127 / a), ties away from zero, of the exact quotient: the fp32 product is off by less
// than 2^-15 at 127, so only a value that close to a border between two codes is decided by the exact
// comparison 254 |t| >= (2 j - 1) a (both sides have at most 32 significant bits).
__device__ __forceinline__ int code_s8(float t, float a, float inv) {
  const float v = fabsf(t) * inv + 0.5f;
  const float j = rintf(v);
  float k = floorf(v);
  if (fabsf(v - j) < 6.2e-5f)
    k = 254.0 * static_cast<double>(fabsf(t)) >= (2.0 * j - 1.0) * static_cast<double>(a) ? j : j - 1.0f;
  const int q = static_cast<int>(fminf(k, 127.0f));
  return t < 0.0f ? -q : q;
}
__device__ __forceinline__ void codes_s8(const float (&t)[16], float a, uint32_t (&w)[4]) {
  const float inv = __fdiv_rn(127.0f, a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[i] |= (static_cast<uint32_t>(code_s8(t[4 * i + j], a, inv)) & 0xFFu) << (8 * j);
  }
}

// Largest value over the lanes that hold one block of 128 columns.
__device__ __forceinline__ uint32_t block_max(uint32_t a) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}
__device__ __forceinline__ float floored(uint32_t bits) {
  return __uint_as_float(max(bits, __float_as_uint(kFloor)));   // NaN bits are above every number's
}

// Sum and bitwise maximum over the block; `red` holds 2 x 32 words.
__device__ __forceinline__ void block_sum_max(float& s, uint32_t& m, uint32_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  m = __reduce_max_sync(0xffffffffu, m);
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (l == 0) {
    red[w] = __float_as_uint(s);
    red[32 + w] = m;
  }
  __syncthreads();
  s = l < nw ? __uint_as_float(red[l]) : 0.0f;
  m = l < nw ? red[32 + l] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  m = __reduce_max_sync(0xffffffffu, m);
}

// ---------------------------------------------------------------------------- norm
// One block per row.  e4m3: one pass; the codes of a 128-column block leave as soon as its lanes
// know their maximum, the maxima wait in shared memory for the row's sum.  int8: the summed row waits in
// shared memory for the row's maximum.
template <bool S8>
__global__ void __launch_bounds__(512) rms_norm_kernel(const Params p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ uint32_t red[64];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const long long row = blockIdx.x;
  const __nv_bfloat16* xr = p.in + row * p.ld_in;
  const __nv_bfloat16* rr = p.residual ? p.residual + row * p.ld_res : nullptr;
  __nv_bfloat16* hr = p.residual ? p.residual_out + row * p.ld_res_out : nullptr;
  uint8_t* qr = p.out + row * p.ld_out;
  const int nchunk = (p.N + kChunk - 1) / kChunk;
  const int lane = threadIdx.x & 31;
  float ss = 0.0f;
  uint32_t most = 0;
  for (int base = threadIdx.x; base - lane < nchunk; base += kAhead * blockDim.x) {
    // all loads of kAhead chunks before the first is used
    Chunk x[kAhead], r[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int c = base + k * blockDim.x;
      x[k] = r[k] = Chunk{};
      if (c < nchunk) {
        x[k] = load_chunk(xr, c * kChunk, p.N, p.vec_in);
        if (rr) r[k] = load_chunk(rr, c * kChunk, p.N, p.vec_res);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int c = base + k * blockDim.x, c0 = c * kChunk;
      if (c - lane >= nchunk) break;             // the whole warp
      Chunk u = x[k];
      float t[16];
      if (rr) {
        float b[16];
        unpack(u, t);
        unpack(r[k], b);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float *s = t + 8 * h, *o = b + 8 * h;
          u.v[h] = make_uint4(pack2(s[0] + o[0], s[1] + o[1]), pack2(s[2] + o[2], s[3] + o[3]),
                              pack2(s[4] + o[4], s[5] + o[5]), pack2(s[6] + o[6], s[7] + o[7]));
        }
        store_chunk(hr, c0, p.N, p.vec_res, u);
      }
      unpack(u, t);
#pragma unroll
      for (int i = 0; i < 16; ++i) ss = fmaf(t[i], t[i], ss);
      if (p.weight) {
        float w[16];
        unpack(load_chunk(p.weight, c0, p.N, p.vec_w), w);
#pragma unroll
        for (int i = 0; i < 16; ++i) t[i] *= w[i];
      }
      const uint32_t mine = absmax_bits(t);
      if (S8) {
        most = max(most, mine);
        if (p.row_bytes && c < nchunk) reinterpret_cast<Chunk*>(dyn)[c] = u;
      } else {
        const uint32_t a = block_max(mine);
        uint32_t codes[4];
        codes_e4m3_exact(t, floored(a), codes);
        store_codes(qr, c0, p.N, p.vec_out, codes);
        if (lane % kLanes == 0 && c < nchunk) reinterpret_cast<uint32_t*>(dyn)[c / kLanes] = a;
      }
    }
  }
  block_sum_max(ss, most, red);
  const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(ss / static_cast<float>(p.N) + p.eps));
  if (!S8) {
    const int nblk = (p.N + kBlock - 1) / kBlock;
    for (int b = threadIdx.x; b < nblk; b += blockDim.x)
      p.scale[row * p.scale_row + b * p.scale_blk] =
          __fdiv_rn(floored(reinterpret_cast<const uint32_t*>(dyn)[b]) * rstd, 448.0f);
    return;
  }
  const float a = floored(most);
  if (threadIdx.x == 0) p.scale[row * p.scale_row] = __fdiv_rn(a * rstd, 127.0f);
  const __nv_bfloat16* again = rr ? hr : xr;
  for (int c = threadIdx.x; c < nchunk; c += blockDim.x) {
    const int c0 = c * kChunk;
    // a thread reads back what it wrote itself
    const Chunk u = p.row_bytes ? reinterpret_cast<const Chunk*>(dyn)[c] : load_chunk(again, c0, p.N, rr ? p.vec_res : p.vec_in);
    float t[16];
    unpack(u, t);
    if (p.weight) {
      float w[16];
      unpack(load_chunk(p.weight, c0, p.N, p.vec_w), w);
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] *= w[i];
    }
    uint32_t codes[4];
    codes_s8(t, a, codes);
    store_codes(qr, c0, p.N, p.vec_out, codes);
  }
}

// ---------------------------------------------------------------------------- gate
template <bool GELU>
__device__ __forceinline__ void gated(const Chunk& g, const Chunk& u, float (&y)[16]) {
  float a[16], b[16];
  unpack(g, a);
  unpack(u, b);
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = (GELU ? gelu_rel(a[i]) : silu_fast(a[i])) * b[i];
}

// e4m3: kLanes lanes per block of 128 columns; nothing is shared beyond them.  A thread block works in one
// row, `segs` of them on each: the row comes from one uniform division.  Sixteen columns per thread halve
// what a block's maximum, division and addresses cost per column: 28 instructions with eight, 21 with sixteen
// (59 -> 54 us at 4096 x 14336, 5.5 TB/s).
template <bool GELU>
__global__ void __launch_bounds__(256) act_mul_e4m3_kernel(const Params p, unsigned segs) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const unsigned row = blockIdx.x / segs, seg = blockIdx.x - row * segs;
  const int c0 = (seg * blockDim.x + threadIdx.x) * kChunk;
  const __nv_bfloat16* xr = p.in + row * p.ld_in;
  float y[16];
  gated<GELU>(load_chunk(xr, c0, p.N, p.vec_in), load_chunk(xr + p.N, c0, p.N, p.vec_res), y);   // zeros beyond the row
  const float a = floored(block_max(absmax_bits(y)));    // all lanes of a warp take part in its shuffles
  if (c0 >= p.N) return;
  uint32_t codes[4];
  codes_e4m3(y, a, codes);
  store_codes(p.out + row * p.ld_out, c0, p.N, p.vec_out, codes);
  if (threadIdx.x % kLanes == 0) p.scale[row * p.scale_row + c0 / kBlock * p.scale_blk] = __fdiv_rn(a, 448.0f);
}

// int8: one block per row; the products wait in shared memory for the row's maximum, or are formed again
// in a row too long for it.
template <bool GELU>
__global__ void __launch_bounds__(512) act_mul_s8_kernel(const Params p) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ uint32_t red[64];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const long long row = blockIdx.x;
  const __nv_bfloat16* xr = p.in + row * p.ld_in;
  const int nchunk = (p.N + kChunk - 1) / kChunk;
  float4* kept = reinterpret_cast<float4*>(dyn);       // [4][nchunk]: neighbouring lanes side by side
  float none = 0.0f;
  uint32_t most = 0;
  for (int c = threadIdx.x; c < nchunk; c += blockDim.x) {
    float y[16];
    gated<GELU>(load_chunk(xr, c * kChunk, p.N, p.vec_in), load_chunk(xr + p.N, c * kChunk, p.N, p.vec_res), y);
    most = max(most, absmax_bits(y));
    if (p.row_bytes) {
#pragma unroll
      for (int i = 0; i < 4; ++i) kept[i * nchunk + c] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
    }
  }
  block_sum_max(none, most, red);
  const float a = floored(most);
  if (threadIdx.x == 0) p.scale[row * p.scale_row] = __fdiv_rn(a, 127.0f);
  for (int c = threadIdx.x; c < nchunk; c += blockDim.x) {
    float y[16];
    if (p.row_bytes) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = kept[i * nchunk + c];
        y[4 * i] = f.x; y[4 * i + 1] = f.y; y[4 * i + 2] = f.z; y[4 * i + 3] = f.w;
      }
    } else {
      gated<GELU>(load_chunk(xr, c * kChunk, p.N, p.vec_in), load_chunk(xr + p.N, c * kChunk, p.N, p.vec_res), y);
    }
    uint32_t codes[4];
    codes_s8(y, a, codes);
    store_codes(p.out + row * p.ld_out, c * kChunk, p.N, p.vec_out, codes);
  }
}

// ---------------------------------------------------------------------------- host
static int aligned(const void* p, long long pitch_bytes, int to) {
  return (reinterpret_cast<uintptr_t>(p) % to) == 0 && pitch_bytes % to == 0;
}

static xf_status check(const char* what, const xf_quantize_desc* d, long long in_cols) {
  if (!d) {
    set_error("%s: null descriptor", what);
    return XF_ERR_INVALID_PROBLEM;
  }
  if (d->M < 0 || d->N <= 0) {
    set_error("%s: extents must be positive (M=%d N=%d)", what, d->M, d->N);
    return XF_ERR_INVALID_PROBLEM;
  }
  if (d->out_dtype != XF_DT_S8 && d->out_dtype != XF_DT_E4M3) {
    set_error("%s: the output is int8 or e4m3 (got dtype %d)", what, d->out_dtype);
    return XF_ERR_INVALID_DATA_TYPE;
  }
  if (d->N > (1 << 20)) {
    set_error("%s: rows of at most %d columns (got %d)", what, 1 << 20, d->N);
    return XF_ERR_NOT_SUPPORTED;
  }
  if (d->M == 0) return XF_SUCCESS;
  if (!d->out || !d->scale || !d->input) {
    set_error("%s: null pointer", what);
    return XF_ERR_INVALID_PROBLEM;
  }
  if (d->ld_in < in_cols || d->ld_out < d->N || d->scale_row_stride < 1 ||
      (d->out_dtype == XF_DT_E4M3 && d->N > kBlock && d->scale_blk_stride < 1)) {
    set_error("%s: pitches too small (ld_in=%lld ld_out=%lld scale strides %lld, %lld; N=%d)", what,
              (long long)d->ld_in, (long long)d->ld_out, (long long)d->scale_row_stride,
              (long long)d->scale_blk_stride, d->N);
    return XF_ERR_INVALID_LAYOUT;
  }
  if (!d->residual != !d->residual_out) {
    set_error("%s: residual and residual_out go together", what);
    return XF_ERR_INVALID_PROBLEM;
  }
  if (d->residual && (d->ld_res < d->N || d->ld_res_out < d->N)) {
    set_error("%s: residual pitches %lld, %lld smaller than N=%d", what, (long long)d->ld_res,
              (long long)d->ld_res_out, d->N);
    return XF_ERR_INVALID_LAYOUT;
  }
  auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  if (((bits(d->input) | bits(d->residual) | bits(d->residual_out) | bits(d->weight)) & 1) || (bits(d->scale) & 3)) {
    set_error("%s: pointers must be aligned to their element size", what);
    return XF_ERR_MISALIGNED_OPERAND;
  }
  return XF_SUCCESS;
}

static Params params_of(const xf_quantize_desc* d) {
  Params p = {};
  p.in = static_cast<const __nv_bfloat16*>(d->input); p.ld_in = d->ld_in;
  p.residual = static_cast<const __nv_bfloat16*>(d->residual); p.ld_res = d->ld_res;
  p.residual_out = static_cast<__nv_bfloat16*>(d->residual_out); p.ld_res_out = d->ld_res_out;
  p.weight = static_cast<const __nv_bfloat16*>(d->weight);
  p.out = static_cast<uint8_t*>(d->out); p.ld_out = d->ld_out;
  p.scale = d->scale; p.scale_row = d->scale_row_stride; p.scale_blk = d->scale_blk_stride;
  p.M = d->M; p.N = d->N; p.eps = d->eps;
  p.vec_in = aligned(d->input, d->ld_in * 2, 16);
  p.vec_out = aligned(d->out, d->ld_out, 16);
  return p;
}

// Launches with programmatic stream serialization, like the products: the kernel waits for the previous
// grid before its first global access.
template <typename... Args>
static xf_status launch(const char* what, void (*fn)(Args...), unsigned grid, unsigned threads, size_t smem, void* stream,
                        Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, args...);
  if (e != cudaSuccess) {
    set_error("launch of %s failed: %s", what, cudaGetErrorString(e));
    return XF_ERR_INTERNAL;
  }
  return XF_SUCCESS;
}

// Threads for a row: one chunk each where there are few rows, kAhead where other rows keep the SM busy
// (4096 x 8192 with residual: 42.4 us, 5.5 TB/s; four chunks each 52 us).
static unsigned row_threads(int M, int N) {
  const int chunks = (N + kChunk - 1) / kChunk, each = M >= 512 ? kAhead : 1;
  const int t = ((chunks + each - 1) / each + 31) / 32 * 32;
  return t > 512 ? 512 : t;
}

// int8 rows up to this size wait in shared memory (48 KB need no opt-in): 24064 columns of the norm, 12032 of the gate,
// whose products wait in fp32.  Longer ones are read and, in the gate, activated twice: 4096 x 11008 66 us,
// 4096 x 14336 124 us.
static const int kRowBytes = 47 * 1024;

}  // namespace quantize
}  // namespace xf

extern "C" {

xf_status xf_rms_norm_quantize(const xf_quantize_desc* d, void* stream) {
  using namespace xf;
  using namespace xf::quantize;
  const char* what = "rms_norm_quantize";
  const xf_status s = quantize::check(what, d, d ? d->N : 0);
  if (s != XF_SUCCESS || d->M == 0) return s;
  Params p = params_of(d);
  p.vec_res = d->residual && aligned(d->residual, d->ld_res * 2, 16) && aligned(d->residual_out, d->ld_res_out * 2, 16);
  p.vec_w = aligned(d->weight, 0, 16);
  const int nchunk = (d->N + kChunk - 1) / kChunk;
  if (d->out_dtype == XF_DT_E4M3)
    return launch(what, rms_norm_kernel<false>, d->M, row_threads(d->M, d->N), (nchunk + kLanes - 1) / kLanes * sizeof(uint32_t), stream, p);
  p.row_bytes = nchunk * 32 <= kRowBytes ? nchunk * 32 : 0;
  return launch(what, rms_norm_kernel<true>, d->M, row_threads(d->M, d->N), p.row_bytes, stream, p);
}

xf_status xf_act_mul_quantize(const xf_quantize_desc* d, void* stream) {
  using namespace xf;
  using namespace xf::quantize;
  const char* what = "act_mul_quantize";
  const xf_status s = quantize::check(what, d, d ? 2LL * d->N : 0);
  if (s != XF_SUCCESS || d->M == 0) return s;
  if (d->residual || d->weight) {
    set_error("%s: takes neither residual nor weight", what);
    return XF_ERR_INVALID_PROBLEM;
  }
  Params p = params_of(d);
  p.vec_res = aligned(p.in + d->N, d->ld_in * 2, 16);      // the second half of the row
  if (d->out_dtype == XF_DT_E4M3) {
    const unsigned lanes = (d->N + kChunk - 1) / kChunk, threads = lanes < 256 ? (lanes + 31) / 32 * 32 : 256;
    const unsigned segs = (lanes + threads - 1) / threads;
    const unsigned long long grid = static_cast<unsigned long long>(d->M) * segs;
    if (grid > 0x7FFFFFFFull) {
      set_error("%s: more than 2^31 thread blocks (M=%d N=%d)", what, d->M, d->N);
      return XF_ERR_NOT_SUPPORTED;
    }
    return d->gelu ? launch(what, act_mul_e4m3_kernel<true>, static_cast<unsigned>(grid), threads, 0, stream, p, segs)
                   : launch(what, act_mul_e4m3_kernel<false>, static_cast<unsigned>(grid), threads, 0, stream, p, segs);
  }
  const int nchunk = (d->N + kChunk - 1) / kChunk;
  p.row_bytes = nchunk * 64 <= kRowBytes ? nchunk * 64 : 0;
  return d->gelu ? launch(what, act_mul_s8_kernel<true>, d->M, row_threads(d->M, d->N), p.row_bytes, stream, p)
                 : launch(what, act_mul_s8_kernel<false>, d->M, row_threads(d->M, d->N), p.row_bytes, stream, p);
}

}  // extern "C"
