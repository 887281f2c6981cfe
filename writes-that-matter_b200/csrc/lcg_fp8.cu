// Producers of the 8-bit path's operands: e4m3 codes with one fp32 scale per block of 128
// values of a row (activations) or per 128 x 128 tile (weights), from a bf16 matrix, from the
// residual norm and from SwiGLU.
//
// One block:  a = max(max |x|, 2^-100),  scale = a / 448,  code = e4m3(x * (448 / a)),
// with correctly rounded fp32 divisions and product and one rounding to e4m3 (to nearest even,
// saturating: the product can pass 448 by its own rounding).  The floor on a keeps 448 / a finite and makes a
// block of zeros an ordinary one.  The maximum is taken over the magnitudes' bit patterns, whose
// order is that of the magnitudes with infinity and NaN on top, so one infinity or NaN leaves the
// block with an infinite or NaN scale and every value of it decodes to NaN.
//
// All of them are bound by HBM: every value is read once, held in registers between the maximum
// and the conversion, and written once.
#include <cuda_bf16.h>

#include "lcg_common.h"

namespace lcg {
namespace {

constexpr int kBlock = 128;                    // values under one scale
constexpr float kTop = 448.f;                  // largest e4m3 value
constexpr uint32_t kFloorBits = 27u << 23;     // 2^-100

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    f[2 * t] = __uint_as_float(w[t] << 16);
    f[2 * t + 1] = __uint_as_float(w[t] & 0xffff0000u);
  }
}

// Largest magnitude bit pattern of eight packed bf16 values, as fp32 bits.
__device__ __forceinline__ uint32_t amax_bits8(const uint4& q) {
  const uint32_t m = __vmaxu2(__vmaxu2(q.x & 0x7fff7fffu, q.y & 0x7fff7fffu),
                              __vmaxu2(q.z & 0x7fff7fffu, q.w & 0x7fff7fffu));
  return max(m << 16, m & 0xffff0000u);
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) {      // a NaN stays one
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t amax_bits8(const float (&f)[8]) {
  const float m = max3_abs(max3_abs(f[0], f[1], f[2]), max3_abs(f[3], f[4], f[5]), max3_abs(f[6], f[7], f[7]));
  return __float_as_uint(m) & 0x7fffffffu;
}

// Four fp32 values, scaled, -> four e4m3 codes, the first in the low byte.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, uint64_t inv2) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b64 p, q;\n\t"
      ".reg .b32 a, b, c, d;\n\t"
      ".reg .b16 l, h;\n\t"
      "mov.b64 p, {%1, %2};\n\t"
      "mov.b64 q, {%3, %4};\n\t"
      "mul.rn.f32x2 p, p, %5;\n\t"
      "mul.rn.f32x2 q, q, %5;\n\t"
      "mov.b64 {a, b}, p;\n\t"
      "mov.b64 {c, d}, q;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 l, b, a;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h, d, c;\n\t"
      "mov.b32 %0, {l, h};\n\t"
      "}"
      : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d), "l"(inv2));
  return r;
}
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float inv) {
  uint64_t inv2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(inv2) : "f"(inv));
  return make_uint2(encode4(f[0], f[1], f[2], f[3], inv2), encode4(f[4], f[5], f[6], f[7], inv2));
}

// 448 / a for the 16 lanes of a block, and in its odd lanes a / 448, the block's scale: one division, of
// different operands in even and odd lanes, as both are as long as half the rest of a block's work.
__device__ __forceinline__ float inverse_and_scale(float a, float& scale) {
  const bool odd = threadIdx.x & 1;
  scale = (odd ? a : kTop) / (odd ? kTop : a);
  return __shfl_sync(0xffffffffu, scale, (threadIdx.x & 31) & ~1);
}

// Maximum over the 16 lanes that hold one block (eight values each).
__device__ __forceinline__ uint32_t block_max16(uint32_t bits) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  return max(bits, kFloorBits);
}

// Read once: past L1.
__device__ __forceinline__ uint4 ldg_stream(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p, int left, bool vec) {
  // `left`: values of the row from p on; what lies past them reads as zero.
  if (left <= 0) return make_uint4(0u, 0u, 0u, 0u);
  if (vec && left >= 8) return ldg_stream(p);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) w[e >> 1] |= static_cast<uint32_t>(s[e]) << (16 * (e & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The (row, block) of the groups of 16 lanes that a CTA takes in turn, 16 apart.  All in 32 bits.
struct Walk {
  uint32_t groups, kblocks, step_row, step_blk;      // 16 = step_row * kblocks + step_blk
};
__device__ __forceinline__ void advance(const Walk& w, uint32_t& row, uint32_t& blk) {
  row += w.step_row;
  blk += w.step_blk;
  if (blk >= w.kblocks) blk -= w.kblocks, ++row;
}

struct ScaleOut {
  float* p;
  int64_t row, blk;      // strides in elements
};

// Codes of eight values at column `col` of a row: the row's pitch is a multiple of 16 bytes, and
// the columns past K up to that multiple are written as zeros.
__device__ __forceinline__ void store8(uint8_t* row, int col, int kpad, const uint2& o) {
  if (col < kpad) *reinterpret_cast<uint2*>(row + col) = o;
}
// In a block with a NaN the zeros read past K would get NaN codes.  A vector that lies past K as a whole is
// chosen to be zero; one that K cuts (K not a multiple of 8) has its end zeroed behind the store, by the thread that
// wrote it.  (A mask for both on the way to the store took swiglu from 71 to 78 us.)
__device__ __forceinline__ uint2 zero_past(int col, int K, const uint2& o) {
  return col < K ? o : make_uint2(0u, 0u);
}
__device__ __forceinline__ void zero_cut(uint8_t* row, int col, int K) {
  if (col < K)
    for (int c = K; c < col + 8; ++c) row[c] = 0;
}

// A 16-lane group to a block, 16 groups to a CTA, kRowUnroll blocks in turn to a group with all their
// loads in flight (4096 x 5120: one block at a time 19 us).  Five CTAs an SM.  Padding is
// zeroed while the loads are under way (4096 x 5128: 13.8 us of device time, 13.4 without, 15.6 where chosen at the store).
constexpr int kRowUnroll = 4;
template <int kTail>      // 0: K is a multiple of 16, 1: of 8, 2: of neither
__global__ void __launch_bounds__(256, 5)
k_quantize_rows(const __nv_bfloat16* __restrict__ x, const Walk w, int K, int64_t ldx, bool vec,
                uint8_t* __restrict__ q, int64_t ldq, ScaleOut sc) {
  const uint32_t g0 = blockIdx.x * (16u * kRowUnroll) + (threadIdx.x >> 4);
  const int sub = threadIdx.x & 15;
  const int kpad = (K + 15) & ~15;
  const uint32_t row0 = g0 / w.kblocks, blk0 = g0 - row0 * w.kblocks;
  uint4 v[kRowUnroll];
  uint32_t row = row0, blk = blk0;
#pragma unroll
  for (int j = 0; j < kRowUnroll; ++j) {
    const int col = static_cast<int>(blk) * kBlock + sub * 8;
    const bool in = g0 + 16 * j < w.groups;
    v[j] = load8(x + row * ldx + col, in ? K - col : 0, vec);
    if (kTail > 0 && in && col >= K && col < kpad) *reinterpret_cast<uint2*>(q + row * ldq + col) = make_uint2(0u, 0u);
    advance(w, row, blk);
  }
  row = row0;
  blk = blk0;
#pragma unroll
  for (int j = 0; j < kRowUnroll; ++j) {
    const float a = __uint_as_float(block_max16(amax_bits8(v[j])));
    float scale;
    const float inv = inverse_and_scale(a, scale);
    if (g0 + 16 * j < w.groups) {
      float f[8];
      unpack8(v[j], f);
      const int col = static_cast<int>(blk) * kBlock + sub * 8;
      store8(q + row * ldq, col, K, encode8(f, inv));
      if (kTail == 2) zero_cut(q + row * ldq, col, K);
      if (sub == 1) sc.p[row * sc.row + blk * sc.blk] = scale;
    }
    advance(w, row, blk);
  }
}

// A CTA to two neighbouring 128 x 128 tiles, a warp to 512 contiguous bytes of a row (one tile to a CTA,
// with 256 bytes of each row, took 78 us for 5120 x 17408): 512 threads hold eight vectors of eight values
// each, lanes 0-15 of the left tile and 16-31 of the right one.
__global__ void __launch_bounds__(512)
k_quantize_tiles(const __nv_bfloat16* __restrict__ x, int64_t M, int K, int64_t ldx, bool vec,
                 uint8_t* __restrict__ q, int64_t ldq, ScaleOut sc) {
  __shared__ uint32_t s_max[2][16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, side = lane >> 4;
  const int col = static_cast<int>(blockIdx.x) * (2 * kBlock) + lane * 8;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kBlock + warp;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kBlock), M - static_cast<int64_t>(blockIdx.y) * kBlock)) - warp;
  const __nv_bfloat16* p = x + row0 * ldx + col;
  uint4 v[8];
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = load8(p + 16 * i * ldx, 16 * i < rows ? K - col : 0, vec);
#pragma unroll
  for (int i = 0; i < 8; ++i) bits = max(bits, amax_bits8(v[i]));
  bits = block_max16(bits);
  if ((lane & 15) == 0) s_max[side][warp] = bits;
  __syncthreads();
  bits = block_max16(s_max[side][lane & 15]);
  float scale;
  const float inv = inverse_and_scale(__uint_as_float(bits), scale);
  uint8_t* o = q + row0 * ldq;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (16 * i < rows) {
      float f[8];
      unpack8(v[i], f);
      store8(o + 16 * i * ldq, col, (K + 15) & ~15, zero_past(col, K, encode8(f, inv)));
    }
  }
  if (isnan(inv) && K % 8 != 0) {
    for (int i = 0; 16 * i < rows; ++i) zero_cut(o + 16 * i * ldq, col, K);
  }
  const int blk = 2 * static_cast<int>(blockIdx.x) + side;
  if (warp == 0 && (lane & 15) == 1 && blk * kBlock < K) sc.p[blockIdx.y * sc.row + blk * sc.blk] = scale;
}

// h = bf16(delta + residual) -> residual_out, y = h * rsqrt(mean h^2 + eps) * (w + 1) quantised
// from its fp32 value.  One 16-lane group holds a block throughout, eight values to a lane.

__device__ __forceinline__ uint4 add_bf16x8(const uint4& x, const uint4& y) {
  float a[8], b[8];
  unpack8(x, a);
  unpack8(y, b);
  uint32_t o[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a[2 * t] + b[2 * t], a[2 * t + 1] + b[2 * t + 1]);
    o[t] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
// Squares of eight values added to two running sums.
__device__ __forceinline__ void add_squares(const uint4& h, uint64_t& ss) {
  float f[8];
  unpack8(h, f);
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint64_t p = pair(f[e], f[e + 1]);
    asm("fma.rn.f32x2 %0, %1, %1, %0;" : "+l"(ss) : "l"(p));
  }
}
__device__ __forceinline__ float sum_warp(uint64_t ss) {
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(ss));
  lo += hi;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lo += __shfl_xor_sync(0xffffffffu, lo, o);
  return lo;
}
// Vector v of a normalised row: quantised and stored.  All lanes; `in`: the vector lies in the row.
// Past the row's end h is 0: such a value is 0, or NaN where rstd is, as its block then is.
__device__ __forceinline__ void norm_store(const uint4& h, const uint4& w, float rstd, int v, bool in, int kpad,
                                           uint8_t* row, float* scales, int64_t blk_stride) {
  float y[8], wf[8];
  unpack8(h, y);
  unpack8(w, wf);
  const uint64_t one = pair(1.f, 1.f), r2 = pair(rstd, rstd);
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    uint64_t a = pair(y[e], y[e + 1]), b = pair(wf[e], wf[e + 1]);
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a) : "l"(r2));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(b) : "l"(one));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a) : "l"(b));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(y[e]), "=f"(y[e + 1]) : "l"(a));
  }
  const float a = __uint_as_float(block_max16(in ? amax_bits8(y) : 0u));
  float scale;
  const float inv = inverse_and_scale(a, scale);
  store8(row, v * 8, kpad, in ? encode8(y, inv) : make_uint2(0u, 0u));
  if ((v & 15) == 1 && v * 8 - 8 < kpad) scales[(v >> 4) * blk_stride] = scale;
}

// A CTA of at most 512 threads to a row, kVpt vectors to a thread: vector i of a thread is vector
// tid + i * blockDim of the row (blockDim a multiple of 32, so that a block's lanes stay together).  Two
// vectors rather than one (8192 x 5120 with a delta: 54.6 us against 48.4) halve what the reduction over
// the row costs, which every warp pays; a warp to a row pays it once but leaves 11 warps on an SM (127 us).
constexpr int kNormThreads = 512;
template <int kVpt>
__global__ void __launch_bounds__(kNormThreads, kVpt == 2 ? 4 : kVpt == 4 ? 2 : 1)
k_add_rmsnorm_fp8(const __nv_bfloat16* __restrict__ delta, const __nv_bfloat16* residual,
                  const __nv_bfloat16* __restrict__ w, int K, float inv_k, float eps, __nv_bfloat16* residual_out,
                  uint8_t* __restrict__ q, int64_t ldq, ScaleOut sc) {
  __shared__ float s_part[32];
  const int64_t row = blockIdx.x;
  const int nvec = K / 8;
  const int tid = threadIdx.x, lane = tid & 31;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  uint4 h[kVpt], d[kVpt], wv[kVpt];
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int v = tid + i * static_cast<int>(blockDim.x);
    h[i] = v < nvec ? *reinterpret_cast<const uint4*>(residual + row * K + v * 8) : zero;
    if (delta != nullptr) d[i] = v < nvec ? ldg_stream(delta + row * K + v * 8) : zero;
    wv[i] = v < nvec ? __ldg(reinterpret_cast<const uint4*>(w + v * 8)) : zero;
  }
  uint64_t ss = 0;
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int v = tid + i * static_cast<int>(blockDim.x);
    if (delta != nullptr) {
      h[i] = add_bf16x8(d[i], h[i]);
      if (v < nvec) *reinterpret_cast<uint4*>(residual_out + row * K + v * 8) = h[i];
    }
    add_squares(h[i], ss);
  }
  float part = sum_warp(ss);
  if (lane == 0) s_part[tid >> 5] = part;
  __syncthreads();
  part = lane < static_cast<int>(blockDim.x >> 5) ? s_part[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  const float rstd = rsqrtf(fmaf(part, inv_k, eps));
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int v = tid + i * static_cast<int>(blockDim.x);
    norm_store(h[i], wv[i], rstd, v, v < nvec, (K + 15) & ~15, q + row * ldq, sc.p + row * sc.row, sc.blk);
  }
}

// silu(g) = g / (1 + e^-g) with the hardware's base-2 exponential and reciprocal, subnormals to 0: right down to
// g = -87, where 1 / (1 + e^-g) is still a normal number.
constexpr float kFarGate = -87.f;
__device__ __forceinline__ float silu(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * r;
}
// silu(g) * u below that, where 1 + e^g is 1 and silu(g) alone may leave the range that its product with a large u is
// in: the exponential is split in two.
__device__ __forceinline__ float silu_far(float g, float u) {
  const float half = expf(0.5f * g);
  return (g * half) * (half * u);
}
__device__ __forceinline__ __nv_bfloat162 min8(const uint4& q) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
  return __hmin2(__hmin2(h[0], h[1]), __hmin2(h[2], h[3]));      // NaN left out
}

// One vector of a block: computed, quantised and stored; all lanes of a warp.  `in`: the block is one of the matrix's.
template <bool kFar>
__device__ __forceinline__ void glu_vector(const uint4& gv, const uint4& uv, bool in, uint32_t row, uint32_t blk, int inter,
                                           uint8_t* q, int64_t ldq, const ScaleOut& sc) {
  const int sub = threadIdx.x & 15;
  float gf[8], uf[8];
  unpack8(gv, gf);
  unpack8(uv, uf);
#pragma unroll
  for (int e = 0; e < 8; ++e) gf[e] = kFar && gf[e] < kFarGate ? silu_far(gf[e], uf[e]) : silu(gf[e]) * uf[e];
  const float a = __uint_as_float(block_max16(amax_bits8(gf)));
  float scale;
  const float inv = inverse_and_scale(a, scale);
  if (in) {
    const int col = static_cast<int>(blk) * kBlock + sub * 8;
    store8(q + row * ldq, col, (inter + 15) & ~15, zero_past(col, inter, encode8(gf, inv)));
    if (sub == 1) sc.p[row * sc.row + blk * sc.blk] = scale;
  }
}

// silu(g) * u quantised from its fp32 value.  A 16-lane group to a block of the
// result, kGluUnroll blocks in turn with all their loads in flight (4096 x 17408: 72, 68 and 64 us for one, two and four; with
// the search for far gates 3 % more).
constexpr int kGluUnroll = 4;
__device__ __forceinline__ void glu_load(const __nv_bfloat16* z, int64_t ldz, uint32_t row, uint32_t blk, bool in, int inter,
                                         uint4& gv, uint4& uv) {
  const int col = static_cast<int>(blk) * kBlock + (threadIdx.x & 15) * 8;
  const __nv_bfloat16* p = z + row * ldz + col;
  gv = load8(p, in ? inter - col : 0, true);
  uv = load8(p + inter, in ? inter - col : 0, true);
}
// The same blocks of a warp that has met a far gate, one by one and read again: the usual path keeps no registers and
// takes no branch for them (a branch in each vector took 74 us for 62 of device time).
__device__ __noinline__ void glu_far(const __nv_bfloat16* z, const Walk& w, int inter, int64_t ldz, uint8_t* q,
                                     int64_t ldq, const ScaleOut& sc) {
  const uint32_t g0 = blockIdx.x * (16u * kGluUnroll) + (threadIdx.x >> 4);
  uint32_t row = g0 / w.kblocks, blk = g0 - row * w.kblocks;
#pragma unroll 1
  for (int j = 0; j < kGluUnroll; ++j) {
    const bool in = g0 + 16 * j < w.groups;
    uint4 gv, uv;
    glu_load(z, ldz, row, blk, in, inter, gv, uv);
    glu_vector<true>(gv, uv, in, row, blk, inter, q, ldq, sc);
    advance(w, row, blk);
  }
}
__global__ void __launch_bounds__(256, 4)
k_swiglu_fp8(const __nv_bfloat16* __restrict__ z, const __grid_constant__ Walk w, int inter, int64_t ldz,
             uint8_t* __restrict__ q, int64_t ldq, const __grid_constant__ ScaleOut sc) {
  const uint32_t g0 = blockIdx.x * (16u * kGluUnroll) + (threadIdx.x >> 4);
  const uint32_t row0 = g0 / w.kblocks, blk0 = g0 - row0 * w.kblocks;
  uint4 gv[kGluUnroll], uv[kGluUnroll];
  uint32_t row = row0, blk = blk0;
#pragma unroll
  for (int j = 0; j < kGluUnroll; ++j) {
    glu_load(z, ldz, row, blk, g0 + 16 * j < w.groups, inter, gv[j], uv[j]);
    advance(w, row, blk);
  }
  __nv_bfloat162 least = min8(gv[0]);
#pragma unroll
  for (int j = 1; j < kGluUnroll; ++j) least = __hmin2(least, min8(gv[j]));
  if (__any_sync(0xffffffffu, fminf(__low2float(least), __high2float(least)) < kFarGate)) {
    glu_far(z, w, inter, ldz, q, ldq, sc);
    return;
  }
  row = row0;
  blk = blk0;
#pragma unroll
  for (int j = 0; j < kGluUnroll; ++j) {
    glu_vector<false>(gv[j], uv[j], g0 + 16 * j < w.groups, row, blk, inter, q, ldq, sc);
    advance(w, row, blk);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What every producer asks of its outputs.
int check_codes(const void* q, int64_t ldq, int64_t K, const float* scale) {
  if (!q || !scale) return fail(LCG_ERR_BAD_ARG, "NULL argument");
  if (ldq < (K + 15) / 16 * 16 || ldq % 16 != 0)
    return fail(LCG_ERR_BAD_ARG, "the codes' pitch must be a multiple of 16 bytes and hold K=%lld rounded up to one, got %lld",
                (long long)K, (long long)ldq);
  if (!aligned16(q)) return fail(LCG_ERR_MISALIGNED, "the codes must be 16-byte aligned");
  if (!aligned(scale, 4)) return fail(LCG_ERR_MISALIGNED, "the scales must be aligned to their type");
  return LCG_OK;
}

int make_walk(int64_t M, int64_t kblocks, int unroll, Walk* w, unsigned* grid) {
  if (M > 0x40000000LL / kblocks)
    return fail(LCG_ERR_UNSUPPORTED_SHAPE, "too many blocks: M=%lld, %lld blocks a row", (long long)M, (long long)kblocks);
  w->groups = static_cast<uint32_t>(M * kblocks);
  w->kblocks = static_cast<uint32_t>(kblocks);
  w->step_row = 16u / w->kblocks;
  w->step_blk = 16u % w->kblocks;
  *grid = (w->groups + 16 * unroll - 1) / (16 * unroll);
  return LCG_OK;
}

}  // namespace
}  // namespace lcg

using namespace lcg;

extern "C" int lcg_quantize_fp8(const void* x, int64_t M, int64_t K, int64_t ldx, int block_rows, void* q,
                                int64_t ldq, float* scale, int64_t scale_row_stride, int64_t scale_block_stride,
                                void* stream) {
  if (!x) return fail(LCG_ERR_BAD_ARG, "NULL argument");
  if (block_rows != 1 && block_rows != kBlock)
    return fail(LCG_ERR_BAD_ARG, "block_rows must be 1 or 128, got %d", block_rows);
  if (M < 1 || K < 1 || K > 0x7fffff00LL)
    return fail(LCG_ERR_UNSUPPORTED_SHAPE, "bad extents M=%lld K=%lld", (long long)M, (long long)K);
  if (ldx < K && M > 1) return fail(LCG_ERR_BAD_ARG, "leading dimension below extent");
  if (!aligned(x, 2)) return fail(LCG_ERR_MISALIGNED, "x must be aligned to its type");
  if (int e = check_codes(q, ldq, K, scale)) return e;
  const bool vec = aligned16(x) && (ldx % 8 == 0 || M == 1);
  const int64_t kblocks = (K + kBlock - 1) / kBlock;
  const ScaleOut sc{scale, scale_row_stride, scale_block_stride};
  auto st = static_cast<cudaStream_t>(stream);
  auto xb = static_cast<const __nv_bfloat16*>(x);
  if (block_rows == 1) {
    unsigned grid;
    Walk w;
    if (int e = make_walk(M, kblocks, kRowUnroll, &w, &grid)) return e;
    auto kern = K % 16 == 0 ? k_quantize_rows<0> : K % 8 == 0 ? k_quantize_rows<1> : k_quantize_rows<2>;
    kern<<<grid, 256, 0, st>>>(xb, w, static_cast<int>(K), ldx, vec, static_cast<uint8_t*>(q), ldq, sc);
  } else {
    const int64_t rblocks = (M + kBlock - 1) / kBlock;
    if (rblocks > 65535) return fail(LCG_ERR_UNSUPPORTED_SHAPE, "too many rows: M=%lld", (long long)M);
    k_quantize_tiles<<<dim3(static_cast<unsigned>((kblocks + 1) / 2), static_cast<unsigned>(rblocks)), 512, 0, st>>>(
        xb, M, static_cast<int>(K), ldx, vec, static_cast<uint8_t*>(q), ldq, sc);
  }
  LCG_CUDA_OK(cudaGetLastError());
  count_launch();
  return LCG_OK;
}

extern "C" int lcg_add_rmsnorm_fp8(const void* delta, const void* residual, const void* norm_weight, int64_t M,
                                   int64_t K, float eps, void* residual_out, void* q, int64_t ldq, float* scale,
                                   int64_t scale_row_stride, int64_t scale_block_stride, void* stream) {
  if (!residual || !norm_weight || (delta && !residual_out)) return fail(LCG_ERR_BAD_ARG, "NULL argument");
  if (M < 1 || M > 0x7fffffffLL || K < 8 || K % 8 != 0 || K > 24576)
    return fail(LCG_ERR_UNSUPPORTED_SHAPE, "needs K %% 8 == 0 and K <= 24576, got M=%lld K=%lld", (long long)M,
                (long long)K);
  if ((delta && !aligned16(delta)) || !aligned16(residual) || !aligned16(norm_weight) ||
      (delta && !aligned16(residual_out)))
    return fail(LCG_ERR_MISALIGNED, "all operands must be 16-byte aligned");
  if (int e = check_codes(q, ldq, K, scale)) return e;
  const int nvec = static_cast<int>(K / 8);
  const ScaleOut sc{scale, scale_row_stride, scale_block_stride};
  auto st = static_cast<cudaStream_t>(stream);
  auto db = static_cast<const __nv_bfloat16*>(delta), rb = static_cast<const __nv_bfloat16*>(residual),
       wb = static_cast<const __nv_bfloat16*>(norm_weight);
  auto ho = static_cast<__nv_bfloat16*>(residual_out);
  auto qb = static_cast<uint8_t*>(q);
  const float inv_k = 1.0f / static_cast<float>(K);
  // vectors of the row and of the codes' padding to a multiple of 16
  const int nslots = (nvec + 1) / 2 * 2;
  const int vpt = nslots <= 2 * kNormThreads ? 2 : nslots <= 4 * kNormThreads ? 4 : 6;
  const int threads = ((nslots + vpt - 1) / vpt + 31) / 32 * 32;
  auto kern = vpt == 2 ? k_add_rmsnorm_fp8<2> : vpt == 4 ? k_add_rmsnorm_fp8<4> : k_add_rmsnorm_fp8<6>;
  kern<<<static_cast<unsigned>(M), threads, 0, st>>>(db, rb, wb, static_cast<int>(K), inv_k, eps, ho, qb, ldq, sc);
  LCG_CUDA_OK(cudaGetLastError());
  count_launch();
  return LCG_OK;
}

extern "C" int lcg_swiglu_fp8(const void* z, int64_t M, int64_t I, int64_t ldz, void* q, int64_t ldq, float* scale,
                              int64_t scale_row_stride, int64_t scale_block_stride, void* stream) {
  if (!z) return fail(LCG_ERR_BAD_ARG, "NULL argument");
  if (M < 1 || I < 8 || I % 8 != 0 || I > 0x3fffff00LL || ((ldz < 2 * I || ldz % 8 != 0) && M > 1))
    return fail(LCG_ERR_UNSUPPORTED_SHAPE, "needs I %% 8 == 0 and 16-byte aligned rows, got M=%lld I=%lld",
                (long long)M, (long long)I);
  if (!aligned16(z)) return fail(LCG_ERR_MISALIGNED, "operands must be 16-byte aligned");
  if (int e = check_codes(q, ldq, I, scale)) return e;
  const int64_t kblocks = (I + kBlock - 1) / kBlock;
  unsigned grid;
  Walk w;
  if (int e = make_walk(M, kblocks, kGluUnroll, &w, &grid)) return e;
  k_swiglu_fp8<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(z), w, static_cast<int>(I), ldz, static_cast<uint8_t*>(q), ldq,
      ScaleOut{scale, scale_row_stride, scale_block_stride});
  LCG_CUDA_OK(cudaGetLastError());
  count_launch();
  return LCG_OK;
}
