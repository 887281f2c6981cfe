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
__device__ __forceinline__ uint32_t amax_bits8(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(f[e]) & 0x7fffffffu);
  return m;
}

// Two fp32 values -> two e4m3 codes, `lo` in the low byte.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float inv) {
  uint2 o;
  o.x = cvt_e4m3x2(__fmul_rn(f[0], inv), __fmul_rn(f[1], inv)) |
        (cvt_e4m3x2(__fmul_rn(f[2], inv), __fmul_rn(f[3], inv)) << 16);
  o.y = cvt_e4m3x2(__fmul_rn(f[4], inv), __fmul_rn(f[5], inv)) |
        (cvt_e4m3x2(__fmul_rn(f[6], inv), __fmul_rn(f[7], inv)) << 16);
  return o;
}

// Maximum over the 16 lanes that hold one block (eight values each).
__device__ __forceinline__ uint32_t block_max16(uint32_t bits) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  return max(bits, kFloorBits);
}

__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p, int64_t left, bool vec) {
  // `left`: values of the row from p on; what lies past them reads as zero.
  if (left <= 0) return make_uint4(0u, 0u, 0u, 0u);
  if (vec && left >= 8) return __ldg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) w[e >> 1] |= static_cast<uint32_t>(s[e]) << (16 * (e & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct ScaleOut {
  float* p;
  int64_t row, blk;      // strides in elements
};

// Codes of eight values at column `col` of a row: the row's pitch is a multiple of 16 bytes, and
// the columns past K up to that multiple are written as zeros.
__device__ __forceinline__ void store8(uint8_t* row, int64_t col, int64_t kpad, const uint2& o) {
  if (col < kpad) *reinterpret_cast<uint2*>(row + col) = o;
}

// One 16-lane group per (row, block); 16 groups per CTA.
__global__ void __launch_bounds__(256)
k_quantize_rows(const __nv_bfloat16* __restrict__ x, int64_t groups, int64_t K, int64_t ldx, uint32_t kblocks,
                bool vec, uint8_t* __restrict__ q, int64_t ldq, ScaleOut sc) {
  const int64_t g = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const int sub = threadIdx.x & 15;
  const bool live = g < groups;
  const int64_t gg = live ? g : 0;
  const int64_t row = gg / kblocks;
  const int64_t blk = gg - row * kblocks;
  const int64_t col = blk * kBlock + sub * 8;
  const uint4 v = load8(x + row * ldx + col, K - col, vec);
  const float a = __uint_as_float(block_max16(amax_bits8(v)));
  if (!live) return;
  float f[8];
  unpack8(v, f);
  store8(q + row * ldq, col, (K + 15) & ~int64_t(15), encode8(f, kTop / a));
  if (sub == 0) sc.p[row * sc.row + blk * sc.blk] = a / kTop;
}

// One CTA per 128 x 128 tile: 256 threads hold eight vectors of eight values each.
__global__ void __launch_bounds__(256)
k_quantize_tiles(const __nv_bfloat16* __restrict__ x, int64_t M, int64_t K, int64_t ldx, bool vec,
                 uint8_t* __restrict__ q, int64_t ldq, ScaleOut sc) {
  __shared__ uint32_t s_max[8];
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kBlock + (threadIdx.x & 15) * 8;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kBlock + (threadIdx.x >> 4);
  uint4 v[8];
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    v[i] = load8(x + row * ldx + col, row < M ? K - col : 0, vec);
    bits = max(bits, amax_bits8(v[i]));
  }
  bits = __reduce_max_sync(0xffffffffu, bits);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = bits;
  __syncthreads();
  bits = kFloorBits;
#pragma unroll
  for (int w = 0; w < 8; ++w) bits = max(bits, s_max[w]);
  const float a = __uint_as_float(bits);
  const float inv = kTop / a;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = row0 + 16 * i;
    if (row >= M) continue;
    float f[8];
    unpack8(v[i], f);
    store8(q + row * ldq, col, (K + 15) & ~int64_t(15), encode8(f, inv));
  }
  if (threadIdx.x == 0) sc.p[blockIdx.y * sc.row + blockIdx.x * sc.blk] = a / kTop;
}

// h = bf16(delta + residual) -> residual_out, y = h * rsqrt(mean h^2 + eps) * (w + 1) quantised
// from its fp32 value.  One CTA per row, kVpt vectors of eight values per thread held from the
// load to the conversion; vector i of a thread is vector tid + i * blockDim of the row, and
// blockDim is a multiple of 32, so the 16 lanes of a block stay together.
template <int kVpt>
__global__ void __launch_bounds__(1024)
k_add_rmsnorm_fp8(const __nv_bfloat16* __restrict__ delta, const __nv_bfloat16* residual,
                  const __nv_bfloat16* __restrict__ w, int K, float eps, __nv_bfloat16* residual_out,
                  uint8_t* __restrict__ q, int64_t ldq, ScaleOut sc) {
  __shared__ float s_part[32];
  const int64_t row = blockIdx.x;
  const int nvec = K / 8;
  const int tid = threadIdx.x, lane = tid & 31;
  float h[kVpt][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int v = tid + i * static_cast<int>(blockDim.x);
    uint4 r = make_uint4(0u, 0u, 0u, 0u);
    if (v < nvec) {
      r = *reinterpret_cast<const uint4*>(residual + row * K + v * 8);
      if (delta != nullptr) {
        const uint4 d = __ldg(reinterpret_cast<const uint4*>(delta + row * K + v * 8));
        float df[8], rf[8];
        unpack8(d, df);
        unpack8(r, rf);
        uint32_t o[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const __nv_bfloat162 p = __floats2bfloat162_rn(df[2 * t] + rf[2 * t], df[2 * t + 1] + rf[2 * t + 1]);
          o[t] = *reinterpret_cast<const uint32_t*>(&p);
        }
        r = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(residual_out + row * K + v * 8) = r;
      }
    }
    unpack8(r, h[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(h[i][e], h[i][e], ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) s_part[tid >> 5] = ss;
  __syncthreads();
  float part = lane < static_cast<int>(blockDim.x >> 5) ? s_part[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  const float rstd = rsqrtf(part / static_cast<float>(K) + eps);
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int v = tid + i * static_cast<int>(blockDim.x);
    float wf[8];
    unpack8(v < nvec ? __ldg(reinterpret_cast<const uint4*>(w + v * 8)) : make_uint4(0u, 0u, 0u, 0u), wf);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[i][e] = h[i][e] * rstd * (wf[e] + 1.0f);
    // past the row's end h is 0: such a value is 0, or NaN where rstd is, as its block then is
    const float a = __uint_as_float(block_max16(v < nvec ? amax_bits8(h[i]) : 0u));
    store8(q + row * ldq, v * 8, (K + 15) & ~15, v < nvec ? encode8(h[i], kTop / a) : make_uint2(0u, 0u));
    if ((v & 15) == 0 && v < nvec) sc.p[row * sc.row + (v >> 4) * sc.blk] = a / kTop;
  }
}

// silu(g) * u quantised from its fp32 value; silu(g) = g / (1 + e^-g).  One 16-lane group per
// (row, block) of the result.
__global__ void __launch_bounds__(256)
k_swiglu_fp8(const __nv_bfloat16* __restrict__ z, int64_t groups, int64_t inter, int64_t ldz, uint32_t kblocks,
             uint8_t* __restrict__ q, int64_t ldq, ScaleOut sc) {
  const int64_t g = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const int sub = threadIdx.x & 15;
  const bool live = g < groups;
  const int64_t gg = live ? g : 0;
  const int64_t row = gg / kblocks;
  const int64_t blk = gg - row * kblocks;
  const int64_t col = blk * kBlock + sub * 8;
  const __nv_bfloat16* p = z + row * ldz + col;
  float gf[8], uf[8];
  unpack8(load8(p, inter - col, true), gf);
  unpack8(load8(p + inter, inter - col, true), uf);
#pragma unroll
  for (int e = 0; e < 8; ++e) gf[e] = __fdividef(gf[e], 1.0f + __expf(-gf[e])) * uf[e];
  const float a = __uint_as_float(block_max16(amax_bits8(gf)));
  if (!live) return;
  store8(q + row * ldq, col, (inter + 15) & ~int64_t(15), encode8(gf, kTop / a));
  if (sub == 0) sc.p[row * sc.row + blk * sc.blk] = a / kTop;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What every producer asks of its outputs.
int check_codes(const void* q, int64_t ldq, int64_t K, const float* scale) {
  if (!q || !scale) return fail(LCG_ERR_BAD_ARG, "NULL argument");
  if (ldq < (K + 15) / 16 * 16 || ldq % 16 != 0)
    return fail(LCG_ERR_BAD_ARG, "the codes' pitch must be a multiple of 16 bytes and hold K=%lld rounded up to one, got %lld",
                (long long)K, (long long)ldq);
  if (!aligned16(q)) return fail(LCG_ERR_MISALIGNED, "the codes must be 16-byte aligned");
  return LCG_OK;
}

int group_grid(int64_t M, int64_t kblocks, unsigned* grid) {
  const int64_t ctas = (M * kblocks + 15) / 16;
  if (M > (int64_t(1) << 40) / kblocks || ctas > 0x7fffffffLL)
    return fail(LCG_ERR_UNSUPPORTED_SHAPE, "too many blocks: M=%lld, %lld blocks a row", (long long)M, (long long)kblocks);
  *grid = static_cast<unsigned>(ctas);
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
  if (int e = check_codes(q, ldq, K, scale)) return e;
  const bool vec = aligned16(x) && (ldx % 8 == 0 || M == 1);
  const int64_t kblocks = (K + kBlock - 1) / kBlock;
  const ScaleOut sc{scale, scale_row_stride, scale_block_stride};
  auto st = static_cast<cudaStream_t>(stream);
  auto xb = static_cast<const __nv_bfloat16*>(x);
  if (block_rows == 1) {
    unsigned grid;
    if (int e = group_grid(M, kblocks, &grid)) return e;
    k_quantize_rows<<<grid, 256, 0, st>>>(xb, M * kblocks, K, ldx, static_cast<uint32_t>(kblocks), vec,
                                          static_cast<uint8_t*>(q), ldq, sc);
  } else {
    const int64_t rblocks = (M + kBlock - 1) / kBlock;
    if (rblocks > 65535) return fail(LCG_ERR_UNSUPPORTED_SHAPE, "too many rows: M=%lld", (long long)M);
    k_quantize_tiles<<<dim3(static_cast<unsigned>(kblocks), static_cast<unsigned>(rblocks)), 256, 0, st>>>(
        xb, M, K, ldx, vec, static_cast<uint8_t*>(q), ldq, sc);
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
  const int vpt = (nvec + 1023) / 1024;
  // whole 16-byte groups of codes: the vectors are rounded up to an even count, the threads to whole warps
  const int threads = (((nvec + 1) / 2 * 2 + vpt - 1) / vpt + 31) / 32 * 32;
  const ScaleOut sc{scale, scale_row_stride, scale_block_stride};
  auto kern = vpt == 1 ? k_add_rmsnorm_fp8<1> : vpt == 2 ? k_add_rmsnorm_fp8<2> : k_add_rmsnorm_fp8<3>;
  kern<<<static_cast<unsigned>(M), threads, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(delta), static_cast<const __nv_bfloat16*>(residual),
      static_cast<const __nv_bfloat16*>(norm_weight), static_cast<int>(K), eps,
      static_cast<__nv_bfloat16*>(residual_out), static_cast<uint8_t*>(q), ldq, sc);
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
  if (int e = group_grid(M, kblocks, &grid)) return e;
  k_swiglu_fp8<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(z), M * kblocks, I, ldz, static_cast<uint32_t>(kblocks),
      static_cast<uint8_t*>(q), ldq, ScaleOut{scale, scale_row_stride, scale_block_stride});
  LCG_CUDA_OK(cudaGetLastError());
  count_launch();
  return LCG_OK;
}
