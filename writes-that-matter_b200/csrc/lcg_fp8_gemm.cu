// The 8-bit product with a scale per block of 128:
//   c[m, n] = bf16( sum over blocks t:  a_scale[m, t] * b_scale[n / 128, t] * sum over k in t: a[m, k] * b[n, k] )
// a (M, K) and b (N, K) are e4m3 codes, the block sums and the scaled sum are fp32.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "lcg_common.h"

namespace lcg {
namespace {

constexpr int kBlock = 128;

struct Fp8Operand {
  const uint8_t* q;
  int64_t ld;
  const float* scale;
  int64_t s_row, s_blk;
};

__device__ __forceinline__ float decode(uint8_t v) {
  __nv_fp8_e4m3 x;
  x.__x = v;
  return static_cast<float>(x);
}

// 64 x 64 tile per CTA, 4 x 4 outputs per thread, 32 columns of K at a time.
__global__ void __launch_bounds__(256)
k_gemm_fp8_simple(Fp8Operand a, Fp8Operand b, __nv_bfloat16* __restrict__ c, int64_t ldc, int64_t M, int64_t N, int64_t K) {
  __shared__ float sa[32][65], sb[32][65];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 64, n0 = static_cast<int64_t>(blockIdx.x) * 64;
  float acc[4][4] = {};
  for (int64_t t = 0; t * kBlock < K; ++t) {
    float part[4][4] = {};
    for (int64_t k0 = t * kBlock; k0 < min(K, (t + 1) * kBlock); k0 += 32) {
      __syncthreads();
      for (int i = threadIdx.x; i < 64 * 32; i += 256) {
        const int r = i >> 5, k = i & 31;
        const bool in = k0 + k < K;
        sa[k][r] = in && m0 + r < M ? decode(a.q[(m0 + r) * a.ld + k0 + k]) : 0.f;
        sb[k][r] = in && n0 + r < N ? decode(b.q[(n0 + r) * b.ld + k0 + k]) : 0.f;
      }
      __syncthreads();
      for (int k = 0; k < 32; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], part[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
        if (m < M && n < N)
          acc[i][j] = fmaf(part[i][j], a.scale[m * a.s_row + t * a.s_blk] * b.scale[(n / kBlock) * b.s_row + t * b.s_blk],
                           acc[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m < M && n < N) c[m * ldc + n] = __float2bfloat16_rn(acc[i][j]);
    }
}

}  // namespace
}  // namespace lcg

using namespace lcg;

extern "C" int lcg_gemm_fp8(const void* a, int64_t lda, const float* a_scale, int64_t a_scale_row_stride,
                            int64_t a_scale_block_stride, const void* b, int64_t ldb, const float* b_scale,
                            int64_t b_scale_row_stride, int64_t b_scale_block_stride, void* c, int64_t ldc, int64_t M,
                            int64_t N, int64_t K, int32_t* status, void* stream) {
  (void)status;
  if (!a || !a_scale || !b || !b_scale || !c) return fail(LCG_ERR_BAD_ARG, "NULL operand");
  if (M < 1 || N < 1 || K < 1 || M > 0x7fffff00LL || N > 0x7fffff00LL || K > 0x7fffff00LL)
    return fail(LCG_ERR_UNSUPPORTED_SHAPE, "bad extents M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  const int64_t k16 = (K + 15) / 16 * 16;
  if (M == 1) lda = k16;      // the pitch of a single row is never used
  if (N == 1) ldb = k16;
  if (M == 1 && ldc < N) ldc = (N + 7) / 8 * 8;
  if (lda < K || ldb < K || ldc < N) return fail(LCG_ERR_BAD_ARG, "leading dimension below extent");
  if (lda % 16 != 0 || ldb % 16 != 0 || ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u) != 0)
    return fail(LCG_ERR_MISALIGNED, "codes must be 16-byte aligned with a pitch of a multiple of 16 bytes");
  if (ldc % 8 != 0 || (reinterpret_cast<uintptr_t>(c) & 15u) != 0)
    return fail(LCG_ERR_MISALIGNED, "the output must be 16-byte aligned with a pitch of a multiple of 8 elements");
  const Fp8Operand oa{static_cast<const uint8_t*>(a), lda, a_scale, a_scale_row_stride, a_scale_block_stride};
  const Fp8Operand ob{static_cast<const uint8_t*>(b), ldb, b_scale, b_scale_row_stride, b_scale_block_stride};
  if ((M + 63) / 64 > 65535) return fail(LCG_ERR_UNSUPPORTED_SHAPE, "too many rows: M=%lld", (long long)M);
  k_gemm_fp8_simple<<<dim3(static_cast<unsigned>((N + 63) / 64), static_cast<unsigned>((M + 63) / 64)), 256, 0,
                      static_cast<cudaStream_t>(stream)>>>(oa, ob, static_cast<__nv_bfloat16*>(c), ldc, M, N, K);
  LCG_CUDA_OK(cudaGetLastError());
  count_launch();
  return LCG_OK;
}
