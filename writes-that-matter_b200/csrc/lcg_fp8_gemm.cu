// The 8-bit product with a scale per block of 128:
//   c[m, n] = bf16( sum over blocks t:  a_scale[m, t] * b_scale[n / 128, t] * sum over k in t: a[m, k] * b[n, k] )
// a (M, K) and b (N, K) are e4m3 codes.  The tensor cores sum one block of 128 into TMEM
// (tcgen05.mma kind::f8f6f4, fp32); the scales differ from block to block, so every block's sum is
// read back, scaled and added to fp32 registers while the next block is being multiplied.
//
// Two kernels:
//   k_gemm_fp8      many rows: 2-CTA pairs, 256 x kBN tiles, bound by the tensor cores (or by the
//                   read-back, which moves 4 bytes of TMEM and does one FMA for every 128 MACs);
//   k_gemm_fp8_few  few rows: the weight takes the 128-row side of the instruction and the tokens
//                   the column side, K is split over a cluster, bound by reading the weight once.
#include <cuda_bf16.h>

#include <atomic>
#include <cstring>

#include "lcg_common.h"
#include "lcg_ptx.cuh"

namespace lcg {
namespace {

constexpr int kBlock = 128;              // K values under one scale = bytes of a swizzle row
constexpr int kSliceK = 32;              // K per tcgen05.mma
constexpr int kTileRows = 128;           // TMEM lanes
constexpr int kOperandBytes = kTileRows * kBlock;

struct Scales {
  const float* p;
  int64_t row, blk;                      // strides in elements
};

__device__ __forceinline__ void bar_sync(int id, int nthreads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Codes left in the status word by a wait that ran out (the GEMM family's, lcg_gemm.cu).
constexpr int kCodeProducer = 101, kCodeMmaAcc = 102, kCodeMmaFull = 103, kCodeEpilogue = 104;

// ================================================================ many rows
// A pair multiplies 256 rows of a by kBN rows of b; TMEM holds the sums of 512 / kBN blocks.  The
// read-back walks these stages in a loop unrolled over four blocks, so that barriers, parities and TMEM
// addresses are constants; the stages that the last K blocks of a tile leave over are only passed on.
// (With the MMA issuer unrolled as well and more waits inlined, the loops did not fit the instruction
// cache: 1054 us for 4096 x 34816 x 5120.  Four stages of 128 columns under a 256-wide tile, two MMAs to a slice of K, give
// the read-back more slack but read a's tile from shared memory twice: 765 us where two of 256 took 695.)
//
// 12 warps: 0 TMA producer, 1 MMA issuer, 2 and 3 scales, 4-7 and 8-11 read-back: every warp one
// TMEM lane quarter, each warpgroup half of the columns.
template <int kBN>
struct Many {
  static constexpr int kAcc = 512 / kBN;                    // TMEM stages
  static constexpr int kBRows = kBN / 2;                    // rows of b each CTA of the pair loads
  static constexpr int kStageBytes = kOperandBytes + kBRows * kBlock;
  static constexpr int kStages = kBN == 256 ? 5 : 7;
  static constexpr int kCols = kBN / 2;                     // columns per read-back warpgroup
  static constexpr int kStoreBytes = 32 * 128;              // a warp's staged 32 x 64 bf16
  static constexpr int kGroup = 4;                          // K blocks whose scales travel together
  static_assert(kGroup % kAcc == 0, "scales change between walks of the stages");
  static constexpr int kSlots = 4;
  static constexpr int kSlotFloats = kGroup * 2 * kTileRows;
  static constexpr int kSmemBytes = kStages * kStageBytes + 8 * kStoreBytes + kSlots * kSlotFloats * 4 + 256 + 1024;
};
constexpr int kManyThreads = 384;

struct ManyParams {
  Scales a, b;
  __nv_bfloat16* c;
  int64_t ldc;
  int32_t m, n, k_blocks, tiles_m, tiles_n, group_m, num_tiles;
  int32_t* status;
};

template <int kBN>
__global__ void __launch_bounds__(kManyThreads, 1)
k_gemm_fp8(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
           const __grid_constant__ CUtensorMap tma_c, const __grid_constant__ ManyParams p) {
  using T = Many<kBN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t store_base = base + T::kStages * T::kStageBytes;
  const uint32_t scale_base = store_base + 8 * T::kStoreBytes;
  float* scales = reinterpret_cast<float*>(smem_raw + (scale_base - raw));
  const uint32_t bar_base = scale_base + T::kSlots * T::kSlotFloats * 4;
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (T::kStages + s); };
  auto acc_full_bar = [&](uint32_t s) { return bar_base + 8u * (2 * T::kStages + s); };
  auto acc_empty_bar = [&](uint32_t s) { return bar_base + 8u * (2 * T::kStages + T::kAcc + s); };
  auto scale_full_bar = [&](uint32_t s) { return bar_base + 8u * (2 * T::kStages + 2 * T::kAcc + s); };
  auto scale_empty_bar = [&](uint32_t s) { return bar_base + 8u * (2 * T::kStages + 2 * T::kAcc + T::kSlots + s); };
  const uint32_t misc = bar_base + 8u * (2 * T::kStages + 2 * T::kAcc + 2 * T::kSlots);
  static_assert(8 * (2 * T::kStages + 2 * T::kAcc + 2 * T::kSlots) + 8 <= 256, "barrier area");
  volatile uint32_t* misc_gen = reinterpret_cast<volatile uint32_t*>(smem_raw + (misc - raw));
  // misc_gen[0] = TMEM base, [1] = abort flag

  // warp-uniform by construction, so that the single-thread roles keep their state in uniform registers
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t cta_rank = cluster_ctarank();
  const bool leader = cta_rank == 0;
  const int pair = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;
  const WaitCtl ctl{&misc_gen[1], p.status};

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < T::kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (uint32_t s = 0; s < T::kAcc; ++s) {
      mbar_init(acc_full_bar(s), 1);
      mbar_init(acc_empty_bar(s), 16);     // the read-back warps of both CTAs
    }
    for (uint32_t s = 0; s < T::kSlots; ++s) {
      mbar_init(scale_full_bar(s), 2);     // both scale warps
      mbar_init(scale_empty_bar(s), 8);    // the read-back warps of this CTA
    }
    misc_gen[1] = 0u;
    fence_mbar_init();
    prefetch_tensormap(&tma_a);
    prefetch_tensormap(&tma_b);
    prefetch_tensormap(&tma_c);
  }
  if (warp == 1) {
    tmem_alloc<2>(misc, 512);
    tmem_relinquish<2>();
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  tcgen05_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, misc_gen[0], 0);

  // Bands of group_m tile rows, tile row fastest inside a band (lcg_gemm.cu: tile_coord).
  auto tile_at = [&](int t, int& tm, int& tn) {
    const int band_sz = p.group_m * p.tiles_n;
    const int band = t / band_sz;
    const int rem = t - band * band_sz;
    const int gm = min(p.group_m, p.tiles_m - band * p.group_m);
    tm = band * p.group_m + rem % gm;
    tn = rem / gm;
  };

  if (warp < 4) {
    regs_dec<40>();
    if (warp == 0) {
      // ---------------------------------------------------------- TMA producer
      uint32_t stage = 0, wait_parity = 1;
      const uint32_t full_leader = mapa_shared(full_bar(0), 0);
      for (int t = pair; t < p.num_tiles; t += num_pairs) {
        int tm, tn;
        tile_at(t, tm, tn);
        const int a_row = tm * 2 * kTileRows + static_cast<int>(cta_rank) * kTileRows;
        const int b_row = tn * kBN + static_cast<int>(cta_rank) * T::kBRows;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          mbar_wait_inline(empty_bar(stage), wait_parity, ctl, kCodeProducer);
          if (elect_one()) {
            if (leader) mbar_arrive_expect_tx(full_bar(stage), 2 * T::kStageBytes);
            const uint32_t sa = base + stage * T::kStageBytes;
            const uint32_t bar = full_leader + 8u * stage;
            tma_load_2d_pair(sa, &tma_a, bar, kb * kBlock, a_row);
            tma_load_2d_pair(sa + kOperandBytes, &tma_b, bar, kb * kBlock, b_row);
          }
          __syncwarp();
          if (++stage == T::kStages) {
            stage = 0;
            wait_parity ^= 1u;
          }
        }
      }
      drain_ring(T::kStages, stage, wait_parity,
                 [&](uint32_t s, uint32_t parity) { mbar_wait_inline(empty_bar(s), parity, ctl, kCodeProducer); });
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer
      // The whole warp walks the loop and one lane issues: descriptors and addresses then live in
      // uniform registers.  With one lane in the loop every instruction first moved its operands
      // there, 75 cycles for each MMA, more than the MMA takes.
      if (leader) {
        constexpr uint32_t idesc = make_idesc_e4m3(2 * kTileRows, kBN);
        const uint64_t adesc0 = make_kmajor_sw128_desc(base);
        const uint64_t bdesc0 = make_kmajor_sw128_desc(base + kOperandBytes);
        uint32_t stage = 0, parity = 0, as = 0, acc_parity = 1;
        auto next_stage = [&] {
          if (++as == T::kAcc) {
            as = 0;
            acc_parity ^= 1u;
          }
        };
        for (int t = pair; t < p.num_tiles; t += num_pairs) {
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            const uint64_t soff = static_cast<uint64_t>(stage * (T::kStageBytes >> 4));
            bool acc_ok, full_ok;
            mbar_try_wait_both(acc_empty_bar(as), acc_parity, full_bar(stage), parity, acc_ok, full_ok);
            if (!acc_ok) mbar_wait_inline(acc_empty_bar(as), acc_parity, ctl, kCodeMmaAcc);
            if (!full_ok) mbar_wait_inline(full_bar(stage), parity, ctl, kCodeMmaFull);
            tcgen05_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kBlock / kSliceK; ++k)
                umma_fp8<2>(tmem_base + as * kBN, adesc0 + soff + 2u * k, bdesc0 + soff + 2u * k, idesc, k > 0);
              umma_commit<2>(acc_full_bar(as));
              umma_commit<2>(empty_bar(stage));
            }
            __syncwarp();
            next_stage();
            if (++stage == T::kStages) {
              stage = 0;
              parity ^= 1u;
            }
          }
          while (as != 0) {          // every tile starts at stage 0
            mbar_wait_inline(acc_empty_bar(as), acc_parity, ctl, kCodeMmaAcc);
            if (elect_one()) umma_commit<2>(acc_full_bar(as));
            __syncwarp();
            next_stage();
          }
        }
      }
    } else {
      // ---------------------------------------------------------------- scales
      // a's scale times b's for every row and both warpgroups' columns, kGroup blocks at a time:
      // slot[block][warpgroup][row].  Read by the read-back warps themselves, their latency showed up
      // in every second block.
      const int r = threadIdx.x - 64;
      uint32_t slot = 0, wait_parity = 1;
      for (int t = pair; t < p.num_tiles; t += num_pairs) {
        int tm, tn;
        tile_at(t, tm, tn);
        const int row0 = tm * 2 * kTileRows + static_cast<int>(cta_rank) * kTileRows + r;
        const float* sa0 = p.a.p + min(row0, p.m - 1) * p.a.row;
        const float* sa1 = p.a.p + min(row0 + 64, p.m - 1) * p.a.row;
        const float* sb0 = p.b.p + (min(tn * kBN, p.n - 1) / kBlock) * p.b.row;
        const float* sb1 = p.b.p + (min(tn * kBN + T::kCols, p.n - 1) / kBlock) * p.b.row;
        for (int kb0 = 0; kb0 < p.k_blocks; kb0 += T::kGroup) {
          float a0[T::kGroup], a1[T::kGroup], b0[T::kGroup], b1[T::kGroup];
#pragma unroll
          for (int i = 0; i < T::kGroup; ++i) {
            const int kb = min(kb0 + i, p.k_blocks - 1);
            a0[i] = __ldg(sa0 + kb * p.a.blk);
            a1[i] = __ldg(sa1 + kb * p.a.blk);
            b0[i] = __ldg(sb0 + kb * p.b.blk);
            b1[i] = __ldg(sb1 + kb * p.b.blk);
          }
          mbar_wait_inline(scale_empty_bar(slot), wait_parity, ctl, kCodeProducer);
          float* dst = scales + slot * T::kSlotFloats + r;
#pragma unroll
          for (int i = 0; i < T::kGroup; ++i) {
            dst[(2 * i) * kTileRows] = a0[i] * b0[i];
            dst[(2 * i) * kTileRows + 64] = a1[i] * b0[i];
            dst[(2 * i + 1) * kTileRows] = a0[i] * b1[i];
            dst[(2 * i + 1) * kTileRows + 64] = a1[i] * b1[i];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(scale_full_bar(slot));
          if (++slot == T::kSlots) {
            slot = 0;
            wait_parity ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else {
    regs_inc<232>();
    // ---------------------------------------------------------------- read-back
    const int quarter = warp & 3;
    const int wg = (warp >> 2) - 1;
    const uint32_t acc_empty_leader = mapa_shared(acc_empty_bar(0), 0);
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + wg * T::kCols;
    const uint32_t buf = store_base + (warp - 4) * T::kStoreBytes;
    const float* my_scale = scales + wg * kTileRows + quarter * 32 + lane;
    uint32_t acc_parity = 0, slot = 0, slot_parity = 0;
    for (int t = pair; t < p.num_tiles; t += num_pairs) {
      uint64_t acc[T::kCols / 2];
#pragma unroll
      for (int j = 0; j < T::kCols / 2; ++j) acc[j] = 0;
      // Loads of 32 columns.  The wait is for all of a warp's loads, so there is one in flight: each is issued
      // before the one in front of it is used, across the stages of a tile too.
      constexpr int kChunks = T::kCols / 32;
      constexpr uint32_t kFlip = (T::kGroup / T::kAcc) & 1;     // whether a group leaves the stages' parity changed
      uint32_t group_parity = acc_parity;
      uint32_t v[2][32];
      mbar_wait_inline(acc_full_bar(0), acc_parity, ctl, kCodeEpilogue);
      tcgen05_fence_after();
      tmem_ld_32x32(lane_addr, v[0]);
      for (int kb0 = 0; kb0 < p.k_blocks; kb0 += T::kGroup) {
        mbar_wait_inline(scale_full_bar(slot), slot_parity, ctl, kCodeEpilogue);
        float sc[T::kGroup];
#pragma unroll
        for (int i = 0; i < T::kGroup; ++i) sc[i] = my_scale[slot * T::kSlotFloats + 2 * i * kTileRows];
        __syncwarp();
        if (lane == 0) mbar_arrive(scale_empty_bar(slot));
        if (++slot == T::kSlots) {
          slot = 0;
          slot_parity ^= 1u;
        }
#pragma unroll
        for (int i = 0; i < T::kGroup; ++i) {
          if (kb0 + i < p.k_blocks) {
            const uint64_t s2 = pack_f32x2(__float_as_uint(sc[i]), __float_as_uint(sc[i]));
            const uint32_t as = i % T::kAcc, next = (i + 1) % T::kAcc;
            const uint32_t next_parity = group_parity ^ (((i + 1) / T::kAcc) & 1);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              tmem_ld_wait(v[c & 1]);
              if (c + 1 < kChunks) {
                tmem_ld_32x32(lane_addr + as * kBN + (c + 1) * 32, v[(c + 1) & 1]);
              } else {          // everything is in registers: the stage goes back, the next one begins
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty_leader + 8u * as);
                if (kb0 + i + 1 < p.k_blocks) {
                  mbar_wait_inline(acc_full_bar(next), next_parity, ctl, kCodeEpilogue);
                  tcgen05_fence_after();
                  tmem_ld_32x32(lane_addr + next * kBN, v[0]);
                }
              }
#pragma unroll
              for (int j = 0; j < 16; ++j)
                acc[c * 16 + j] = fma_f32x2(pack_f32x2(v[c & 1][2 * j], v[c & 1][2 * j + 1]), s2, acc[c * 16 + j]);
            }
          }
        }
        group_parity ^= kFlip;
      }
      const int last_walk = (p.k_blocks - 1) / T::kAcc;
      for (int s = (p.k_blocks - 1) % T::kAcc + 1; s < T::kAcc; ++s) {      // passed on (see the issuer)
        mbar_wait_inline(acc_full_bar(s), acc_parity ^ (last_walk & 1), ctl, kCodeEpilogue);
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty_leader + 8u * s);
      }
      acc_parity ^= (last_walk + 1) & 1;
      // bf16, 64 columns at a time through this warp's staging buffer
      int tm, tn;
      tile_at(t, tm, tn);
      const int row0 = tm * 2 * kTileRows + static_cast<int>(cta_rank) * kTileRows + quarter * 32;
      const int col0 = tn * kBN + wg * T::kCols;
#pragma unroll
      for (int h = 0; h < T::kCols / 64; ++h) {
        if (lane == 0) bulk_wait_group_read<0>();
        __syncwarp();
        uint32_t pk[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          float lo, hi;
          unpack_f32x2(acc[h * 32 + j], lo, hi);
          pk[j] = pack_bf16x2(lo, hi);
        }
#pragma unroll
        for (int c = 0; c < 8; ++c)
          st_shared_v4(buf + lane * 128 + ((c ^ (lane & 7)) << 4), pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
        const int col = col0 + h * 64;
        if (col + 64 > p.n && (p.n & 7) != 0) {
          // A bulk store writes whole 16-byte pieces, past the last column where N is not a multiple
          // of 8: the edge goes out element by element.
          __syncwarp();
          for (int r = 0; r < 32 && row0 + r < p.m; ++r)
            for (int e = lane; e < 64 && col + e < p.n; e += 32) {
              uint16_t v;
              asm volatile("ld.shared.u16 %0, [%1];"
                           : "=h"(v) : "r"(buf + r * 128 + (((e >> 3) ^ (r & 7)) << 4) + (e & 7) * 2) : "memory");
              reinterpret_cast<uint16_t*>(p.c)[static_cast<int64_t>(row0 + r) * p.ldc + col + e] = v;
            }
          __syncwarp();
        } else {
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) {
            if (row0 < p.m && col < p.n) tma_store_2d(&tma_c, buf, col, row0);
            bulk_commit_group();
          }
        }
      }
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }

  // -------------------------------------------------------------------- teardown
  if (misc_gen[1] != 0u && warp == 0) {      // a wait ran out: let loads in flight land first
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc<2>(tmem_base, 512);
  }
}

// ================================================================= few rows
// Warps: 0 TMA producer, 1 MMA issuer, 2-5 (2-9 for 128 tokens) read-back, 64 tokens at most to a warp.  A
// CTA multiplies 128 rows of the weight by kBT tokens over its share of the K blocks; the CTAs of a
// cluster share one tile's K and add their parts in rank order through distributed shared memory.
template <int kBT>
struct Few {
  static constexpr int kStageBytes = kOperandBytes + kBT * kBlock;
  static constexpr int kCtas = kBT == 128 ? 1 : 2;          // CTAs to an SM
  static constexpr int kStages = kBT == 16 ? 6 : kBT == 32 ? 5 : kBT == 64 ? 4 : 6;
  static constexpr int kReaders = kBT == 128 ? 8 : 4;       // read-back warps
  static constexpr int kThreads = 64 + 32 * kReaders;
  static constexpr int kCols = kBT * 4 / kReaders;          // tokens to a warp
  static constexpr int kAcc = 4;
  static constexpr int kTmemCols = kAcc * kBT;
  static constexpr int kAhead = 4;                          // K blocks whose scales are staged together
  static constexpr int kScaleBytes = 2 * kAhead * kBT * 4;
  static constexpr int kSmemBytes = kStages * kStageBytes + kScaleBytes + 256 + 1024;
};
constexpr int kMaxSplit = 8;

struct FewParams {
  Scales a, b;
  __nv_bfloat16* c;
  int64_t ldc;
  int32_t m, n, k_blocks, split;      // m <= kBT: one tile of tokens
  int32_t* status;
};

template <int kBT>
__global__ void __launch_bounds__(Few<kBT>::kThreads, Few<kBT>::kCtas)
k_gemm_fp8_few(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x,
               const __grid_constant__ FewParams p) {
  using T = Few<kBT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - raw);
  float* part = reinterpret_cast<float*>(gen);              // after the last product: [kBT][128] sums
  float* scales = reinterpret_cast<float*>(gen + T::kStages * T::kStageBytes);
  const uint32_t bar_base = base + T::kStages * T::kStageBytes + T::kScaleBytes;
  auto full_bar = [&](uint32_t s) { return bar_base + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar_base + 8u * (T::kStages + s); };
  auto acc_full_bar = [&](uint32_t s) { return bar_base + 8u * (2 * T::kStages + s); };
  auto acc_empty_bar = [&](uint32_t s) { return bar_base + 8u * (2 * T::kStages + T::kAcc + s); };
  const uint32_t misc = bar_base + 8u * (2 * T::kStages + 2 * T::kAcc);
  volatile uint32_t* misc_gen = reinterpret_cast<volatile uint32_t*>(smem_raw + (misc - raw));

  // warp-uniform by construction, so that the single-thread roles keep their state in uniform registers
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = blockIdx.x / p.split;
  const int n0 = tile * kTileRows;
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * rank / p.split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (rank + 1) / p.split);
  const WaitCtl ctl{&misc_gen[1], p.status};

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < T::kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (uint32_t s = 0; s < T::kAcc; ++s) {
      mbar_init(acc_full_bar(s), 1);
      mbar_init(acc_empty_bar(s), T::kReaders);
    }
    misc_gen[1] = 0u;
    fence_mbar_init();
    prefetch_tensormap(&tma_w);
    prefetch_tensormap(&tma_x);
  }
  if (warp == 1) {
    tmem_alloc<1>(misc, T::kTmemCols);
    tmem_relinquish<1>();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, misc_gen[0], 0);

  if (warp == 0) {
    uint32_t stage = 0, wait_parity = 1;
    for (int kb = kb0; kb < kb1; ++kb) {
      mbar_wait_inline(empty_bar(stage), wait_parity, ctl, kCodeProducer);
      if (elect_one()) {
        mbar_arrive_expect_tx(full_bar(stage), T::kStageBytes);
        const uint32_t sw = base + stage * T::kStageBytes;
        tma_load_2d(sw, &tma_w, full_bar(stage), kb * kBlock, n0);
        tma_load_2d(sw + kOperandBytes, &tma_x, full_bar(stage), kb * kBlock, 0);
      }
      __syncwarp();
      if (++stage == T::kStages) {
        stage = 0;
        wait_parity ^= 1u;
      }
    }
    drain_ring(T::kStages, stage, wait_parity,
               [&](uint32_t s, uint32_t parity) { mbar_wait_inline(empty_bar(s), parity, ctl, kCodeProducer); });
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_e4m3(kTileRows, kBT);
    const uint64_t wdesc0 = make_kmajor_sw128_desc(base);
    const uint64_t xdesc0 = make_kmajor_sw128_desc(base + kOperandBytes);
    uint32_t stage = 0, parity = 0, as = 0, acc_parity = 1;
    for (int kb = kb0; kb < kb1; ++kb) {
      mbar_wait_inline(acc_empty_bar(as), acc_parity, ctl, kCodeMmaAcc);
      mbar_wait_inline(full_bar(stage), parity, ctl, kCodeMmaFull);
      tcgen05_fence_after();
      const uint64_t soff = static_cast<uint64_t>(stage * (T::kStageBytes >> 4));
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kBlock / kSliceK; ++k)
          umma_fp8<1>(tmem_base + as * kBT, wdesc0 + soff + 2u * k, xdesc0 + soff + 2u * k, idesc, k > 0);
        umma_commit<1>(acc_full_bar(as));
        umma_commit<1>(empty_bar(stage));
      }
      __syncwarp();
      if (++stage == T::kStages) {
        stage = 0;
        parity ^= 1u;
      }
      if (++as == T::kAcc) {
        as = 0;
        acc_parity ^= 1u;
      }
    }
  } else {
    // ---------------------------------------------------------------- read-back
    constexpr int kReadThreads = 32 * T::kReaders;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int tok0 = ((warp - 2) >> 2) * T::kCols;         // this warp's first token of the tile
    const int pt = threadIdx.x - 64;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + tok0;
    // Scales of kAhead blocks at a time, a's times b's, staged by all the read-back warps: [block][token].
    constexpr int kPer = (T::kAhead * kBT + kReadThreads - 1) / kReadThreads;
    float na[kPer], nb[kPer];
    const float* sb = p.b.p + tile * p.b.row;
    auto fetch = [&](int kbs) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = pt + i * kReadThreads;
        const int kb = kbs + e / kBT, j = e % kBT;
        const bool in = e < T::kAhead * kBT && kb < kb1 && j < p.m;
        na[i] = in ? __ldg(p.a.p + j * p.a.row + kb * p.a.blk) : 0.f;
        nb[i] = in ? __ldg(sb + kb * p.b.blk) : 0.f;
      }
    };
    uint64_t acc[T::kCols / 2];
#pragma unroll
    for (int j = 0; j < T::kCols / 2; ++j) acc[j] = 0;
    uint32_t as = 0, acc_parity = 0;
    fetch(kb0);
    constexpr int kChunks = T::kCols / 16;
    uint32_t v[2][16];
    mbar_wait_inline(acc_full_bar(as), acc_parity, ctl, kCodeEpilogue);
    tcgen05_fence_after();
    tmem_ld_32x16(lane_addr, v[0]);
    int flip = 0;
    for (int kbs = kb0; kbs < kb1; kbs += T::kAhead, flip ^= 1) {
      float* stage_s = scales + flip * T::kAhead * kBT;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (pt + i * kReadThreads < T::kAhead * kBT) stage_s[pt + i * kReadThreads] = na[i] * nb[i];
      // past this barrier every warp is done with the other half, which the next round overwrites
      bar_sync(1, kReadThreads);
      fetch(kbs + T::kAhead);
#pragma unroll
      for (int i = 0; i < T::kAhead; ++i) {
        if (kbs + i < kb1) {
          const ulonglong2* s4 = reinterpret_cast<const ulonglong2*>(stage_s + i * kBT + tok0);
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            // one load in flight ahead of its use, across the stages too (as in k_gemm_fp8)
            uint32_t (&u)[16] = v[(i * kChunks + c) & 1];
            uint32_t (&w)[16] = v[(i * kChunks + c + 1) & 1];
            ulonglong2 sc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[j] = s4[c * 4 + j];
            tmem_ld_wait(u);
            if (c + 1 < kChunks) {
              tmem_ld_32x16(lane_addr + as * kBT + (c + 1) * 16, w);
            } else {
              tcgen05_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(acc_empty_bar(as));
              if (++as == T::kAcc) {
                as = 0;
                acc_parity ^= 1u;
              }
              if (kbs + i + 1 < kb1) {
                mbar_wait_inline(acc_full_bar(as), acc_parity, ctl, kCodeEpilogue);
                tcgen05_fence_after();
                tmem_ld_32x16(lane_addr + as * kBT, w);
              }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              acc[c * 8 + 2 * j] = fma_f32x2(pack_f32x2(u[4 * j], u[4 * j + 1]), sc[j].x, acc[c * 8 + 2 * j]);
              acc[c * 8 + 2 * j + 1] = fma_f32x2(pack_f32x2(u[4 * j + 2], u[4 * j + 3]), sc[j].y, acc[c * 8 + 2 * j + 1]);
            }
          }
        }
      }
    }
    if (p.split == 1) {
      if (n0 + row < p.n) {
#pragma unroll
        for (int j = 0; j < T::kCols / 2; ++j) {
          float lo, hi;
          unpack_f32x2(acc[j], lo, hi);
          __nv_bfloat16* dst = p.c + static_cast<int64_t>(tok0 + 2 * j) * p.ldc + n0 + row;
          if (tok0 + 2 * j < p.m) dst[0] = __float2bfloat16_rn(lo);
          if (tok0 + 2 * j + 1 < p.m) dst[p.ldc] = __float2bfloat16_rn(hi);
        }
      }
    } else {
      // The last product is complete, so the operand stages are free to hold the partial sums.
#pragma unroll
      for (int j = 0; j < T::kCols / 2; ++j) {
        float lo, hi;
        unpack_f32x2(acc[j], lo, hi);
        part[(tok0 + 2 * j) * kTileRows + row] = lo;
        part[(tok0 + 2 * j + 1) * kTileRows + row] = hi;
      }
    }
  }

  // ------------------------------------------------------------ join and teardown
  __syncwarp();
  if (p.split > 1) {
    cluster_arrive();
    cluster_wait();
    // rank r joins the tokens r, r + split, ..., a half of the CTA to every other one of them
    const int row = threadIdx.x & (kTileRows - 1);
    const int half = threadIdx.x >> 7;
    constexpr int kHalves = T::kThreads / kTileRows;
    if (half < kHalves && n0 + row < p.n) {
      for (int j = rank + half * p.split; j < p.m; j += kHalves * p.split) {
        const uint32_t addr = base + static_cast<uint32_t>(j * kTileRows + row) * 4u;
        float sum = 0.f;
        for (int r = 0; r < p.split; ++r) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(addr, r)) : "memory");
          sum += v;
        }
        p.c[static_cast<int64_t>(j) * p.ldc + n0 + row] = __float2bfloat16_rn(sum);
      }
    }
    __syncwarp();
    cluster_arrive();          // nobody leaves while its part is being read
    cluster_wait();
  }
  if (misc_gen[1] != 0u && warp == 0) {      // a wait ran out: let loads in flight land first
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc<1>(tmem_base, T::kTmemCols);
  }
}

// ============================================================== host side
template <typename Kern>
int configure(Kern kern, int smem, bool (&configured)[64]) {
  int dev = 0;
  LCG_CUDA_OK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    LCG_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return LCG_OK;
}

template <typename Kern, typename... Args>
int launch(Kern kern, unsigned grid, unsigned threads, int smem, unsigned cluster, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LCG_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, args...));
  count_launch();
  return LCG_OK;
}

struct Call {
  const void *a, *b;
  int64_t lda, ldb;
  Scales as, bs;
  void* c;
  int64_t ldc, m, n, k;
  int32_t* status;
  cudaStream_t stream;
};

int codes_map(CUtensorMap* map, const void* q, int64_t k, int64_t rows, int64_t ld, int box, const char* what) {
  return make_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q, k, rows, ld, box, what);
}

template <int kBN>
int run_many(const Call& q) {
  using T = Many<kBN>;
  CUtensorMap ma, mb, mc;
  if (int e = codes_map(&ma, q.a, q.k, q.m, q.lda, kTileRows, "a")) return e;
  if (int e = codes_map(&mb, q.b, q.k, q.n, q.ldb, T::kBRows, "b")) return e;
  if (int e = make_tensor_map(&mc, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, q.c, q.n, q.m, q.ldc, 32, "c")) return e;
  ManyParams p;
  std::memset(&p, 0, sizeof(p));
  p.a = q.as;
  p.b = q.bs;
  p.c = static_cast<__nv_bfloat16*>(q.c);
  p.ldc = q.ldc;
  p.m = static_cast<int32_t>(q.m);
  p.n = static_cast<int32_t>(q.n);
  p.k_blocks = static_cast<int32_t>((q.k + kBlock - 1) / kBlock);
  p.tiles_m = static_cast<int32_t>((q.m + 2 * kTileRows - 1) / (2 * kTileRows));
  p.tiles_n = static_cast<int32_t>((q.n + kBN - 1) / kBN);
  p.num_tiles = p.tiles_m * p.tiles_n;
  const int pairs = sm_count() / 2;
  p.group_m = pick_group_m(p.tiles_m, pairs);
  p.status = q.status;
  static bool configured[64] = {};
  if (int e = configure(k_gemm_fp8<kBN>, T::kSmemBytes, configured)) return e;
  const int groups = p.num_tiles < pairs ? p.num_tiles : pairs;
  return launch(k_gemm_fp8<kBN>, static_cast<unsigned>(2 * groups), kManyThreads, T::kSmemBytes, 2, q.stream, ma, mb, mc, p);
}

template <int kBT>
int run_few(const Call& q) {
  using T = Few<kBT>;
  CUtensorMap mw, mx;
  if (int e = codes_map(&mw, q.b, q.k, q.n, q.ldb, kTileRows, "b")) return e;
  if (int e = codes_map(&mx, q.a, q.k, q.m, q.lda, kBT, "a")) return e;
  FewParams p;
  std::memset(&p, 0, sizeof(p));
  p.a = q.as;
  p.b = q.bs;
  p.c = static_cast<__nv_bfloat16*>(q.c);
  p.ldc = q.ldc;
  p.m = static_cast<int32_t>(q.m);
  p.n = static_cast<int32_t>(q.n);
  p.k_blocks = static_cast<int32_t>((q.k + kBlock - 1) / kBlock);
  p.status = q.status;
  const int64_t tiles = (q.n + kTileRows - 1) / kTileRows;
  // Split K so that the GPU is filled: rounds of clusters times the K blocks of a CTA.  How many clusters of
  // a size run at once is asked once per device, for one CTA to an SM as the runtime counts them: the
  // GPU's parts are not multiples of each size (15 of 7, 22 of 6; 5120 x 17408 and one token, 40
  // clusters: 25.1 us with 7 in two rounds, 20.8 with 6 in one).
  static bool configured[64] = {};
  if (int e = configure(k_gemm_fp8_few<kBT>, T::kSmemBytes, configured)) return e;
  static std::atomic<int> at_once[64][kMaxSplit + 1];
  int dev = 0;
  LCG_CUDA_OK(cudaGetDevice(&dev));
  int split = 1;
  double best = 1e30;
  for (int s = 1; s <= kMaxSplit && s <= p.k_blocks; ++s) {
    int clusters = dev >= 0 && dev < 64 ? at_once[dev][s].load(std::memory_order_relaxed) : 0;
    if (clusters == 0) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(static_cast<unsigned>(s));
      cfg.blockDim = dim3(T::kThreads);
      cfg.dynamicSmemBytes = T::kSmemBytes;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = static_cast<unsigned>(s);
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      LCG_CUDA_OK(cudaOccupancyMaxActiveClusters(&clusters, k_gemm_fp8_few<kBT>, &cfg));
      if (clusters < 1) clusters = 1;
      if (dev >= 0 && dev < 64) at_once[dev][s].store(clusters, std::memory_order_relaxed);
    }
    clusters *= T::kCtas;
    const double rounds = static_cast<double>((tiles + clusters - 1) / clusters);
    const double cost = rounds * ((p.k_blocks + s - 1) / s) + 0.5 * s;      // a rank to add costs half a block's time
    if (cost < best) {
      best = cost;
      split = s;
    }
  }
  p.split = split;
  return launch(k_gemm_fp8_few<kBT>, static_cast<unsigned>(tiles * split), T::kThreads, T::kSmemBytes,
                static_cast<unsigned>(split), q.stream, mw, mx, p);
}

}  // namespace
}  // namespace lcg

using namespace lcg;

extern "C" int lcg_gemm_fp8(const void* a, int64_t lda, const float* a_scale, int64_t a_scale_row_stride,
                            int64_t a_scale_block_stride, const void* b, int64_t ldb, const float* b_scale,
                            int64_t b_scale_row_stride, int64_t b_scale_block_stride, void* c, int64_t ldc, int64_t M,
                            int64_t N, int64_t K, int32_t* status, void* stream) {
  if (!a || !a_scale || !b || !b_scale || !c) return fail(LCG_ERR_BAD_ARG, "NULL operand");
  // 2^30: tile origins and the rows past the edge stay inside 32 bits
  constexpr int64_t kMost = int64_t(1) << 30;
  if (M < 1 || N < 1 || K < 1 || M > kMost || N > kMost || K > kMost)
    return fail(LCG_ERR_UNSUPPORTED_SHAPE, "bad extents M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  const int64_t k16 = (K + 15) / 16 * 16;
  if (M == 1) lda = k16;      // the pitch of a single row is never used
  if (N == 1) ldb = k16;
  if (M == 1) ldc = (N + 7) / 8 * 8;
  if (lda < K || ldb < K || ldc < N) return fail(LCG_ERR_BAD_ARG, "leading dimension below extent");
  if (lda % 16 != 0 || ldb % 16 != 0 || ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u) != 0)
    return fail(LCG_ERR_MISALIGNED, "codes must be 16-byte aligned with a pitch of a multiple of 16 bytes");
  if (ldc % 8 != 0 || (reinterpret_cast<uintptr_t>(c) & 15u) != 0)
    return fail(LCG_ERR_MISALIGNED, "the output must be 16-byte aligned with a pitch of a multiple of 8 elements");
  if (!aligned(a_scale, 4) || !aligned(b_scale, 4) || !aligned(status, 4))
    return fail(LCG_ERR_MISALIGNED, "scales and status must be aligned to their type");
  if (((M + 255) / 256) * ((N + 127) / 128) > 0x7fffffffLL) return fail(LCG_ERR_UNSUPPORTED_SHAPE, "too many tiles");
  const Call q{a, b, lda, ldb, Scales{a_scale, a_scale_row_stride, a_scale_block_stride},
               Scales{b_scale, b_scale_row_stride, b_scale_block_stride}, c, ldc, M, N, K, status,
               static_cast<cudaStream_t>(stream)};
  // Up to 128 rows the weight-stationary form: 128 rows of 5120 x 17408 take 33 us in it and 35 in
  // pairs, of 34816 x 5120 43 and 48; 192 rows, two token tiles, take 48 and 35.
  if (M <= 16) return run_few<16>(q);
  if (M <= 32) return run_few<32>(q);
  if (M <= 64) return run_few<64>(q);
  if (M <= 128) return run_few<128>(q);
  // 256-wide tiles unless 128-wide ones fill the last wave so much better that their dearer operand
  // traffic is made up for: 1.1 of the time per column (4096 x 34816 x 5120: 730 us against 650).
  const int64_t pairs = sm_count() / 2;
  const int64_t rows = (M + 255) / 256;
  const double wide = 2.0 * static_cast<double>((rows * ((N + 255) / 256) + pairs - 1) / pairs);
  const double narrow = 1.1 * static_cast<double>((rows * ((N + 127) / 128) + pairs - 1) / pairs);
  return narrow < wide ? run_many<128>(q) : run_many<256>(q);
}
