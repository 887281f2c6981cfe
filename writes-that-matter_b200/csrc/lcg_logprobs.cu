// Log probabilities of given tokens, the entropy of each row, and its most likely tokens, in one
// pass over the logits.
//
// With m = max x, S = sum e^(x - m) and T = sum e^(x - m) (x - m) over a row (a masked value, -inf,
// adds nothing to either):  log p(token) = (x[token] - m) - ln S,  H = ln S - T / S.  The pass keeps a
// running m and rescales S and T when it grows.
//
// Alternatives.  A segment is what one warp reads in one load (32 vectors of 16 bytes).  The pass
// leaves each segment's maximum in shared memory.  Of any partition into runs of consecutive ids, the
// `top` best values (larger first, lower id first among equals) lie in the `top` best runs by the
// same order of their maxima: a run outside has `top` runs before it, each with a value that comes
// before all of its own.  So the `top` best segments are read again, and the values in them that are
// not below the worst of those segments' maxima, seldom more than two or three times `top`, are each
// ranked by counting.  Where they are more than 256 (long ties, rising rows), the same rule is applied
// once more, to the vectors of those segments: at most 32 x 8 values are then left, whatever the row
// holds.  (The second rule for every row, with its threshold searched by the whole CTA, took longer than
// the pass: 436 us against 199 for 4096 rows of 151936 bf16 without alternatives.)
//
// Many rows: 4096 x 151936 bf16 without alternatives run at HBM's rate (198 us of device time, up to 220
// among other calls; 190 at the copy rate; 66 instructions to a warp's 512 bytes, the exponential unit at 2/3 of its
// rate); 20 alternatives add 9300 instructions a row, which no longer fit beside the pass (238 and up to 270 us).  One
// row is bound by the latency of the selection.  A row is one CTA's, or a cluster's of up to eight when there
// are too few rows to fill the GPU; the CTAs' parts are joined through distributed shared memory in
// rank order, so the result does not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "lcg_common.h"
#include "lcg_ptx.cuh"

namespace lcg {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxCands = kMaxCluster * kMaxTop;      // = 32 vectors of 8 values
constexpr int64_t kMaxColumns = 1 << 20;     // a row's segment maxima then take at most 32 KiB
constexpr int kUnroll = 4;                   // 16-byte loads of a thread in flight

// -------------------------------------------------------------------- values
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  __device__ static void unpack(const uint4& q, float (&f)[4]) {
    f[0] = __uint_as_float(q.x), f[1] = __uint_as_float(q.y), f[2] = __uint_as_float(q.z), f[3] = __uint_as_float(q.w);
  }
  __device__ static float max(const uint4& q) {
    return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  __device__ static void unpack(const uint4& q, float (&f)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f[2 * t] = __uint_as_float(w[t] << 16);
      f[2 * t + 1] = __uint_as_float(w[t] & 0xffff0000u);
    }
  }
  __device__ static float max(const uint4& q) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8;
  __device__ static void unpack(const uint4& q, float (&f)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&q);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float2 v = __half22float2(h[t]);
      f[2 * t] = v.x;
      f[2 * t + 1] = v.y;
    }
  }
  __device__ static float max(const uint4& q) {
    const __half2* h = reinterpret_cast<const __half2*>(&q);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ uint32_t minus_inf_bits();
template <>
__device__ __forceinline__ uint32_t minus_inf_bits<float>() { return 0xff800000u; }
template <>
__device__ __forceinline__ uint32_t minus_inf_bits<__half>() { return 0xfc00u; }
template <>
__device__ __forceinline__ uint32_t minus_inf_bits<__nv_bfloat16>() { return 0xff80u; }

// Largest value of a warp, NaN left out.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {     // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  return pack_f32x2(__float_as_uint(lo), __float_as_uint(hi));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Order of the alternatives as whole numbers: larger is better, 0 and -0 alike, NaN with -inf; 0 is
// no value's.  The low bits that T's values leave alike are dropped: fewer bits to search.
template <typename T>
struct Key;
template <>
struct Key<float> { static constexpr int kLow = 0; };
template <>
struct Key<__nv_bfloat16> { static constexpr int kLow = 16; };
template <>
struct Key<__half> { static constexpr int kLow = 13; };
template <typename T>
__device__ __forceinline__ uint32_t order_key(float v) {
  v = v + 0.0f;
  if (v != v) v = -CUDART_INF_F;
  const uint32_t b = __float_as_uint(v);
  return ((b & 0x80000000u) ? ~b : b | 0x80000000u) >> Key<T>::kLow;
}
template <typename T>
__device__ __forceinline__ float key_value(uint32_t key) {
  constexpr int kLow = Key<T>::kLow;
  const uint32_t full = key << kLow;
  return __uint_as_float((full & 0x80000000u) ? full & 0x7fffffffu : ~(full | ((1u << kLow) - 1u)));
}

// A running maximum with the sums that go with it; T in units of ln 2, as the exponentials are taken
// to the base 2.
struct Sums {
  float m, s, t;
};
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// S and T of `a` seen from the maximum m >= a.m (the difference of two -inf is taken as 0).
__device__ __forceinline__ void rescale(Sums& a, float m) {
  const float d = a.m == m ? 0.f : (a.m - m) * kLog2e;
  const float f = ex2(d);
  a.t = a.s == 0.f ? 0.f : f == 0.f ? 0.f : f * fmaf(a.s, d, a.t);
  a.s = a.s * f;
  a.m = m;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  rescale(a, m);
  rescale(b, m);
  return Sums{m, a.s + b.s, a.t + b.t};
}

// ---------------------------------------------------------------- one row
// The first n <= 8 of `parts` joined as a tree, the same one every time; all lanes of a warp.
__device__ __forceinline__ Sums join_warps(const Sums* parts, int n) {
  const int lane = threadIdx.x & 7;      // every eight lanes the same
  Sums a = lane < n ? parts[lane] : Sums{-CUDART_INF_F, 0.f, 0.f};
#pragma unroll
  for (int o = 1; o < 8; o *= 2) {
    const Sums b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
                 __shfl_xor_sync(0xffffffffu, a.t, o)};
    a = (lane & o) ? join(b, a) : join(a, b);
  }
  return a;
}

template <typename T>
struct Row {
  static constexpr int kN = Vec<T>::kN;
  const T* x;          // the row
  const uint4* grid;   // the 16-byte grid that covers it
  int head;            // values of the first vector in front of the row
  int V;
  int full0, full1;    // vectors [full0, full1) lie inside the row
  __device__ Row(const T* row, int v) : x(row), V(v) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(row);
    head = static_cast<int>((p & 15u) / sizeof(T));
    grid = reinterpret_cast<const uint4*>(p & ~uintptr_t(15));
    full0 = head > 0 ? 1 : 0;
    full1 = (V + head) / kN;
  }
  __device__ int vectors() const { return (V + head + kN - 1) / kN; }
  // Vector i with -inf outside the row; only what lies inside is read.
  __device__ uint4 load(int i) const {
    if (i >= full0 && i < full1) return __ldg(grid + i);
    constexpr int kPerWord = 4 / static_cast<int>(sizeof(T));
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = 0;
#pragma unroll
      for (int e = 0; e < kPerWord; ++e) {
        const int id = i * kN - head + j * kPerWord + e;
        uint32_t bits = minus_inf_bits<T>();
        if (id >= 0 && id < V) {
          if constexpr (sizeof(T) == 4)
            bits = reinterpret_cast<const uint32_t*>(x)[id];
          else
            bits = reinterpret_cast<const unsigned short*>(x)[id];
        }
        w[j] |= bits << (16 * e);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// A value and its id as one number: larger is better, and the lower id among equal values.
__device__ __forceinline__ uint64_t entry(uint32_t key, uint32_t id) {
  return (static_cast<uint64_t>(key) << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ uint32_t entry_id(uint64_t e) { return 0xffffffffu - static_cast<uint32_t>(e); }
__device__ __forceinline__ uint32_t entry_key(uint64_t e) { return static_cast<uint32_t>(e >> 32); }
// How many of list[from, n) step by step of 2 * stride come before e; the list is padded with zeros to a
// multiple of 4 * stride.
template <int kStride>
__device__ __forceinline__ int place_of(const uint64_t* list, int n, int from, uint64_t e) {
  int place = 0;
  for (int i = from; i < n; i += 4 * kStride) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(list + i + 2 * j * kStride);
      place += (q.x > e) + (q.y > e);
    }
  }
  return place;
}

constexpr int kPick = 128;      // what select ranks by counting, two threads to an entry

struct SelectScratch {
  uint64_t pick[kPick];
  uint32_t tau[kWarps];
  uint32_t least;
  int found;
};

// The same by one warp, whatever the keys: the threshold is searched bit by bit from the top.
template <int kBits>
__device__ void search(const uint32_t* keys, int n, int k, uint32_t* out, SelectScratch& sc) {
  const int lane = threadIdx.x & 31;
  const uint32_t below = (1u << lane) - 1u;
  auto count = [&](uint32_t bound) {
    int c = 0;
#pragma unroll 4
    for (int i = lane; i < n; i += 32) c += keys[i] >= bound;
    return __reduce_add_sync(0xffffffffu, c);
  };
  uint32_t cut = 0;
  int ties = n;                        // how many keys equal to the cut are taken
  bool exact = false;
  for (int b = kBits - 1; b >= 0 && !exact; --b) {
    const uint32_t cand = cut | (1u << b);
    const int c = count(cand);
    if (c >= k) cut = cand;
    exact = c == k;
  }
  if (!exact) ties = k - count(cut + 1u);
  int at = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t key = i < n ? keys[i] : 0u;
    const uint32_t equal = __ballot_sync(0xffffffffu, i < n && key == cut);
    const bool in = i < n && (key > cut || (key == cut && __popc(equal & below) < ties));
    const uint32_t ins = __ballot_sync(0xffffffffu, in);
    if (in) out[at + __popc(ins & below)] = i;
    at += __popc(ins);
    ties = max(0, ties - __popc(equal));
  }
  if (lane == 0) sc.least = cut;
}

// The indexes of the k best of keys[0, n), equal ones by rising index, into out; k < n, k <= 32; the whole
// CTA.  Leaves the least of the chosen keys in sc.least.
//
// Every warp holds an eighth of the keys and gives the ceil(k / 8)-th best of its lanes' own maxima; the
// least of those is a bound that k keys reach, and few more do: some 50 for k = 20 on values in no
// order.  They are ranked by counting.  Where more than 128 reach it (ties), one warp searches.
template <int kBits>
__device__ void select(const uint32_t* keys, int n, int k, uint32_t* out, SelectScratch& sc) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sc.found = 0;
  uint32_t mine = 0;
  for (int i = lane * kWarps + warp; i < n; i += kThreads) mine = max(mine, keys[i]);
  for (int j = kWarps; ; j += kWarps) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, mine);
    if (j >= k) {
      if (lane == 0) sc.tau[warp] = top;
      break;
    }
    if (lane == __ffs(__ballot_sync(0xffffffffu, mine == top)) - 1) mine = 0;
  }
  __syncthreads();
  uint32_t bound = sc.tau[lane & (kWarps - 1)];
  bound = __reduce_min_sync(0xffffffffu, bound);
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + lane * kWarps + warp;
    const uint32_t key = i < n ? keys[i] : 0u;
    const bool in = i < n && key >= bound;
    const uint32_t ins = __ballot_sync(0xffffffffu, in);
    if (ins != 0u) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&sc.found, __popc(ins));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(ins & ((1u << lane) - 1u));
      if (in && at < kPick) sc.pick[at] = entry(key, i);
    }
  }
  __syncthreads();
  const int found = sc.found;
  if (found <= kPick) {
    if (tid >= found && tid < ((found + 7) & ~7)) sc.pick[tid] = 0;
    __syncthreads();
    if (warp * 16 < found) {
      const uint64_t e = tid / 2 < found ? sc.pick[tid / 2] : 0;
      int place = place_of<2>(sc.pick, found, 2 * (tid & 1), e);
      place += __shfl_xor_sync(0xffffffffu, place, 1);
      if (e != 0 && place < k && (tid & 1) == 0) {
        out[place] = entry_id(e);
        if (place == k - 1) sc.least = entry_key(e);
      }
    }
  } else if (warp == 0) {
    search<kBits>(keys, n, k, out, sc);
  }
  __syncthreads();
}

struct Params {
  const void* logits;
  const void* tokens;
  int64_t ld;
  int32_t V, top, token_bytes, cluster;
  float *logprob, *entropy, *top_logprobs;
  int64_t* top_ids;
};

static_assert(kMaxCluster <= kWarps && kMaxTop <= 32 && kMaxCands == kThreads, "a warp to a CTA's part, a lane to an entry");

template <typename T>
__global__ void __launch_bounds__(kThreads, 5)
k_token_logprobs(const __grid_constant__ Params p) {
  constexpr int kN = Vec<T>::kN;
  extern __shared__ __align__(16) uint32_t s_keys[];      // segment maxima, as keys
  __shared__ Sums s_sums[kWarps];
  __shared__ Sums s_part;                          // this CTA's sums, read by rank 0
  __shared__ __align__(16) uint64_t s_best[kMaxTop];      // this CTA's best, in order, then zeros; read by rank 0
  __shared__ uint32_t s_run[kMaxTop], s_vec[kMaxTop];     // chosen segments, chosen vectors of theirs
  __shared__ __align__(16) uint32_t s_vec_key[kMaxTop * 32];
  __shared__ __align__(16) uint64_t s_cand[kMaxCands];
  __shared__ __align__(16) SelectScratch s_select;
  __shared__ int s_count;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = p.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int64_t row = blockIdx.x / p.cluster;
  const Row<T> r(static_cast<const T*>(p.logits) + row * p.ld, p.V);
  const int nvec = r.vectors();
  const int nseg = (nvec + 31) / 32;
  const int seg0 = static_cast<int>(static_cast<int64_t>(nseg) * rank / p.cluster);
  const int seg1 = static_cast<int>(static_cast<int64_t>(nseg) * (rank + 1) / p.cluster);

  // the token's value is fetched now and used at the end
  float xt = CUDART_NAN_F;
  if (rank == 0 && tid == 0) {
    const int64_t t = p.token_bytes == 8 ? static_cast<const int64_t*>(p.tokens)[row]
                                         : static_cast<int64_t>(static_cast<const int32_t*>(p.tokens)[row]);
    if (t >= 0 && t < p.V) xt = to_float(r.x[t]);
  }

  // ------------------------------------------------------------------ the pass
  // m is the warp's: equal in its lanes.  S and T are each lane's own, two of each.
  float m = -CUDART_INF_F;
  uint64_t s2 = 0, t2 = 0;
  const uint64_t scale2 = pair(kLog2e, kLog2e);
  auto take = [&](const uint4 (&q)[kUnroll], int seg, int count) {
    float mx[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) mx[u] = u < count ? warp_max(Vec<T>::max(q[u])) : -CUDART_INF_F;
    if (p.top > 0 && lane < count) {          // a lane to a segment
      float v = mx[0];
#pragma unroll
      for (int u = 1; u < kUnroll; ++u) v = lane == u ? mx[u] : v;
      s_keys[seg + lane * kWarps - seg0] = order_key<T>(v);
    }
    float grown = m;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) grown = fmaxf(grown, mx[u]);
    if (grown > m) {
      float slo, shi, tlo, thi;
      unpack_f32x2(s2, slo, shi);
      unpack_f32x2(t2, tlo, thi);
      Sums lo{m, slo, tlo}, hi{m, shi, thi};
      rescale(lo, grown);
      rescale(hi, grown);
      s2 = pair(lo.s, hi.s);
      t2 = pair(lo.t, hi.t);
      m = grown;
    }
    const float minus_m = m == -CUDART_INF_F ? 0.f : -m;
    const uint64_t shift2 = pair(minus_m, minus_m);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (u < count) {
        float f[kN];
        Vec<T>::unpack(q[u], f);
#pragma unroll
        for (int e = 0; e < kN; e += 2) {
          float lo, hi;
          unpack_f32x2(mul2(add2(pair(f[e], f[e + 1]), shift2), scale2), lo, hi);
          // a masked value's difference is -inf, which must not meet the 0 of its exponential
          lo = max_nan(lo, -200.f);
          hi = max_nan(hi, -200.f);
          const uint64_t e2 = pair(ex2(lo), ex2(hi));
          s2 = add2(s2, e2);
          t2 = fma_f32x2(e2, pair(lo, hi), t2);
        }
      }
    }
  };
  {
    const int inner0 = (r.full0 + 31) / 32, inner1 = r.full1 / 32;    // segments that lie inside the row
    int seg = seg0 + warp;
    for (; seg + (kUnroll - 1) * kWarps < seg1; seg += kUnroll * kWarps) {
      uint4 q[kUnroll];
      if (seg >= inner0 && seg + (kUnroll - 1) * kWarps < inner1) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) q[u] = __ldg(r.grid + (seg + u * kWarps) * 32 + lane);
      } else {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) q[u] = r.load((seg + u * kWarps) * 32 + lane);
      }
      take(q, seg, kUnroll);
    }
    if (seg < seg1) {
      uint4 q[kUnroll];
      const int count = (seg1 - seg + kWarps - 1) / kWarps;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (u < count) q[u] = r.load((seg + u * kWarps) * 32 + lane);
      take(q, seg, count);
    }
  }
  // Lanes, warps, CTAs: always in the same order.
  {
    float slo, shi, tlo, thi;
    unpack_f32x2(s2, slo, shi);
    unpack_f32x2(t2, tlo, thi);
    float s = slo + shi, t = tlo + thi;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    if (lane == 0) s_sums[warp] = Sums{m, s, t};
  }
  if (tid == 0) s_count = 0;
  if (tid < kMaxTop) s_best[tid] = 0;
  __syncthreads();
  if (warp == kWarps - 1) {
    const Sums a = join_warps(s_sums, kWarps);
    if (lane == 0) s_part = a;
  }

  // -------------------------------------------------------------- alternatives
  const int first = max(0, seg0 * 32 * kN - r.head);
  const int last = min(r.V, seg1 * 32 * kN - r.head);
  const int want = min(p.top, last - first);        // of this CTA's part of the row
  if (want > 0) {
    const int n = seg1 - seg0;
    const int runs = min(want, n);
    constexpr int kBits = 32 - Key<T>::kLow;
    if (n > want) {
      select<kBits>(s_keys, n, want, s_run, s_select);
    } else {
      if (tid < n) s_run[tid] = tid;
      __syncthreads();
    }
    // Candidates: value e of the vector at id0 for each bit e of `in`.  They are few, so each takes its place by
    // itself and is read again (from L1) rather than picked out of registers.
    auto append = [&](uint32_t in, int id0) {
      while (in != 0u) {
        const int id = id0 + __ffs(in) - 1;
        in &= in - 1u;
        const int at = atomicAdd(&s_count, 1);
        if (at < kMaxCands) s_cand[at] = entry(order_key<T>(to_float(r.x[id])), static_cast<uint32_t>(id));
      }
    };
    // No value below the least of the chosen maxima is among the best: there are `want` that are not.
    // (Where all segments are chosen there is no such bound.)
    const uint32_t least = n > want ? s_select.least : 0u;
    const float least_value = least == 0u ? -CUDART_INF_F : key_value<T>(least);
    auto id_of = [&](int run, int e) { return ((seg0 + static_cast<int>(s_run[run >> 5])) * 32 + (run & 31)) * kN - r.head + e; };
    if (n > want || last - first <= kMaxCands) {
      uint4 q[kMaxTop / kWarps];
#pragma unroll
      for (int u = 0; u < kMaxTop / kWarps; ++u) {
        const int j = warp + u * kWarps;
        const int v = j < runs ? (seg0 + static_cast<int>(s_run[j])) * 32 + lane : nvec;
        q[u] = v < nvec ? r.load(v) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < kMaxTop / kWarps; ++u) {
        const int j = warp + u * kWarps;
        if (j >= runs) break;
        const int id0 = id_of(j * 32 + lane, 0);
        float f[kN];
        Vec<T>::unpack(q[u], f);
        uint32_t in = 0;
        if (least_value > -CUDART_INF_F) {          // few lanes hold a candidate: values compare faster than keys
#pragma unroll
          for (int e = 0; e < kN; ++e)
            if (f[e] >= least_value) in |= 1u << e;
        } else {                                     // a NaN ranks with -inf
#pragma unroll
          for (int e = 0; e < kN; ++e)
            if (order_key<T>(f[e]) >= least) in |= 1u << e;
        }
        if (id0 < 0) in &= 0xffffffffu << -id0;                     // the row's own values only
        if (id0 + kN > r.V) in &= id0 < r.V ? (1u << (r.V - id0)) - 1u : 0u;
        append(in, id0);
      }
    } else if (tid == 0) {
      s_count = kMaxCands + 1;
    }
    __syncthreads();
    if (s_count > kMaxCands) {
      // Too many: the best vectors of these segments, each by its best value (0 where it holds none of the
      // row), the segments in rising order so that a lower index is a lower id.
      uint32_t run = 0;
      int place = 0;
      if (tid < runs) {
        run = s_run[tid];
        for (int j = 0; j < runs; ++j) place += s_run[j] < run;
      }
      __syncthreads();
      if (tid < runs) s_run[place] = run;
      __syncthreads();
      const int nv = runs * 32;
      for (int i = tid; i < nv; i += kThreads) {
        const int id0 = id_of(i, 0);
        const int v = (id0 + r.head) / kN;
        uint32_t key = 0;
        if (v < nvec) {
          float f[kN];
          Vec<T>::unpack(r.load(v), f);
#pragma unroll
          for (int e = 0; e < kN; ++e)
            if (id0 + e >= 0 && id0 + e < r.V) key = max(key, order_key<T>(f[e]));
        }
        s_vec_key[i] = key;
      }
      if (tid == 0) s_count = 0;
      __syncthreads();
      const int vecs = min(want, nv);
      if (nv > want) {
        select<kBits>(s_vec_key, nv, want, s_vec, s_select);
      } else {
        if (tid < nv) s_vec[tid] = tid;
        __syncthreads();
      }
      const uint32_t least_of_vecs = nv > want ? s_select.least : 0u;
      const int at = tid / kN;
      const int id = at < vecs ? id_of(static_cast<int>(s_vec[at]), tid % kN) : -1;
      const uint32_t key = id >= 0 && id < r.V ? order_key<T>(to_float(r.x[id])) : 0u;
      append(key != 0u && key >= least_of_vecs ? 1u : 0u, id);
      __syncthreads();
    }
    const int cands = s_count;
    if (tid >= cands && tid < ((cands + 7) & ~7)) s_cand[tid] = 0;
    __syncthreads();
    if (tid < cands) {
      const uint64_t e = s_cand[tid];
      const int place = place_of<2>(s_cand, cands, 0, e) + place_of<2>(s_cand, cands, 2, e);
      if (place < want) s_best[place] = e;
    }
  }
  __syncthreads();

  // ---------------------------------------------------------------- the row
  Sums a = s_part;
  if (p.cluster > 1) {
    cluster_arrive();
    cluster_wait();
    if (rank == 0) {
      // A warp to each CTA's part: its sums and its best, all at once.
      auto remote = [&](const void* local) {
        uint32_t v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];"
                     : "=r"(v) : "r"(mapa_shared(smem_u32(local), static_cast<uint32_t>(warp))) : "memory");
        return v;
      };
      uint64_t e = 0;
      if (warp < p.cluster) {
        if (lane < 3) reinterpret_cast<uint32_t*>(&s_sums[warp])[lane] = remote(reinterpret_cast<uint32_t*>(&s_part) + lane);
        if (lane < p.top) {
          const uint32_t* b = reinterpret_cast<const uint32_t*>(s_best + lane);
          e = (static_cast<uint64_t>(remote(b + 1)) << 32) | remote(b);
        }
        // each part's last bounds the row's last from below
        if (lane == p.top - 1) s_select.pick[warp] = e;
      }
      if (tid == 0) s_count = 0;
      __syncthreads();
      a = join_warps(s_sums, p.cluster);
      if (p.top > 0) {
        uint64_t bound = 1;
        for (int c = 0; c < p.cluster; ++c) bound = max(bound, s_select.pick[c]);
        const bool in = e >= bound;
        const uint32_t ins = __ballot_sync(0xffffffffu, in);
        int at = 0;
        if (lane == 0 && ins != 0u) at = atomicAdd(&s_count, __popc(ins));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(ins & ((1u << lane) - 1u));
        if (in) s_cand[at] = e;
        __syncthreads();
        const int total = s_count;
        if (tid >= total && tid < ((total + 7) & ~7)) s_cand[tid] = 0;
        __syncthreads();
        if (tid < total) {
          const uint64_t mine = s_cand[tid];
          const int place = place_of<2>(s_cand, total, 0, mine) + place_of<2>(s_cand, total, 2, mine);
          if (place < p.top) s_best[place] = mine;
        }
        __syncthreads();
      }
    }
  }
  if (rank == 0) {
    // a row that is all -inf has S = 0 and m = -inf: no distribution, NaN throughout
    const float lse = a.m == -CUDART_INF_F ? CUDART_NAN_F : logf(a.s);
    if (tid == 0) {
      p.logprob[row] = (xt - a.m) - lse;
      p.entropy[row] = lse - a.t / a.s * kLn2;
    }
    if (tid < p.top) {
      const uint64_t e = s_best[tid];
      p.top_ids[row * p.top + tid] = entry_id(e);
      p.top_logprobs[row * p.top + tid] = (key_value<T>(entry_key(e)) - a.m) - lse;
    }
  }
  __syncwarp();              // the cluster barriers are for whole warps
  if (p.cluster > 1) {       // nobody leaves while its part is being read
    cluster_arrive();
    cluster_wait();
  }
}

template <typename T>
int run(const Params& p, int64_t M, cudaStream_t stream) {
  const int64_t row_vectors = (p.V + 2 * Vec<T>::kN - 2) / Vec<T>::kN + 1;       // with any alignment
  const int64_t segments = (row_vectors + 31) / 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(M * p.cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = p.top > 0 ? static_cast<size_t>(segments / p.cluster + 1) * 4 : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LCG_CUDA_OK(cudaLaunchKernelEx(&cfg, k_token_logprobs<T>, p));
  count_launch();
  return LCG_OK;
}

}  // namespace
}  // namespace lcg

using namespace lcg;

extern "C" int lcg_token_logprobs(const void* logits, int dtype, int64_t M, int64_t V, int64_t ld, const void* tokens,
                                  int token_bytes, int top, float* logprob, float* entropy, float* top_logprobs,
                                  int64_t* top_ids, void* stream) {
  if (!logits || !tokens || !logprob || !entropy || (top > 0 && (!top_logprobs || !top_ids)))
    return fail(LCG_ERR_BAD_ARG, "NULL argument");
  if (M < 1 || M > 0x7fffffffLL / kMaxCluster || V < 1 || V > kMaxColumns)
    return fail(LCG_ERR_UNSUPPORTED_SHAPE, "needs 1 <= V <= %lld, got M=%lld V=%lld", (long long)kMaxColumns,
                (long long)M, (long long)V);
  if (ld < V && M > 1) return fail(LCG_ERR_BAD_ARG, "leading dimension below extent");
  if (token_bytes != 4 && token_bytes != 8) return fail(LCG_ERR_BAD_ARG, "token ids must have 4 or 8 bytes");
  if (top < 0 || top > kMaxTop || top > V)
    return fail(LCG_ERR_BAD_ARG, "top must be between 0 and min(%d, V), got %d", kMaxTop, top);
  if (dtype != LCG_DTYPE_BF16 && dtype != LCG_DTYPE_FP16 && dtype != LCG_DTYPE_FP32)
    return fail(LCG_ERR_BAD_ARG, "unknown dtype %d", dtype);
  const unsigned width = dtype == LCG_DTYPE_FP32 ? 4 : 2;
  if (!aligned(logits, width) || !aligned(tokens, token_bytes) || !aligned(logprob, 4) || !aligned(entropy, 4) ||
      (top > 0 && (!aligned(top_logprobs, 4) || !aligned(top_ids, 8))))
    return fail(LCG_ERR_MISALIGNED, "logits, tokens and results must be aligned to their types");
  Params p;
  p.logits = logits;
  p.tokens = tokens;
  p.ld = ld;
  p.V = static_cast<int32_t>(V);
  p.top = top;
  p.token_bytes = token_bytes;
  p.logprob = logprob;
  p.entropy = entropy;
  p.top_logprobs = top_logprobs;
  p.top_ids = top_ids;
  // CTAs to a row, each with at least 16 segments (two loads a warp).
  const int64_t segments = (V * static_cast<int64_t>(width) + 511) / 512;
  // The cluster grows while the grid has fewer than two CTAs an SM, so it ends below four.  Past that the
  // join and the choice in every CTA cost more than the shorter pass saves.  Against growing while there
  // are fewer than four, at 151936 bf16 with 20 alternatives: 100 rows 19.5 us against 27.8, 200 rows
  // 27.4 / 36.1, 500 rows 43.9 / 57.8; 333 x 50257 fp32 22.0 / 23.1.  Fewer than one: 100 rows 22.1,
  // 200 rows 31.5.
  p.cluster = 1;
  while (p.cluster < kMaxCluster && M * p.cluster < 2 * sm_count() && segments / (2 * p.cluster) >= 16) p.cluster *= 2;
  auto st = static_cast<cudaStream_t>(stream);
  if (dtype == LCG_DTYPE_BF16) return run<__nv_bfloat16>(p, M, st);
  if (dtype == LCG_DTYPE_FP16) return run<__half>(p, M, st);
  return run<float>(p, M, st);
}
