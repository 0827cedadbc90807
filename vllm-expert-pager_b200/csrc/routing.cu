// Routing kernels: top-k experts of every token, the balance loss with the
// per-expert counts, and the gradient of the logits of both.
//
// With l a token's logits, m = max l, Z = sum exp(l - m), p_e = exp(l_e - m) / Z,
// the k largest logits S (equal logits: the lower expert first; -inf is never
// chosen) and n the tokens that count:
//
//   weights      w_j = p_{S_j}, or p_{S_j} / sum_i p_{S_i} (renormalised)
//   counts       c_e = number of choices of expert e
//   loss         L = E sum_e f_e P_e,  f_e = c_e / (n k),  P_e = sum_t p_te / n
//   gradient     dl_e = p_e (h_e - sum_u p_u h_u),  h_e = dL (E / n) f_e + dw_j [S_j = e]
//                (renormalised weights instead: dl_{S_j} += w_j (dw_j - sum_i w_i dw_i))
//
// One warp owns a token: the logits stay in registers (VPL a lane), maxima go
// through one redux instruction on order-preserving integer keys, and a token's
// reads are whole 16-byte vectors.  For the choice a lane's logits become integers
// that hold their order and their expert (see Choice), sorted in registers; each of
// the k steps then takes the largest first one of the lanes' runs.  Sums over tokens (P, c) are kept per lane
// over a warp's tokens (P's 32 bits hold 32 tokens at most, then 64 bits take them: over
// 2^26 tokens 32 bits lose 1e-4 of P), added over the CTA's warps in their order, and over
// the CTAs in theirs by a second small launch: no atomics on floats, so the loss does not
// depend on the order in which CTAs run.
//
// Few experts or tokens: bound by latency (one token of 256 experts 3.0 us).  Many:
// the loss of 65536 x 512 logits in 32 bits reads 134 MB in 37 us (40 with the sum over
// CTAs) at 57 % of the issue slots (exponentials and sums of 512 values a token), its
// gradient reads and writes 268 MB in 48 us, 5.6 TB/s (44 behind the forward pass, which
// leaves logits in L2).  16384 x 256 with the choice of 8 and the loss: 19 us forward, 75 %
// of the issue slots, 7.5 us backward.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace xp {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kSumCtas = 8;       // CTAs (one cluster) of the sum over CTAs
constexpr int kSumThreads = 1024;
constexpr int kFold = 32;         // tokens whose probabilities are summed in 32 bits
constexpr int kMaxCtas = 444;     // most CTAs of the forward kernel (3 for each of 148 SMs)

// Threads of a CTA of the forward kernel and CTAs on an SM, by the values per lane: what
// the registers allow without spills up to 256 experts, with at most 24 bytes of them up to
// 512.  Longer rows spill (up to 200 bytes at 1024 experts, 1.4 KB above, the backward
// kernel up to 1.5 KB above): 30000 x 1024 logits in 32 bits take 45 us for the loss, 269
// with the choice of 8 and 43 backward, 10000 x 4096 114, 449 and 128.
constexpr int forward_threads(int vpl) { return vpl <= 8 ? 512 : 256; }
constexpr int forward_blocks(int vpl) { return vpl <= 8 ? 2 : (vpl <= 16 ? 3 : (vpl <= 32 ? 2 : 1)); }
constexpr int kBackThreads = 256;  // the backward kernel's
constexpr int backward_blocks(int vpl) {
  return vpl <= 8 ? 4 : (vpl <= 16 ? 3 : (vpl <= 32 ? 2 : 1));
}
constexpr int most_experts(int vpl) { return 32 * vpl; }
constexpr int values_per_lane(int64_t E) {
  return E <= 64 ? 2 : (E <= 256 ? 8 : (E <= 512 ? 16 : (E <= 1024 ? 32 : 128)));
}

// A float's order as an unsigned integer; NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = x != x ? 0x7fffffffu : __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// A logit and its expert as one integer: larger logits above smaller ones, of equal
// ones the lower expert above; 0 is nothing, kOpen the least that can be chosen
// (above -inf).  16-bit logits need 16 bits for their order, so that one 32-bit
// maximum decides; 32-bit logits take 64 bits and two.
template <typename T>
struct Choice {
  using K = uint32_t;
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr K kOpen = (kHalf ? 0x0400u : 0x0080u) << 16;
  static __device__ __forceinline__ K make(float x, int e) {
    x = x + 0.0f;  // -0 equals 0
    uint32_t u = kHalf ? static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x))) << 16
                       : __float_as_uint(x);
    if (x != x) u = 0x7fff0000u;
    u ^= static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u;
    return (u & 0xffff0000u) | (0xffffu - e);
  }
  static __device__ __forceinline__ int expert(K k) { return 0xffff - static_cast<int>(k & 0xffff); }
  static __device__ __forceinline__ float logit(K k) {
    const uint32_t u = (k & 0x80000000u ? k ^ 0x80000000u : ~k) & 0xffff0000u;
    return kHalf ? __half2float(__ushort_as_half(static_cast<unsigned short>(u >> 16)))
                 : __uint_as_float(u);
  }
  static __device__ __forceinline__ K warp_max(K k) { return __reduce_max_sync(kFull, k); }
};

template <>
struct Choice<float> {
  using K = uint64_t;
  static constexpr K kOpen = 0x00800000ull << 32;
  static __device__ __forceinline__ K make(float x, int e) {
    return static_cast<K>(key_of(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(e));
  }
  static __device__ __forceinline__ int expert(K k) {
    return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k));
  }
  static __device__ __forceinline__ float logit(K k) {
    return of_key(static_cast<uint32_t>(k >> 32));
  }
  static __device__ __forceinline__ K warp_max(K k) {
    const uint32_t hi = static_cast<uint32_t>(k >> 32), top = __reduce_max_sync(kFull, hi);
    const unsigned who = __ballot_sync(kFull, hi == top);
    const uint32_t lo = static_cast<uint32_t>(k);
    // Equal logits in several lanes: the lower expert.
    const uint32_t low = (who & (who - 1)) ? __reduce_max_sync(kFull, hi == top ? lo : 0u)
                                           : __shfl_sync(kFull, lo, __ffs(who) - 1);
    return static_cast<K>(top) << 32 | low;
  }
};

// Sorts n values in descending order (Batcher's odd-even merges; unrolled whole).
template <int n, typename K>
__device__ __forceinline__ void sort_down(K (&k)[n]) {
#pragma unroll
  for (int p = 1; p < n; p *= 2)
#pragma unroll
    for (int d = p; d >= 1; d /= 2)
#pragma unroll
      for (int j = d % p; j + d < n; j += 2 * d)
#pragma unroll
        for (int i = 0; i < d; ++i)
          if (i + j + d < n && (i + j) / (2 * p) == (i + j + d) / (2 * p)) {
            const K u = k[i + j], w = k[i + j + d];
            k[i + j] = u > w ? u : w;
            k[i + j + d] = u > w ? w : u;
          }
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
  return x;
}

// exp(x) for x <= 0 by the hardware's power of two (2 steps of 2^-23, and 1.2 for each unit
// of x from the rounding of x log2 e); below 2^-126 it is 0.  With the product's rounding
// carried along (3 steps at any x) the loss of 65536 x 512 logits took 42.8 us, with expf
// 45.0, so 40.0: where x is large the probability is small, and the rounding of the
// difference x itself adds half as much.
__device__ __forceinline__ float exp_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
  return y;
}

template <typename T>
struct Pack;  // 16 bytes of logits
template <>
struct Pack<float> {
  static constexpr uint32_t kMinusInf = 0xff800000u;
  static constexpr int kN = 4;
  static __device__ __forceinline__ float at(const uint4 &q, int i) {
    return __uint_as_float((&q.x)[i]);
  }
};
template <>
struct Pack<__nv_bfloat16> {
  static constexpr uint32_t kMinusInf = 0xff80ff80u;
  static constexpr int kN = 8;
  static __device__ __forceinline__ float at(const uint4 &q, int i) {
    const uint32_t w = (&q.x)[i >> 1];
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
};
template <>
struct Pack<__half> {
  static constexpr uint32_t kMinusInf = 0xfc00fc00u;
  static constexpr int kN = 8;
  static __device__ __forceinline__ float at(const uint4 &q, int i) {
    const uint32_t w = (&q.x)[i >> 1];
    return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w >> 16 : w)));
  }
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ void narrow(float *p, float x) { *p = x; }
__device__ __forceinline__ void narrow(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void narrow(__half *p, float x) { *p = __float2half_rn(x); }

// How a row of E values lies in the lanes' registers: V neighbours a lane, so
// that a lane's values are whole 16-byte vectors where the row allows it.
template <typename T, int VPL, bool VEC>
struct Row {
  static constexpr int kV = !VEC ? 1 : (VPL < Pack<T>::kN ? VPL : Pack<T>::kN);
  static_assert(!VEC || kV == Pack<T>::kN, "vector rows hold whole 16-byte vectors");

  static __device__ __forceinline__ int expert(int i, int lane) {
    return ((i / kV) * 32 + lane) * kV + i % kV;
  }

  // Where an expert's sum stands in a row of sums, and such a row's length: skewed so that
  // neither the lanes' values of one register nor neighbouring experts share banks.
  static __device__ __forceinline__ int place(int e) { return kV > 1 ? e + e / kV : e; }
  static constexpr int kPlaces = 32 * VPL + (kV > 1 ? 32 * VPL / kV : 0);

  // A row in two steps, so that the next one can be on its way.  Places past the
  // row's end hold -inf from the start; no fetch touches them.
  struct Raw {
    uint4 q[VEC ? VPL / kV : 1];
    T x[VEC ? 1 : VPL];

    __device__ __forceinline__ Raw() {
      const uint32_t w = Pack<T>::kMinusInf;
      if constexpr (VEC) {
#pragma unroll
        for (int c = 0; c < VPL / kV; ++c) q[c] = make_uint4(w, w, w, w);
      } else {
#pragma unroll
        for (int c = 0; c < VPL; ++c) narrow(&x[c], -INFINITY);
      }
    }
  };

  static __device__ __forceinline__ void fetch(const T *row, int E, int lane, Raw &raw) {
#pragma unroll
    for (int c = 0; c < VPL / kV; ++c) {
      const int e = (c * 32 + lane) * kV;
      if (e >= E) continue;
      if constexpr (VEC)
        raw.q[c] = __ldg(reinterpret_cast<const uint4 *>(row + e));
      else
        raw.x[c] = row[e];
    }
  }

  static __device__ __forceinline__ void open(const Raw &raw, float *v) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      if constexpr (VEC)
        v[i] = Pack<T>::at(raw.q[i / kV], i % kV);
      else
        v[i] = widen(raw.x[i]);
    }
  }

  // The lane's values of a row of floats in shared memory (16-byte aligned; places
  // past its end are read too, as far as the row is padded).
  static __device__ __forceinline__ void gather(const float *row, int lane, float *v) {
#pragma unroll
    for (int i = 0; i < VPL; i += (VEC ? 4 : 1)) {
      const float *p = row + expert(i, lane);
      if constexpr (VEC) {
        const float4 q = *reinterpret_cast<const float4 *>(p);
        v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
      } else {
        v[i] = *p;
      }
    }
  }

  static __device__ __forceinline__ void store(T *row, int E, int lane, const float *v) {
#pragma unroll
    for (int c = 0; c < VPL / kV; ++c) {
      const int e = (c * 32 + lane) * kV;
      if (e >= E) continue;
      if constexpr (VEC) {
        __align__(16) T w[kV];
#pragma unroll
        for (int i = 0; i < kV; ++i) narrow(&w[i], v[c * kV + i]);
        *reinterpret_cast<uint4 *>(row + e) = *reinterpret_cast<const uint4 *>(w);
      } else {
        narrow(row + e, v[c]);
      }
    }
  }
};

// The largest value that is not NaN (-inf: there is none), and whether the row has
// anything to take a softmax of: a finite value, +inf or NaN.
template <int VPL>
__device__ __forceinline__ float row_max(const float *v, bool *live) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < VPL; ++i) m = fmaxf(m, v[i]);
  if (m != m) m = -INFINITY;  // all of this lane's
  m = of_key(__reduce_max_sync(kFull, key_of(m)));
  *live = true;
  if (m == -INFINITY) {  // rare: NaN alone, or nothing
    bool nan = false;
#pragma unroll
    for (int i = 0; i < VPL; ++i) nan |= v[i] != v[i];
    *live = __any_sync(kFull, nan);
  }
  return m;
}

struct ForwardArgs {
  const void *logits;
  int64_t T, stride;
  int E, topk, renormalize;
  const uint8_t *valid;
  float *weights;
  int32_t *ids;
  const void *given;  // ids chosen elsewhere (then weights and ids are not written)
  int given_bytes;
  int64_t *counts;  // [E]
  int64_t *tokens;  // the tokens that count (may be NULL)
  float *loss;      // NULL: no balance loss
  // One row per CTA, for the sum over CTAs: P (its 64 bits in two words), c, n.
  int32_t *part_p, *part_q, *part_c, *part_n;
};

// Writes the count of an expert; returns its share of n^2 k sum_e f_e P_e.
__device__ __forceinline__ double finish(const ForwardArgs &a, int e, double p, int c) {
  a.counts[e] = c;
  return c * p;
}

__device__ __forceinline__ float loss_of(const ForwardArgs &a, double s, int n) {
  return n == 0 ? 0.0f
                : static_cast<float>(a.E * s / (static_cast<double>(n) * n * a.topk));
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
  return x;
}

// kGiven: the ids were chosen elsewhere.
template <typename T, int VPL, bool VEC, bool kGiven>
__global__ void __launch_bounds__(forward_threads(VPL), forward_blocks(VPL))
    forward_kernel(const __grid_constant__ ForwardArgs a) {
  using R = Row<T, VPL, VEC>;
  // Rows too long for a second set of registers keep their sums of p in shared
  // memory, a row for each warp.
  constexpr bool kAccShared = VPL > 32;
  extern __shared__ __align__(16) unsigned char smem[];
  const int E = a.E, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool balance = a.loss != nullptr;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // The sums of p in 64 bits, a row for each warp (one row in all where the rows below
  // are); those in 32 bits; the counts.
  double *total = reinterpret_cast<double *>(smem);
  float *sum = reinterpret_cast<float *>(
      total + (!balance ? 0 : (kAccShared ? E : warps * R::kPlaces)));
  int *cnt = reinterpret_cast<int *>(sum + (balance && kAccShared ? warps * E : 0));
  __shared__ int tokens;
  __shared__ double loss_part[16];

  for (int e = threadIdx.x; e < E; e += blockDim.x) cnt[e] = 0;
  if (balance && kAccShared)
    for (int e = threadIdx.x; e < warps * E; e += blockDim.x) sum[e] = 0.0f;
  if (threadIdx.x == 0) tokens = 0;
  __syncthreads();

  float acc[kAccShared ? 1 : VPL];
  if constexpr (!kAccShared) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] = 0.0f;
  }
  // What the 32 bits hold goes to the 64: of a warp by itself, or (rows in shared memory)
  // of all warps together.
  auto fold = [&](bool folded) {  // before this time
    if constexpr (kAccShared) {
      __syncthreads();
      for (int e = threadIdx.x; e < E; e += blockDim.x) {
        double s = folded ? total[e] : 0.0;
        for (int w = 0; w < warps; ++w) s += sum[w * E + e], sum[w * E + e] = 0.0f;
        total[e] = s;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        double *at = total + warp * R::kPlaces + R::place(R::expert(i, lane));
        *at = folded ? *at + acc[i] : acc[i];
        acc[i] = 0.0f;
      }
    }
  };
  int mine = 0, rounds = 0;  // tokens of this warp that count; the CTA's rounds
  const int64_t step = static_cast<int64_t>(gridDim.x) * warps;
  int64_t t = static_cast<int64_t>(blockIdx.x) * warps + warp;
  // A token's row is fetched while the one before it is worked on, its flag one
  // token earlier still.
  auto counts = [&](int64_t u) { return u < a.T && (!a.valid || a.valid[u]); };
  auto row_of = [&](int64_t u) { return static_cast<const T *>(a.logits) + u * a.stride; };
  constexpr bool kAhead = VPL <= 32;
  typename R::Raw raw;
  bool live = counts(t), next_live = counts(t + step);
  if (live) R::fetch(row_of(t), E, lane, raw);
  // As many rounds for all of the CTA's warps, where they fold together.
  for (int64_t t0 = kAccShared ? t - warp : t; t0 < a.T; t0 += step, t += step) {
    if (kAccShared && balance && rounds++ % kFold == 0 && rounds > 1) fold(rounds > kFold + 1);
    float v[VPL];
    const bool here = live;
    if (here) R::open(raw, v);
    live = next_live;
    if (kAhead) {
      next_live = counts(t + 2 * step);
      if (live) R::fetch(row_of(t + step), E, lane, raw);
    }
    if (!here) {
      if (!kGiven && t < a.T && lane < a.topk) {
        a.weights[t * a.topk + lane] = 0.0f;
        a.ids[t * a.topk + lane] = -1;
      }
      if (!kAhead) {
        next_live = counts(t + 2 * step);
        if (live) R::fetch(row_of(t + step), E, lane, raw);
      }
      continue;
    }
    ++mine;
    int64_t given = -1;  // the first 32 of given ids, on their way during the softmax
    if (kGiven && lane < a.topk) given = load_id(a.given, a.given_bytes, t * a.topk + lane);
    float z = 0.0f;
    if (kGiven || balance || !a.renormalize) {
      bool any;
      const float m = row_max<VPL>(v, &any);
      if (any) {
        if constexpr (kAccShared) {
#pragma unroll
          for (int i = 0; i < VPL; ++i) z += exp_fast(v[i] - m);
          z = warp_sum(z);
          if (balance) {
            const float inv = 1.0f / z;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
              const int e = R::expert(i, lane);
              if (e < E) sum[warp * E + e] += exp_fast(v[i] - m) * inv;
            }
          }
        } else {
          float p[VPL];
#pragma unroll
          for (int i = 0; i < VPL; ++i) z += p[i] = exp_fast(v[i] - m);
          z = warp_sum(z);
          if (balance) {
            const float inv = 1.0f / z;
#pragma unroll
            for (int i = 0; i < VPL; ++i) acc[i] += p[i] * inv;
          }
        }
      }
    }
    if (!kAccShared && balance && mine % kFold == 0) fold(mine > kFold);
    // Where two rows do not fit the registers the next one is fetched at the end.
    if (!kAhead) next_live = counts(t + 2 * step);
    if constexpr (kGiven) {
      for (int j = lane; j < a.topk; j += 32) {
        if (j >= 32) given = load_id(a.given, a.given_bytes, t * a.topk + j);
        if (given >= 0 && given < E) atomicAdd(&cnt[given], 1);
      }
      if (!kAhead && live) R::fetch(row_of(t + step), E, lane, raw);
      continue;
    }
    // The lanes' choices: sorted where that is cheaper than to look through them
    // again after each step.  Unsorted 32-bit logits keep the 32 bits of their order
    // alone (a value's place gives its expert), half the registers.
    using C = Choice<T>;
    using K = typename C::K;
    constexpr bool kWide = sizeof(K) == 8;
    constexpr bool kSort = VPL <= 8 || (VPL <= 16 && !kWide);
    using Kept = typename std::conditional<kWide && !kSort, uint32_t, K>::type;
    Kept all[VPL] = {};
    K best = 0, mine_k = 0;
    auto choice = [&](int i) {
      if constexpr (kWide && !kSort)
        return all[i] == 0 ? K(0) : static_cast<K>(all[i]) << 32 |
                                        (0xffffffffu - static_cast<uint32_t>(R::expert(i, lane)));
      else
        return all[i];
    };
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = R::expert(i, lane);
      if constexpr (kWide && !kSort)
        all[i] = e < E ? key_of(v[i]) : 0;
      else
        all[i] = e < E ? C::make(v[i], e) : 0;
    }
    if constexpr (kSort) {
      sort_down<VPL>(all);
      best = all[0];
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i) best = best > choice(i) ? best : choice(i);
    }
    int found = 0;
    for (; found < a.topk; ++found) {
      const K top = C::warp_max(best);
      if (top < C::kOpen) break;
      if (lane == found) mine_k = top;
      if (best == top) {  // this lane's: on to its next one
        if constexpr (kSort) {
#pragma unroll
          for (int i = 0; i + 1 < VPL; ++i) all[i] = all[i + 1];
          all[VPL - 1] = 0;
          best = all[0];
        } else {
          best = 0;
#pragma unroll
          for (int i = 0; i < VPL; ++i) {
            if (choice(i) == top) all[i] = 0;
            best = best > choice(i) ? best : choice(i);
          }
        }
      }
    }
    const int my_id = lane < found ? C::expert(mine_k) : -1;
    const float l = C::logit(mine_k), top = __shfl_sync(kFull, l, 0);
    float w = lane < found ? exp_fast(l - top) : 0.0f;
    if (a.renormalize) z = warp_sum(w);
    if (lane < a.topk) {
      a.weights[t * a.topk + lane] = lane < found ? w / z : 0.0f;
      a.ids[t * a.topk + lane] = my_id;
    }
    if (lane < found) atomicAdd(&cnt[my_id], 1);
    if (!kAhead && live) R::fetch(row_of(t + step), E, lane, raw);
  }

  if (lane == 0 && mine) atomicAdd(&tokens, mine);
  if (balance) fold(kAccShared ? rounds > kFold : mine >= kFold);
  __syncthreads();
  double part = 0.0;
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    double p = 0.0;
    if (balance) {
      if constexpr (kAccShared) {
        p = total[e];
      } else {
        for (int w = 0; w < warps; ++w) p += total[w * R::kPlaces + R::place(e)];
      }
    }
    if (gridDim.x == 1) {
      part += finish(a, e, p, cnt[e]);
    } else {
      const int64_t at = static_cast<int64_t>(blockIdx.x) * E + e;
      a.part_c[at] = cnt[e];
      if (balance) {
        a.part_p[at] = __double2hiint(p);
        a.part_q[at] = __double2loint(p);
      }
    }
  }
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) a.part_n[blockIdx.x] = tokens;
    return;
  }
  if (threadIdx.x == 0 && a.tokens) *a.tokens = tokens;
  if (!balance) return;
  part = warp_sum(part);
  if (lane == 0) loss_part[warp] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < warps; ++w) s += loss_part[w];
    *a.loss = loss_of(a, s, tokens);
  }
}

// The sum over the forward kernel's CTAs: one cluster, each CTA a block of
// experts (threads along the experts, so that a warp reads whole lines), the
// loss through distributed shared memory.
__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    sum_kernel(const __grid_constant__ ForwardArgs a, int rows) {
  __shared__ double sp[kSumThreads];
  __shared__ int sc[kSumThreads];
  __shared__ double block_loss;
  __shared__ int tokens;
  cg::cluster_group cluster = cg::this_cluster();
  const int E = a.E, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool balance = a.loss != nullptr;
  if (tid == 0) tokens = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the forward kernel's end
  int n = tid < rows ? a.part_n[tid] : 0;
  n = __reduce_add_sync(kFull, n);
  if (lane == 0) atomicAdd(&tokens, n);
  __syncthreads();
  n = tokens;
  double loss = 0.0;
  constexpr int kCols = 32, kGroups = kSumThreads / kCols;
  constexpr int kEach = (kMaxCtas + kGroups - 1) / kGroups;
  for (int e0 = blockIdx.x * kCols; e0 < E; e0 += kSumCtas * kCols) {
    const int e = e0 + lane;
    int hi[kEach], lo[kEach], d[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {  // all of a thread's loads under way at once
      const int r = warp + i * kGroups;
      const bool in = e < E && r < rows;
      const int64_t at = static_cast<int64_t>(r) * E + e;
      d[i] = in ? a.part_c[at] : 0;
      hi[i] = in && balance ? a.part_p[at] : 0;
      lo[i] = in && balance ? a.part_q[at] : 0;
    }
    double p[2] = {0.0, 0.0};  // two chains of additions
    int c = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) c += d[i];
    if (balance)
#pragma unroll
      for (int i = 0; i < kEach; ++i) p[i & 1] += __hiloint2double(hi[i], lo[i]);
    __syncthreads();
    if (balance) sp[tid] = p[0] + p[1];
    sc[tid] = c;
    __syncthreads();
    if (warp == 0 && e < E) {
#pragma unroll 8
      for (int g = 1; g < kGroups; ++g) c += sc[g * kCols + lane];
      double q[4] = {0.0, 0.0, 0.0, 0.0};
      if (balance)
#pragma unroll 2
        for (int g = 0; g < kGroups; g += 4)
#pragma unroll
          for (int k = 0; k < 4; ++k) q[k] += sp[(g + k) * kCols + lane];
      loss += finish(a, e, (q[0] + q[1]) + (q[2] + q[3]), c);
    }
  }
  if (blockIdx.x == 0 && tid == 0 && a.tokens) *a.tokens = n;
  if (!balance) return;
  loss = warp_sum(loss);
  if (tid == 0) block_loss = loss;
  cluster.sync();
  if (blockIdx.x == 0 && tid == 0) {
    double s = 0.0;
    for (int b = 0; b < kSumCtas; ++b) s += *cluster.map_shared_rank(&block_loss, b);
    *a.loss = loss_of(a, s, n);
  }
  cluster.sync();  // the blocks' shared memory stays until it has been read
}

struct BackwardArgs {
  const void *logits;
  int64_t T, stride;
  int E, topk, renormalize;
  const uint8_t *valid;
  const int32_t *ids;         // the forward pass's choices and weights (with grad_weights)
  const float *weights;
  const float *grad_weights;  // NULL: no gradient through the weights
  const int64_t *counts;      // [E] (with grad_loss)
  const int64_t *tokens;
  const float *grad_loss;     // NULL: no gradient through the loss
  void *grad;                 // [T, E], contiguous
};

template <typename T, int VPL, bool VEC>
__global__ void __launch_bounds__(kBackThreads, backward_blocks(VPL))
    backward_kernel(const __grid_constant__ BackwardArgs a) {
  using R = Row<T, VPL, VEC>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int E = a.E, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kRow = 32 * VPL;  // a row and its padding
  float *h = reinterpret_cast<float *>(smem);  // dL/dp of the loss
  float *sel = h + kRow + warp * kRow;         // for each warp: the choices' part
  const bool balance = a.grad_loss != nullptr, choices = a.grad_weights != nullptr;
  {
    float s = 0.0f;
    if (balance) {
      const float n = static_cast<float>(a.tokens ? *a.tokens : a.T);
      if (n > 0.0f) s = *a.grad_loss * E / n / (n * a.topk);
    }
    for (int e = threadIdx.x; e < kRow; e += blockDim.x)
      h[e] = balance && e < E ? s * static_cast<float>(a.counts[e]) : 0.0f;
    if (choices)
      for (int e = lane; e < kRow; e += 32) sel[e] = 0.0f;
  }
  __syncthreads();
  const int64_t step = static_cast<int64_t>(gridDim.x) * warps;
  int64_t t = static_cast<int64_t>(blockIdx.x) * warps + warp;
  auto counts = [&](int64_t u) { return u < a.T && (!a.valid || a.valid[u]); };
  auto row_of = [&](int64_t u) { return static_cast<const T *>(a.logits) + u * a.stride; };
  constexpr bool kAhead = VPL <= 32;  // two rows fit the registers
  typename R::Raw raw;
  bool now = counts(t), next = counts(t + step);
  if (kAhead && now) R::fetch(row_of(t), E, lane, raw);
  for (; t < a.T; t += step) {
    float v[VPL];
    T *out = static_cast<T *>(a.grad) + t * E;
    bool live = now;
    if (!kAhead && live) R::fetch(row_of(t), E, lane, raw);
    if (live) R::open(raw, v);
    now = next;
    next = counts(t + 2 * step);
    int id = -1;
    float w = 0.0f, g = 0.0f;
    if (choices && lane < a.topk) {
      id = a.ids[t * a.topk + lane];
      w = a.weights[t * a.topk + lane];
      g = a.grad_weights[t * a.topk + lane];
    }
    if (kAhead && now) R::fetch(row_of(t + step), E, lane, raw);  // the next row, meanwhile
    float m = 0.0f;
    if (live) m = row_max<VPL>(v, &live);
    if (!live) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) v[i] = 0.0f;
      R::store(out, E, lane, v);
      continue;
    }
    float z = 0.0f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      v[i] = exp_fast(v[i] - m);
      z += v[i];
    }
    const float inv = 1.0f / warp_sum(z);
    float inner = 0.0f;  // sum_u p_u h_u
    float u[VPL <= 32 ? VPL : 1];  // h; rows too long for the registers read it twice
    if constexpr (VPL <= 32) {
      if (balance) {
        R::gather(h, lane, u);
      } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) u[i] = 0.0f;
      }
    }
    auto slope = [&](int i) {
      if constexpr (VPL <= 32)
        return u[i];
      else
        return h[R::expert(i, lane)];
    };
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      v[i] *= inv;
      inner += v[i] * slope(i);
    }
    if (balance) inner = warp_sum(inner);
    if (choices) {
      // A chosen probability is its weight, or proportional to it.
      const bool has = id >= 0 && id < E;
      float d = has ? w * g : 0.0f;
      const float both = warp_sum(d);
      if (a.renormalize)
        d -= has ? w * both : 0.0f;
      else
        inner += both;
      if (has) sel[id] = d;
      __syncwarp();
      if constexpr (VPL <= 32) {
        float c[VPL];
        R::gather(sel, lane, c);
#pragma unroll
        for (int i = 0; i < VPL; ++i) v[i] = v[i] * (u[i] - inner) + c[i];
      } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i)
          v[i] = v[i] * (slope(i) - inner) + sel[R::expert(i, lane)];
      }
      __syncwarp();
      if (has) sel[id] = 0.0f;
      __syncwarp();  // another lane may set the same place for the next token
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i) v[i] *= slope(i) - inner;
    }
    R::store(out, E, lane, v);
  }
}

// CTAs of the forward kernel.
int64_t forward_ctas(int64_t T, int64_t E) {
  const int vpl = values_per_lane(E);
  const int64_t warps = forward_threads(vpl) / 32, most = 148 * forward_blocks(vpl);
  const int64_t ctas = (T + warps - 1) / warps;
  return ctas < 1 ? 1 : (ctas < most ? ctas : most);
}

template <typename T, int VPL, bool VEC>
int launch_forward(const ForwardArgs &a, cudaStream_t s) {
  auto fn = a.given ? forward_kernel<T, VPL, VEC, true> : forward_kernel<T, VPL, VEC, false>;
  const int threads = forward_threads(VPL);
  const int64_t ctas = forward_ctas(a.T, a.E);
  auto need = [&](int64_t E, bool loss) {
    int64_t bytes = sizeof(int) * E;
    if (loss)
      bytes += VPL > 32 ? (sizeof(double) + sizeof(float) * (threads / 32)) * E
                        : sizeof(double) * (threads / 32) * Row<T, VPL, VEC>::kPlaces;
    return bytes;
  };
  const int64_t smem = need(a.E, a.loss != nullptr);
  int rc = allow_smem((const void *)fn, smem, need(most_experts(VPL), true));
  if (rc) return rc;
  fn<<<static_cast<unsigned>(ctas), threads, smem, s>>>(a);
  rc = launch_status();
  if (rc || ctas == 1) return rc;
  // The sum's launch overlaps the forward kernel's end (it waits for it itself).
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kSumCtas);
  cfg.blockDim = dim3(kSumThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t err = cudaLaunchKernelEx(&cfg, sum_kernel, a, static_cast<int>(ctas));
  return err == cudaSuccess ? launch_status() : static_cast<int>(err);
}

template <typename T, int VPL, bool VEC>
int launch_backward(const BackwardArgs &a, cudaStream_t s) {
  auto fn = backward_kernel<T, VPL, VEC>;
  const int threads = kBackThreads;
  const int64_t row = sizeof(float) * 32 * VPL, most = row * (1 + threads / 32);
  const int64_t smem = a.grad_weights ? most : row;
  int rc = allow_smem((const void *)fn, smem, most);
  if (rc) return rc;
  const int64_t want = (a.T + threads / 32 - 1) / (threads / 32);
  const int64_t ctas = 148 * backward_blocks(VPL);
  fn<<<static_cast<unsigned>(want < ctas ? want : ctas), threads, smem, s>>>(a);
  return launch_status();
}

// Values per lane by the number of experts; 16-byte vectors where base and
// stride allow them and the row ends on a vector.
template <typename T, typename Args, template <typename, int, bool> class Launch>
int dispatch(const Args &a, bool vec, cudaStream_t s) {
  constexpr int kN = Pack<T>::kN;
  const int E = a.E;
  vec = vec && E % kN == 0;
  switch (values_per_lane(E)) {
    case 2:
      return Launch<T, 2, false>::go(a, s);
    case 8:
      return vec ? Launch<T, 8, true>::go(a, s) : Launch<T, 8, false>::go(a, s);
    case 16:
      return vec ? Launch<T, 16, true>::go(a, s) : Launch<T, 16, false>::go(a, s);
    case 32:
      return vec ? Launch<T, 32, true>::go(a, s) : Launch<T, 32, false>::go(a, s);
    default:
      return vec ? Launch<T, 128, true>::go(a, s) : Launch<T, 128, false>::go(a, s);
  }
}

template <typename T, int VPL, bool VEC>
struct Forward {
  static int go(const ForwardArgs &a, cudaStream_t s) { return launch_forward<T, VPL, VEC>(a, s); }
};
template <typename T, int VPL, bool VEC>
struct Backward {
  static int go(const BackwardArgs &a, cudaStream_t s) {
    return launch_backward<T, VPL, VEC>(a, s);
  }
};

template <typename Args, template <typename, int, bool> class Launch>
int by_type(const Args &a, int dtype, const void *other, cudaStream_t s) {
  const int size = dtype == XP_F32 ? 4 : 2;
  const bool vec = aligned(a.logits, 16) && a.stride * size % 16 == 0 && aligned(other, 16);
  switch (dtype) {
    case XP_F32:
      return dispatch<float, Args, Launch>(a, vec, s);
    case XP_BF16:
      return dispatch<__nv_bfloat16, Args, Launch>(a, vec, s);
    default:
      return dispatch<__half, Args, Launch>(a, vec, s);
  }
}

// Sizes every entry point checks first.
int check_sizes(int dtype, int64_t T, int64_t E, int64_t stride, int64_t topk) {
  if (dtype != XP_F32 && dtype != XP_BF16 && dtype != XP_F16) return XP_EINVAL;
  if (T < 0 || E < 1 || topk < 1 || stride < 0) return XP_EINVAL;
  if (E > XP_MAX_EXPERTS || T > XP_MAX_TOKENS) return XP_ERANGE;
  // A count fits 32 bits.
  if (T > 0 && topk > INT32_MAX / T) return XP_ERANGE;
  return XP_OK;
}

int64_t scratch_need(int64_t T, int64_t E) {
  const int64_t ctas = forward_ctas(T, E);
  return ctas == 1 ? 0 : ctas * (E * 12 + 4);
}

int run_forward(ForwardArgs &a, int dtype, void *scratch, int64_t scratch_bytes, void *stream) {
  const int64_t ctas = forward_ctas(a.T, a.E);
  if (ctas > 1) {
    if (!scratch || !aligned(scratch, 4) || scratch_bytes < scratch_need(a.T, a.E))
      return XP_EINVAL;
    a.part_p = static_cast<int32_t *>(scratch);
    a.part_q = a.part_p + ctas * a.E;
    a.part_c = a.part_q + ctas * a.E;
    a.part_n = a.part_c + ctas * a.E;
  }
  return by_type<ForwardArgs, Forward>(a, dtype, nullptr, as_stream(stream));
}

}  // namespace
}  // namespace xp

using namespace xp;

extern "C" int64_t xp_route_scratch_bytes(int64_t T, int64_t E) {
  if (T < 0 || E < 1 || E > XP_MAX_EXPERTS || T > XP_MAX_TOKENS) return -1;
  return scratch_need(T, E);
}

extern "C" int xp_route(const void *logits, int dtype, int64_t T, int64_t E, int64_t stride,
                        const uint8_t *valid, int64_t topk, int renormalize, float *weights,
                        int32_t *ids, int64_t *counts, int64_t *tokens, float *loss,
                        void *scratch, int64_t scratch_bytes, void *stream) {
  int rc = check_sizes(dtype, T, E, stride, topk);
  if (rc) return rc;
  if (topk > E) return XP_EINVAL;
  if (topk > XP_MAX_TOPK) return XP_ERANGE;
  if (!counts || (T > 0 && (!logits || !weights || !ids))) return XP_EINVAL;
  ForwardArgs a{logits, T, stride, static_cast<int>(E), static_cast<int>(topk), renormalize, valid,
                weights, ids, nullptr, 4, counts, tokens, loss, nullptr, nullptr, nullptr, nullptr};
  return run_forward(a, dtype, scratch, scratch_bytes, stream);
}

extern "C" int xp_balance(const void *logits, int dtype, int64_t T, int64_t E, int64_t stride,
                          const uint8_t *valid, const void *ids, int ids_bytes, int64_t topk,
                          int64_t *counts, int64_t *tokens, float *loss, void *scratch,
                          int64_t scratch_bytes,
                          void *stream) {
  int rc = check_sizes(dtype, T, E, stride, topk);
  if (rc) return rc;
  if ((ids_bytes != 4 && ids_bytes != 8) || !counts || !loss || (T > 0 && (!logits || !ids)))
    return XP_EINVAL;
  // An empty batch has no ids to point at; the kernel then reads none.
  ForwardArgs a{logits, T, stride, static_cast<int>(E), static_cast<int>(topk), 0, valid,
                nullptr, nullptr, T > 0 ? ids : counts, ids_bytes, counts, tokens, loss, nullptr,
                nullptr, nullptr, nullptr};
  return run_forward(a, dtype, scratch, scratch_bytes, stream);
}

extern "C" int xp_route_backward(const void *logits, int dtype, int64_t T, int64_t E,
                                 int64_t stride, const uint8_t *valid, const int32_t *ids,
                                 const float *weights, int64_t topk, int renormalize,
                                 const float *grad_weights, const int64_t *counts, const int64_t *tokens,
                                 const float *grad_loss, void *grad, void *stream) {
  int rc = check_sizes(dtype, T, E, stride, topk);
  if (rc) return rc;
  if (grad_weights && topk > XP_MAX_TOPK) return XP_ERANGE;
  if (T == 0) return XP_OK;
  if (!logits || !grad || (grad_weights && (!ids || !weights)) || (grad_loss && !counts) ||
      (grad_loss && valid && !tokens))
    return XP_EINVAL;
  BackwardArgs a{logits, T, stride, static_cast<int>(E), static_cast<int>(topk), renormalize,
                 valid, ids, weights, grad_weights, counts, tokens,
                 grad_loss, grad};
  return by_type<BackwardArgs, Backward>(a, dtype, grad, as_stream(stream));
}
