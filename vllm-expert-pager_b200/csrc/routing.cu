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
// reads are whole 16-byte vectors.  Sums over tokens (P, c) are kept per lane
// over a warp's tokens, added over the CTA's warps in their order, and over the
// CTAs in theirs by a second small launch: no atomics on floats, so the loss does
// not depend on the order in which CTAs run.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace xp {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;
// Key of -inf (see key_of): entries at or below it cannot be chosen.
constexpr uint32_t kKeyNegInf = 0x007fffffu;
constexpr int kSumCtas = 8;       // CTAs (one cluster) of the sum over CTAs
constexpr int kSumThreads = 1024;
constexpr int kMaxCtas = 444;     // most CTAs of the forward kernel (3 for each of 148 SMs)

// Threads of a CTA of the forward kernel and CTAs on an SM, by the values per lane:
// what the registers allow without spills.
constexpr int forward_threads(int vpl) { return vpl <= 8 ? 512 : 256; }
constexpr int forward_blocks(int vpl) { return vpl <= 8 ? 2 : (vpl <= 16 ? 3 : (vpl <= 32 ? 2 : 1)); }
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

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
  return x;
}

template <typename T>
struct Pack;  // 16 bytes of logits
template <>
struct Pack<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ float at(const uint4 &q, int i) {
    return __uint_as_float((&q.x)[i]);
  }
};
template <>
struct Pack<__nv_bfloat16> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ float at(const uint4 &q, int i) {
    const uint32_t w = (&q.x)[i >> 1];
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  }
};
template <>
struct Pack<__half> {
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

  // A row in two steps, so that the next one can be on its way.
  struct Raw {
    uint4 q[VEC ? VPL / kV : 1];
    T x[VEC ? 1 : VPL];
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

  static __device__ __forceinline__ void open(const Raw &raw, int E, int lane, float *v) {
#pragma unroll
    for (int c = 0; c < VPL / kV; ++c) {
      const bool in = (c * 32 + lane) * kV < E;
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        if constexpr (VEC)
          v[c * kV + i] = in ? Pack<T>::at(raw.q[c], i) : -INFINITY;
        else
          v[c] = in ? widen(raw.x[c]) : -INFINITY;
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
  const void *logits;  // NULL: counts of given ids only
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
  // One row per CTA, for the sum over CTAs: P, c, n.
  float *part_p;
  int32_t *part_c, *part_n;
};

// The loss and the outputs from totals of one block of experts; returns the
// block's share of sum_e f_e P_e.
__device__ __forceinline__ float finish(const ForwardArgs &a, int e, float p, int c, int n) {
  a.counts[e] = c;
  if (n == 0) return 0.0f;
  return (static_cast<float>(c) / (static_cast<float>(n) * a.topk)) * (p / n);
}

template <typename T, int VPL, bool VEC>
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
  int *cnt = reinterpret_cast<int *>(smem);               // [E]
  float *sum = reinterpret_cast<float *>(smem) + E;       // [E], or [warps][E]
  __shared__ int tokens;
  __shared__ float loss_part[16];

  for (int e = threadIdx.x; e < E; e += blockDim.x) cnt[e] = 0;
  if (balance) {
    const int rows = kAccShared ? warps : 1;
    for (int e = threadIdx.x; e < rows * E; e += blockDim.x) sum[e] = 0.0f;
  }
  if (threadIdx.x == 0) tokens = 0;
  __syncthreads();

  float acc[kAccShared ? 1 : VPL];
  if constexpr (!kAccShared) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] = 0.0f;
  }
  int mine = 0;  // tokens of this warp that count
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
  for (; t < a.T; t += step) {
    float v[VPL];
    const bool here = live;
    if (here) R::open(raw, E, lane, v);
    live = next_live;
    if (kAhead) {
      next_live = counts(t + 2 * step);
      if (live) R::fetch(row_of(t + step), E, lane, raw);
    }
    if (!here) {
      if (!a.given && lane < a.topk) {
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
    float z = 0.0f;
    if (balance || (!a.given && !a.renormalize)) {
      bool any;
      const float m = row_max<VPL>(v, &any);
      if (any) {
        if constexpr (kAccShared) {
#pragma unroll
          for (int i = 0; i < VPL; ++i) z += __expf(v[i] - m);
          z = warp_sum(z);
          if (balance) {
            const float inv = 1.0f / z;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
              const int e = R::expert(i, lane);
              if (e < E) sum[warp * E + e] += __expf(v[i] - m) * inv;
            }
          }
        } else {
          float p[VPL];
#pragma unroll
          for (int i = 0; i < VPL; ++i) z += p[i] = __expf(v[i] - m);
          z = warp_sum(z);
          if (balance) {
            const float inv = 1.0f / z;
#pragma unroll
            for (int i = 0; i < VPL; ++i) acc[i] += p[i] * inv;
          }
        }
      }
    }
    if (!kAhead) {
      // (Two rows do not fit the registers; the values are read again below.)
      next_live = counts(t + 2 * step);
    }
    if (a.given) {
      for (int j = lane; j < a.topk; j += 32) {
        const int64_t id = load_id(a.given, a.given_bytes, t * a.topk + j);
        if (id >= 0 && id < E) atomicAdd(&cnt[id], 1);
      }
      if (!kAhead && live) R::fetch(row_of(t + step), E, lane, raw);
      continue;
    }
    uint32_t key[VPL], best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      key[i] = key_of(v[i]);
      if (key[i] > best) best = key[i], at = R::expert(i, lane);
    }
    uint32_t my_key = 0;
    int my_id = -1, found = 0;
    for (; found < a.topk; ++found) {
      const uint32_t top = __reduce_max_sync(kFull, best);
      if (top <= kKeyNegInf) break;
      const unsigned claim = best == top ? static_cast<unsigned>(at) : kFull;
      const unsigned who = __ballot_sync(kFull, best == top);
      const unsigned win = (who & (who - 1)) ? __reduce_min_sync(kFull, claim)
                                             : __shfl_sync(kFull, claim, __ffs(who) - 1);
      if (lane == found) my_key = top, my_id = static_cast<int>(win);
      if (claim == win) {  // the owner takes it out and looks for its next one
        best = 0;
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
          const int e = R::expert(i, lane);
          if (e == static_cast<int>(win)) key[i] = 0;
          if (key[i] > best) best = key[i], at = e;
        }
      }
    }
    const float l = of_key(my_key), top = __shfl_sync(kFull, l, 0);
    float w = lane < found ? __expf(l - top) : 0.0f;
    if (a.renormalize) z = warp_sum(w);
    if (lane < a.topk) {
      a.weights[t * a.topk + lane] = lane < found ? w / z : 0.0f;
      a.ids[t * a.topk + lane] = my_id;
    }
    if (lane < found) atomicAdd(&cnt[my_id], 1);
    if (!kAhead && live) R::fetch(row_of(t + step), E, lane, raw);
  }

  if (lane == 0 && mine) atomicAdd(&tokens, mine);
  if (balance && !kAccShared) {
    for (int w = 0; w < warps; ++w) {
      __syncthreads();
      if (w == warp) {
#pragma unroll
        for (int i = 0; i < (kAccShared ? 1 : VPL); ++i) {
          const int e = R::expert(i, lane);
          if (e < E) sum[e] += acc[i];
        }
      }
    }
  }
  __syncthreads();
  float part = 0.0f;
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    float p = 0.0f;
    if (balance)
      for (int w = 0; w < (kAccShared ? warps : 1); ++w) p += sum[w * E + e];
    if (gridDim.x == 1) {
      part += finish(a, e, p, cnt[e], tokens);
    } else {
      a.part_c[static_cast<int64_t>(blockIdx.x) * E + e] = cnt[e];
      if (balance) a.part_p[static_cast<int64_t>(blockIdx.x) * E + e] = p;
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
    float s = 0.0f;
    for (int w = 0; w < warps; ++w) s += loss_part[w];
    *a.loss = s * E;
  }
}

// The sum over the forward kernel's CTAs: one cluster, each CTA a block of
// experts (threads along the experts, so that a warp reads whole lines), the
// loss through distributed shared memory.
__global__ void __cluster_dims__(kSumCtas, 1, 1) __launch_bounds__(kSumThreads)
    sum_kernel(const __grid_constant__ ForwardArgs a, int rows) {
  __shared__ float sp[kSumThreads];
  __shared__ int sc[kSumThreads];
  __shared__ float block_loss;
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
  float loss = 0.0f;
  constexpr int kCols = 32, kGroups = kSumThreads / kCols;
  constexpr int kEach = (kMaxCtas + kGroups - 1) / kGroups;
  for (int e0 = blockIdx.x * kCols; e0 < E; e0 += kSumCtas * kCols) {
    const int e = e0 + lane;
    float q[kEach];
    int d[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {  // all of a thread's loads under way at once
      const int r = warp + i * kGroups;
      const bool in = e < E && r < rows;
      d[i] = in ? a.part_c[static_cast<int64_t>(r) * E + e] : 0;
      q[i] = in && balance ? a.part_p[static_cast<int64_t>(r) * E + e] : 0.0f;
    }
    float p = 0.0f;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) p += q[i], c += d[i];
    __syncthreads();
    sp[tid] = p;
    sc[tid] = c;
    __syncthreads();
    if (warp == 0 && e < E) {
#pragma unroll 8
      for (int g = 1; g < kGroups; ++g) p += sp[g * kCols + lane], c += sc[g * kCols + lane];
      loss += finish(a, e, p, c, n);
    }
  }
  if (blockIdx.x == 0 && tid == 0 && a.tokens) *a.tokens = n;
  if (!balance) return;
  loss = warp_sum(loss);
  if (tid == 0) block_loss = loss;
  cluster.sync();
  if (blockIdx.x == 0 && tid == 0) {
    float s = 0.0f;
    for (int b = 0; b < kSumCtas; ++b) s += *cluster.map_shared_rank(&block_loss, b);
    *a.loss = s * E;
  }
  cluster.sync();  // the blocks' shared memory stays until it has been read
}

struct BackwardArgs {
  const void *logits;
  int64_t T, stride;
  int E, topk, renormalize;
  const uint8_t *valid;
  const int32_t *ids;         // the forward pass's choices (with grad_weights)
  const float *grad_weights;  // NULL: no gradient through the weights
  const int64_t *counts;      // [E] (with grad_loss)
  const int64_t *tokens;
  const float *grad_loss;     // NULL: no gradient through the loss
  void *grad;                 // [T, E], contiguous
};

template <typename T, int VPL, bool VEC>
__global__ void __launch_bounds__(256, VPL <= 16 ? 4 : (VPL <= 32 ? 2 : 1))
    backward_kernel(const __grid_constant__ BackwardArgs a) {
  using R = Row<T, VPL, VEC>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int E = a.E, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *h = reinterpret_cast<float *>(smem);         // [E]: dL/dp of the loss
  float *sel = h + E + static_cast<int64_t>(warp) * E;  // [E] for each warp: the choices' part
  const bool balance = a.grad_loss != nullptr, choices = a.grad_weights != nullptr;
  {
    float s = 0.0f;
    if (balance) {
      const float n = static_cast<float>(a.tokens ? *a.tokens : a.T);
      if (n > 0.0f) s = *a.grad_loss * E / n / (n * a.topk);
    }
    for (int e = threadIdx.x; e < E; e += blockDim.x)
      h[e] = balance ? s * static_cast<float>(a.counts[e]) : 0.0f;
    if (choices)
      for (int e = lane; e < E; e += 32) sel[e] = 0.0f;
  }
  __syncthreads();
  const int64_t step = static_cast<int64_t>(gridDim.x) * warps;
  int64_t t = static_cast<int64_t>(blockIdx.x) * warps + warp;
  auto counts = [&](int64_t u) { return u < a.T && (!a.valid || a.valid[u]); };
  auto row_of = [&](int64_t u) { return static_cast<const T *>(a.logits) + u * a.stride; };
  typename R::Raw raw;
  bool now = counts(t), next = counts(t + step);
  if (now) R::fetch(row_of(t), E, lane, raw);
  for (; t < a.T; t += step) {
    float v[VPL];
    T *out = static_cast<T *>(a.grad) + t * E;
    const T *row = row_of(t);
    bool live = now;
    if (live) R::open(raw, E, lane, v);
    now = next;
    next = counts(t + 2 * step);
    if (now) R::fetch(row_of(t + step), E, lane, raw);  // the next row, meanwhile
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
      v[i] = __expf(v[i] - m);
      z += v[i];
    }
    const float inv = 1.0f / warp_sum(z);
    float inner = 0.0f;  // sum_u p_u h_u
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = R::expert(i, lane);
      v[i] *= inv;
      if (e < E) inner += v[i] * h[e];
    }
    if (balance) inner = warp_sum(inner);
    if (choices) {
      int id = -1;
      float d = 0.0f;
      if (lane < a.topk) id = a.ids[t * a.topk + lane];
      const bool has = id >= 0 && id < E;
      const float g = has ? a.grad_weights[t * a.topk + lane] : 0.0f;
      float p = has ? __expf(widen(row[id]) - m) : 0.0f;
      if (a.renormalize) {
        const float total = warp_sum(p);
        const float w = has ? p / total : 0.0f;
        d = w * (g - warp_sum(w * g));
      } else {
        d = p * inv * g;
        inner += warp_sum(d);
      }
      if (has) sel[id] = d;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = R::expert(i, lane);
        if (e < E) v[i] = v[i] * (h[e] - inner) + sel[e];
      }
      __syncwarp();
      if (has) sel[id] = 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = R::expert(i, lane);
        if (e < E) v[i] *= h[e] - inner;
      }
    }
    R::store(out, E, lane, v);
  }
}

int set_smem(const void *fn, size_t bytes) {
  if (bytes <= 48 * 1024) return XP_OK;
  cudaError_t err =
      cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  return err == cudaSuccess ? XP_OK : static_cast<int>(err);
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
  auto fn = forward_kernel<T, VPL, VEC>;
  const int threads = forward_threads(VPL);
  const int64_t ctas = forward_ctas(a.T, a.E);
  const int rows = 1 + (a.loss ? (VPL > 32 ? threads / 32 : 1) : 0);
  const size_t smem = sizeof(float) * a.E * rows;
  int rc = set_smem((const void *)fn, smem);
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
  const int threads = 256;
  const size_t smem = sizeof(float) * a.E * (1 + (a.grad_weights ? threads / 32 : 0));
  int rc = set_smem((const void *)fn, smem);
  if (rc) return rc;
  const int64_t want = (a.T + threads / 32 - 1) / (threads / 32);
  const int64_t most = 148 * 8;
  fn<<<static_cast<unsigned>(want < most ? want : most), threads, smem, s>>>(a);
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
  return ctas == 1 ? 0 : ctas * (E * 8 + 4);
}

int run_forward(ForwardArgs &a, int dtype, void *scratch, int64_t scratch_bytes, void *stream) {
  const int64_t ctas = forward_ctas(a.T, a.E);
  if (ctas > 1) {
    if (!scratch || !aligned(scratch, 4) || scratch_bytes < scratch_need(a.T, a.E))
      return XP_EINVAL;
    a.part_p = static_cast<float *>(scratch);
    a.part_c = reinterpret_cast<int32_t *>(a.part_p + ctas * a.E);
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
                weights, ids, nullptr, 4, counts, tokens, loss, nullptr, nullptr, nullptr};
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
                nullptr, nullptr};
  return run_forward(a, dtype, scratch, scratch_bytes, stream);
}

extern "C" int xp_route_backward(const void *logits, int dtype, int64_t T, int64_t E,
                                 int64_t stride, const uint8_t *valid, const int32_t *ids,
                                 int64_t topk, int renormalize, const float *grad_weights,
                                 const int64_t *counts, const int64_t *tokens,
                                 const float *grad_loss, void *grad, void *stream) {
  int rc = check_sizes(dtype, T, E, stride, topk);
  if (rc) return rc;
  if (grad_weights && topk > XP_MAX_TOPK) return XP_ERANGE;
  if (T == 0) return XP_OK;
  if (!logits || !grad || (grad_weights && !ids) || (grad_loss && !counts) ||
      (grad_loss && valid && !tokens))
    return XP_EINVAL;
  BackwardArgs a{logits, T, stride, static_cast<int>(E), static_cast<int>(topk), renormalize,
                 valid, ids, grad_weights, counts, tokens,
                 grad_loss, grad};
  return by_type<BackwardArgs, Backward>(a, dtype, grad, as_stream(stream));
}
