// Low-rank adapters of many requests: out = y + scale_s (x A_s^T) B_s^T, the slot
// s of every row from its adapter id.
//
// Both products run on the tensor cores (16-bit operands, 32-bit sums).  Between
// them stands v = scale_s x A_s^T, r values a row, kept as two 16-bit parts
// (v = hi + lo): the second product then loses 2^-16 of v at most, where one part
// would lose as much as the output's own rounding.  float16 parts are taken of v
// times the power of two that brings the row's largest magnitude to 2^14, so that
// neither end of the type's range is left.
//
// Two kernels, by the number of rows (see kRowsLimit):
//
//  * rows_kernel: short batches, most rows with adapters of their own.  Bound by
//    reading the adapters.  A cluster of CTAs takes up to 8 rows of one adapter
//    and splits both products' long axes; every weight goes from memory straight
//    into a matrix instruction's registers, the weights as its 16-row operand and
//    the rows as its 8 columns.  Which rows belong together each cluster finds
//    out by itself from the ids, so the call is one launch.
//  * tile_kernel: long batches.  Bound by reading x and y and writing out.  A
//    small launch sorts the rows by slot; then a CTA (or a cluster, where there
//    are few tiles) takes up to 64 rows of one adapter and streams x and A, then
//    B and y, through one ring of shared-memory stages, so that the second
//    product's operands are on their way while the first one ends.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace xp {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRowsLimit = 512;   // rows_kernel up to here
constexpr int kGroup = 8;         // rows of a cluster of rows_kernel
constexpr int kTile = 64;         // rows of a tile
constexpr int kStages = 4;        // ring of tile_kernel
constexpr int kPlanThreads = 1024;

struct LowRankArgs {
  const void *x, *y;
  void *out;
  int64_t x_stride, y_stride, out_stride;
  int64_t M, H, N;
  int r, slots;
  const void *a, *b;
  const float *scale;
  const void *ids;
  int ids_bytes;
  const int32_t *slot_of;
  int64_t adapters;
  int vec_x, vec_a, vec_b, vec_y;  // 16-byte accesses to x, A, B, and y with out
  int in_place;
  // The plan of tile_kernel.
  int32_t *perm;   // [M] rows by slot
  int4 *tiles;     // (slot, first place in perm, rows, -)
  int32_t *ntiles;
};

template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  static constexpr bool kNarrowRange = false;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Half<__half> {
  static constexpr bool kNarrowRange = true;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<__half2 *>(&w));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ void narrow(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void narrow(__half *p, float x) { *p = __float2half_rn(x); }

// The high and the low part of two neighbouring values.  Where the high part is
// not finite the low part is 0, so that an infinity stays one.
template <typename T>
__device__ __forceinline__ void split(float u, float w, uint32_t *hi, uint32_t *lo) {
  *hi = Half<T>::pack(u, w);
  const float2 h = Half<T>::unpack(*hi);
  *lo = Half<T>::pack(isfinite(h.x) ? u - h.x : 0.0f, isfinite(h.y) ? w - h.y : 0.0f);
}

// The power of two that brings a row's largest magnitude into [2^14, 2^15); 1 for
// rows of zeros (or less than 2^-126), of infinities and of NaN.
__device__ __forceinline__ float range_factor(float amax) {
  const int e = static_cast<int>(__float_as_uint(amax) >> 23);  // the biased exponent
  return e == 0 || e >= 254 ? 1.0f
                            : __uint_as_float(static_cast<uint32_t>(min(268 - e, 253)) << 23);
}

// The slot of row m, -1 without an adapter.
__device__ __forceinline__ int slot_of_row(const LowRankArgs &a, int64_t m) {
  int64_t s = load_id(a.ids, a.ids_bytes, m);
  if (a.slot_of) s = s >= 0 && s < a.adapters ? a.slot_of[s] : -1;
  return s >= 0 && s < a.slots ? static_cast<int>(s) : -1;
}

// Eight neighbouring values, those from `valid` on as zeros (valid may be <= 0).
template <typename T>
__device__ __forceinline__ uint4 load8(const T *p, int64_t valid, bool vec) {
  if (vec && valid >= 8) return __ldg(reinterpret_cast<const uint4 *>(p));
  uint4 q = make_uint4(0, 0, 0, 0);
  const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < valid) (&q.x)[i >> 1] |= static_cast<uint32_t>(__ldg(h + i)) << (16 * (i & 1));
  return q;
}

__device__ __forceinline__ void copy_row(const LowRankArgs &a, int64_t m, int part, int parts) {
  const uint16_t *y = static_cast<const uint16_t *>(a.y) + m * a.y_stride;
  uint16_t *out = static_cast<uint16_t *>(a.out) + m * a.out_stride;
  const int64_t first = static_cast<int64_t>(part) * kThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(parts) * kThreads;
  if (a.vec_y) {
    for (int64_t n = first; n < a.N / 8; n += step)
      reinterpret_cast<uint4 *>(out)[n] = reinterpret_cast<const uint4 *>(y)[n];
    for (int64_t n = a.N / 8 * 8 + first; n < a.N; n += step) out[n] = y[n];
  } else {
    for (int64_t n = first; n < a.N; n += step) out[n] = y[n];
  }
}

// ---- short batches ----

// kRB: blocks of 16 ranks.
template <typename T, int kRB>
__global__ void __launch_bounds__(kThreads) rows_kernel(const __grid_constant__ LowRankArgs a) {
  constexpr int kR = kRB * 16;
  __shared__ float red[kWarps][kR * kGroup];
  __shared__ float part[kR * kGroup];   // [rank][row]: this CTA's share of v
  __shared__ float vf[kR * kGroup];     // [rank][row]: v
  __shared__ float factor[kGroup];
  __shared__ __align__(16) uint16_t vhi[kGroup][kR + 24], vlo[kGroup][kR + 24];
  __shared__ uint32_t same[kRowsLimit / 32];
  __shared__ int rows[kGroup];
  __shared__ int nrows;

  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int m = blockIdx.x / C, M = static_cast<int>(a.M);
  const int s = slot_of_row(a, m);
  if (s < 0) {
    if (!a.in_place) copy_row(a, m, rank, C);
    return;  // every CTA of the cluster
  }
  // The rows of this adapter: a cluster leads where its row is the first of
  // every eight, and takes these eight.
  for (int w = warp; w < (M + 31) / 32; w += kWarps) {
    const int j = w * 32 + lane;
    const uint32_t b = __ballot_sync(kFull, j < M && slot_of_row(a, j) == s);
    if (lane == 0) same[w] = b;
  }
  __syncthreads();
  if (warp == 0) {
    const int words = (M + 31) / 32;
    uint32_t w = lane < words ? same[lane] : 0;
    int before = __popc(w);  // set bits of the words before this lane's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(kFull, before, o);
      if (lane >= o) before += u;
    }
    const int total = __shfl_sync(kFull, before, 31);
    before -= __popc(w);
    const int mine = __shfl_sync(kFull, before + __popc(w & ((1u << (m & 31)) - 1)), m >> 5);
    if (lane == 0) nrows = mine % kGroup ? 0 : min(kGroup, total - mine);
    for (; w; w &= w - 1, ++before)
      if (before >= mine && before < mine + kGroup) rows[before - mine] = lane * 32 + __ffs(w) - 1;
  }
  __syncthreads();
  const int n_rows = nrows;
  if (n_rows == 0) return;  // every CTA of the cluster

  const T *A = static_cast<const T *>(a.a) + static_cast<int64_t>(s) * a.r * a.H;
  const T *B = static_cast<const T *>(a.b) + static_cast<int64_t>(s) * a.r * a.N;
  const int units = C * kWarps, unit = rank * kWarps + warp;
  const int64_t nblocks = (a.N + 15) / 16;
  // The second product's weights come on their way while the first one runs.
  for (int64_t nb = unit; nb < nblocks; nb += units) {
    const char *p = reinterpret_cast<const char *>(B + nb * 16 * a.r);
    const int64_t bytes = min(static_cast<int64_t>(16), a.N - nb * 16) * a.r * 2;
    for (int64_t o = lane * 128; o < bytes; o += 32 * 128)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p + o));
  }

  // v^T[rank, row]: weights as the 16 rows of an instruction, rows as its columns.
  // A lane's 16 bytes of a weight row are k = 8t .. 8t+7 of a block of 32; rows
  // use the same order, so the sum over k is the same one.
  float c[kRB][4];
#pragma unroll
  for (int i = 0; i < kRB; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = 0.0f;
  const T *x = static_cast<const T *>(a.x) + (g < n_rows ? rows[g] : rows[0]) * a.x_stride;
  const int64_t kblocks = (a.H + 31) / 32;
#pragma unroll 2
  for (int64_t kb = unit; kb < kblocks; kb += units) {
    const int64_t k = kb * 32 + 8 * t;
    const uint4 q = load8(x + k, g < n_rows ? a.H - k : 0, a.vec_x);
#pragma unroll
    for (int i = 0; i < kRB; ++i) {
      const int r0 = i * 16 + g, r1 = r0 + 8;
      const uint4 u = load8(A + r0 * a.H + k, r0 < a.r ? a.H - k : 0, a.vec_a);
      const uint4 w = load8(A + r1 * a.H + k, r1 < a.r ? a.H - k : 0, a.vec_a);
      Half<T>::mma(c[i], u.x, w.x, u.y, w.y, q.x, q.y);
      Half<T>::mma(c[i], u.z, w.z, u.w, w.w, q.z, q.w);
    }
  }
#pragma unroll
  for (int i = 0; i < kRB; ++i) {
    float *p = red[warp] + (i * 16 + g) * kGroup + 2 * t;
    p[0] = c[i][0], p[1] = c[i][1];
    p[8 * kGroup] = c[i][2], p[8 * kGroup + 1] = c[i][3];
  }
  __syncthreads();
  for (int i = tid; i < kR * kGroup; i += kThreads) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += red[w][i];
    part[i] = sum;
  }
  cluster.sync();
  const float scale = a.scale ? a.scale[s] : 1.0f;
  for (int i = tid; i < kR * kGroup; i += kThreads) {
    float sum = 0.0f;
    for (int p = 0; p < C; ++p) sum += cluster.map_shared_rank(part, p)[i];
    vf[i] = sum * scale;
  }
  // The other CTAs have read this one's share when all have arrived; waited for
  // at the end.
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  __syncthreads();
  {  // warp w: row w
    float f = 1.0f;
    if constexpr (Half<T>::kNarrowRange) {
      float amax = 0.0f;
      for (int i = lane; i < kR; i += 32) amax = fmaxf(amax, fabsf(vf[i * kGroup + warp]));
      f = range_factor(__uint_as_float(__reduce_max_sync(kFull, __float_as_uint(amax))));
    }
    for (int i = 2 * lane; i < kR; i += 64) {
      uint32_t hi, lo;
      split<T>(vf[i * kGroup + warp] * f, vf[(i + 1) * kGroup + warp] * f, &hi, &lo);
      *reinterpret_cast<uint32_t *>(&vhi[warp][i]) = hi;
      *reinterpret_cast<uint32_t *>(&vlo[warp][i]) = lo;
    }
    if (kR % 32)  // the second half of the last block of 32
      for (int i = kR + lane; i < kR + 16; i += 32) vhi[warp][i] = vlo[warp][i] = 0;
    if (lane == 0) factor[warp] = 1.0f / f;
  }
  __syncthreads();

  const int row0 = 2 * t, row1 = 2 * t + 1;
  const float f0 = factor[row0], f1 = factor[row1];
  const bool has0 = row0 < n_rows, has1 = row1 < n_rows;
  const T *y0 = static_cast<const T *>(a.y) + (has0 ? rows[row0] : 0) * a.y_stride;
  const T *y1 = static_cast<const T *>(a.y) + (has1 ? rows[row1] : 0) * a.y_stride;
  T *o0 = static_cast<T *>(a.out) + (has0 ? rows[row0] : 0) * a.out_stride;
  T *o1 = static_cast<T *>(a.out) + (has1 ? rows[row1] : 0) * a.out_stride;
  for (int64_t nb = unit; nb < nblocks; nb += units) {
    const int64_t n0 = nb * 16 + g, n1 = n0 + 8;
    const bool in0 = n0 < a.N, in1 = n1 < a.N;
    const float y00 = has0 && in0 ? widen(y0[n0]) : 0.0f, y01 = has1 && in0 ? widen(y1[n0]) : 0.0f;
    const float y10 = has0 && in1 ? widen(y0[n1]) : 0.0f, y11 = has1 && in1 ? widen(y1[n1]) : 0.0f;
    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < (kRB + 1) / 2; ++i) {
      const int k = i * 32 + 8 * t;
      const uint4 u = load8(B + n0 * a.r + k, in0 ? a.r - k : 0, a.vec_b);
      const uint4 w = load8(B + n1 * a.r + k, in1 ? a.r - k : 0, a.vec_b);
      const uint4 h = *reinterpret_cast<const uint4 *>(&vhi[g][k]);
      const uint4 l = *reinterpret_cast<const uint4 *>(&vlo[g][k]);
      Half<T>::mma(d, u.x, w.x, u.y, w.y, h.x, h.y);
      Half<T>::mma(d, u.z, w.z, u.w, w.w, h.z, h.w);
      Half<T>::mma(d, u.x, w.x, u.y, w.y, l.x, l.y);
      Half<T>::mma(d, u.z, w.z, u.w, w.w, l.z, l.w);
    }
    if (has0 && in0) narrow(o0 + n0, y00 + d[0] * f0);
    if (has1 && in0) narrow(o1 + n0, y01 + d[1] * f1);
    if (has0 && in1) narrow(o0 + n1, y10 + d[2] * f0);
    if (has1 && in1) narrow(o1 + n1, y11 + d[3] * f1);
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- long batches ----

// Sorts the rows by slot and cuts each slot's rows into tiles.  The order of a
// slot's rows is free: a row's result does not depend on its tile.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ LowRankArgs a) {
  extern __shared__ int count[];  // [slots + 1]: rows, then the next free place
  __shared__ int sum_rows[32], sum_tiles[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = a.slots + 1, M = static_cast<int>(a.M);  // the last: rows without an adapter
  for (int i = tid; i < n; i += kPlanThreads) count[i] = 0;
  __syncthreads();
  for (int m0 = warp * 32; m0 < M; m0 += kPlanThreads) {
    const int m = m0 + lane;
    int s = -2;
    if (m < M) {
      s = slot_of_row(a, m);
      if (s < 0) s = a.slots;
    }
    const unsigned peers = __match_any_sync(kFull, s);
    if (s >= 0 && lane == __ffs(peers) - 1) atomicAdd(&count[s], __popc(peers));
  }
  __syncthreads();
  // Exclusive sums over the slots, a run of slots per thread.
  const int run = (n + kPlanThreads - 1) / kPlanThreads, i0 = min(tid * run, n),
            i1 = min(i0 + run, n);
  int rows = 0, tiles = 0;
  for (int i = i0; i < i1; ++i) {
    rows += count[i];
    if (i < a.slots || !a.in_place) tiles += (count[i] + kTile - 1) / kTile;
  }
  int rows_before = rows, tiles_before = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(kFull, rows_before, o);
    const int v = __shfl_up_sync(kFull, tiles_before, o);
    if (lane >= o) rows_before += u, tiles_before += v;
  }
  if (lane == 31) sum_rows[warp] = rows_before, sum_tiles[warp] = tiles_before;
  __syncthreads();
  rows_before -= rows;
  tiles_before -= tiles;
  for (int w = 0; w < warp; ++w) rows_before += sum_rows[w], tiles_before += sum_tiles[w];
  for (int i = i0; i < i1; ++i) {
    const int rows_here = count[i];
    count[i] = rows_before;
    if (i < a.slots || !a.in_place)
      for (int o = 0; o < rows_here; o += kTile)
        a.tiles[tiles_before++] =
            make_int4(i < a.slots ? i : -1, rows_before + o, min(kTile, rows_here - o), 0);
    rows_before += rows_here;
  }
  if (tid == kPlanThreads - 1) *a.ntiles = tiles_before;
  __syncthreads();
  for (int m0 = warp * 32; m0 < M; m0 += kPlanThreads) {
    const int m = m0 + lane;
    int s = -2;
    if (m < M) {
      s = slot_of_row(a, m);
      if (s < 0) s = a.slots;
    }
    const unsigned peers = __match_any_sync(kFull, s);
    int place = 0;
    const int leader = __ffs(peers) - 1;
    if (s >= 0 && lane == leader) place = atomicAdd(&count[s], __popc(peers));
    place = __shfl_sync(kFull, place, leader) + __popc(peers & lanemask_lt());
    if (s >= 0) a.perm[place] = m;
  }
}

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// Eight values into shared memory, those from `valid` on as zeros: asynchronously
// where 16-byte accesses are allowed.
template <typename T>
__device__ __forceinline__ void fetch8(uint32_t dst, const T *src, int64_t valid, bool vec) {
  if (vec) {
    const int bytes = valid >= 8 ? 16 : (valid <= 0 ? 0 : static_cast<int>(valid) * 2);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
  } else {
    const uint4 q = load8(src, valid, false);
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(q.x), "r"(q.y), "r"(q.z),
                 "r"(q.w)
                 : "memory");
  }
}

constexpr int kPitch = 144;  // bytes of a row of 64 values: 16 more, so that 8 rows meet 8 banks

template <int kRB>
struct TileSmem {
  static constexpr int kR = kRB * 16;
  static constexpr int kPitchB = kR * 2 + 16;  // bytes of a row of B
  // A stage holds 64 rows x 64 values of x and kR x 64 of A, or 64 rows of B and 64 x 64 of y.
  static constexpr int kFirst = kTile * kPitch + kR * kPitch;
  static constexpr int kSecond = 64 * kPitchB + kTile * kPitch;
  static constexpr int kStage = kFirst > kSecond ? kFirst : kSecond;
  static constexpr int kPitchV = kR + 4;  // floats of a row of v
  static constexpr int kV = kTile * kPitchV * 4;
  static constexpr int kBytes = kStages * kStage + kV;
};

template <typename T, int kRB>
__global__ void __launch_bounds__(kThreads, kRB <= 4 ? 2 : 1)
    tile_kernel(const __grid_constant__ LowRankArgs a) {
  using S = TileSmem<kRB>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int64_t rows[kTile];
  __shared__ float factor[kTile];
  float *v = reinterpret_cast<float *>(smem + kStages * S::kStage);

  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wm = warp & 3, wk = warp >> 2;
  const int tile = blockIdx.x / C;
  if (tile >= *a.ntiles) return;
  const int4 job = a.tiles[tile];
  const int s = job.x, n_rows = job.z;
  if (s < 0) {
    for (int i = 0; i < n_rows; ++i) copy_row(a, a.perm[job.y + i], rank, C);
    return;
  }
  if (tid < kTile) rows[tid] = a.perm[job.y + min(tid, n_rows - 1)];
  __syncthreads();

  const T *A = static_cast<const T *>(a.a) + static_cast<int64_t>(s) * a.r * a.H;
  const T *B = static_cast<const T *>(a.b) + static_cast<int64_t>(s) * a.r * a.N;
  const T *x = static_cast<const T *>(a.x), *y = static_cast<const T *>(a.y);
  // This CTA's blocks of 64 along H and along N.
  const int kb_all = static_cast<int>((a.H + 63) / 64), nb_all = static_cast<int>((a.N + 63) / 64);
  const int k0 = static_cast<int>(static_cast<int64_t>(kb_all) * rank / C);
  const int k1 = static_cast<int>(static_cast<int64_t>(kb_all) * (rank + 1) / C);
  const int n0 = static_cast<int>(static_cast<int64_t>(nb_all) * rank / C);
  const int n1 = static_cast<int>(static_cast<int64_t>(nb_all) * (rank + 1) / C);
  const int first = k1 - k0, chunks = first + n1 - n0;

  auto issue = [&](int c) {
    if (c < chunks) {
      const uint32_t at = smem_addr(smem + (c % kStages) * S::kStage);
      if (c < first) {
        const int64_t k = static_cast<int64_t>(k0 + c) * 64;
        for (int i = tid; i < kTile * 8; i += kThreads) {
          const int row = i >> 3, e = (i & 7) * 8;
          fetch8(at + row * kPitch + e * 2, x + rows[row] * a.x_stride + k + e, a.H - k - e,
                 a.vec_x);
        }
        for (int i = tid; i < S::kR * 8; i += kThreads) {
          const int row = i >> 3, e = (i & 7) * 8;
          fetch8(at + kTile * kPitch + row * kPitch + e * 2,
                 A + static_cast<int64_t>(min(row, a.r - 1)) * a.H + k + e,
                 row < a.r ? a.H - k - e : 0, a.vec_a);
        }
      } else {
        const int64_t n = static_cast<int64_t>(n0 + c - first) * 64;
        for (int i = tid; i < 64 * kRB * 2; i += kThreads) {
          const int row = i / (kRB * 2), e = (i % (kRB * 2)) * 8;
          const bool in = n + row < a.N;
          fetch8(at + row * S::kPitchB + e * 2, B + (in ? n + row : 0) * a.r + e,
                 in ? a.r - e : 0, a.vec_b);
        }
        for (int i = tid; i < kTile * 8; i += kThreads) {
          const int row = i >> 3, e = (i & 7) * 8;
          fetch8(at + 64 * S::kPitchB + row * kPitch + e * 2, y + rows[row] * a.y_stride + n + e,
                 row < n_rows ? a.N - n - e : 0, a.vec_y);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto arrived = [&]() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();
  };

  for (int c = 0; c < kStages - 1; ++c) issue(c);

  // First product: 16 rows a warp, the two halves of the warps take every other
  // 32 values of a block.
  float acc[kRB * 2][4];
#pragma unroll
  for (int i = 0; i < kRB * 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  for (int c = 0; c < first; ++c) {
    arrived();
    issue(c + kStages - 1);
    const uint32_t at = smem_addr(smem + (c % kStages) * S::kStage);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = wk * 32 + h * 16;
      uint32_t p[4];
      ldmatrix4(p, at + (wm * 16 + (lane & 15)) * kPitch + (k + (lane >> 4) * 8) * 2);
#pragma unroll
      for (int i = 0; i < kRB; ++i) {
        uint32_t q[4];  // ranks 16 i .. 16 i + 15: two column blocks of an instruction
        ldmatrix4(q, at + kTile * kPitch + (i * 16 + (lane >> 4) * 8 + (lane & 7)) * kPitch +
                         (k + ((lane >> 3) & 1) * 8) * 2);
        Half<T>::mma(acc[2 * i], p[0], p[1], p[2], p[3], q[0], q[1]);
        Half<T>::mma(acc[2 * i + 1], p[0], p[1], p[2], p[3], q[2], q[3]);
      }
    }
  }
  // v of this CTA's share of H, the second half of the warps onto the first.
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (wk == half) {
#pragma unroll
      for (int i = 0; i < kRB * 2; ++i) {
        float *p = v + (wm * 16 + g) * S::kPitchV + i * 8 + 2 * t, *q = p + 8 * S::kPitchV;
        if (half == 0) {
          p[0] = acc[i][0], p[1] = acc[i][1], q[0] = acc[i][2], q[1] = acc[i][3];
        } else {
          p[0] += acc[i][0], p[1] += acc[i][1], q[0] += acc[i][2], q[1] += acc[i][3];
        }
      }
    }
    __syncthreads();
  }
  const float scale = a.scale ? a.scale[s] : 1.0f;
  {
    // Four lanes a row: the sum over the cluster, the scale and the row's range.
    const int row = tid >> 2, part = tid & 3;
    float *p = v + row * S::kPitchV;
    float u[S::kR / 4], amax = 0.0f;
    if (C > 1) cluster.sync();
#pragma unroll
    for (int i = 0; i < S::kR / 4; ++i) u[i] = 0.0f;
    for (int b = 0; b < C; ++b) {
      const float *q = (C > 1 ? cluster.map_shared_rank(v, b) : v) + row * S::kPitchV;
#pragma unroll
      for (int i = 0; i < S::kR / 4; ++i) u[i] += q[i * 4 + part];
    }
    if (C > 1) cluster.sync();  // all shares are read; now they may be overwritten
    float f = 1.0f;
#pragma unroll
    for (int i = 0; i < S::kR / 4; ++i) u[i] *= scale, amax = fmaxf(amax, fabsf(u[i]));
    if constexpr (Half<T>::kNarrowRange) {
      amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
      f = range_factor(amax);
    }
#pragma unroll
    for (int i = 0; i < S::kR / 4; ++i) p[i * 4 + part] = u[i] * f;
    if (part == 0) factor[row] = 1.0f / f;
  }
  __syncthreads();

  // Second product: v as the row operand, in two parts.
  uint32_t hi[kRB][4], lo[kRB][4];
#pragma unroll
  for (int i = 0; i < kRB; ++i) {
    const float *p = v + (wm * 16 + g) * S::kPitchV + i * 16 + 2 * t, *q = p + 8 * S::kPitchV;
    split<T>(p[0], p[1], &hi[i][0], &lo[i][0]);
    split<T>(q[0], q[1], &hi[i][1], &lo[i][1]);
    split<T>(p[8], p[9], &hi[i][2], &lo[i][2]);
    split<T>(q[8], q[9], &hi[i][3], &lo[i][3]);
  }
  const float f0 = factor[wm * 16 + g], f1 = factor[wm * 16 + g + 8];
  T *out = static_cast<T *>(a.out);
  for (int c = first; c < chunks; ++c) {
    arrived();
    issue(c + kStages - 1);
    unsigned char *stage = smem + (c % kStages) * S::kStage;
    const uint32_t at = smem_addr(stage);
    const int64_t n = static_cast<int64_t>(n0 + c - first) * 64 + wk * 32;
    float d[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) d[i][j] = 0.0f;
#pragma unroll
    for (int i = 0; i < kRB; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t q[4];
        ldmatrix4(q, at + (wk * 32 + j * 16 + (lane >> 4) * 8 + (lane & 7)) * S::kPitchB +
                         (i * 16 + ((lane >> 3) & 1) * 8) * 2);
        Half<T>::mma(d[2 * j], hi[i][0], hi[i][1], hi[i][2], hi[i][3], q[0], q[1]);
        Half<T>::mma(d[2 * j + 1], hi[i][0], hi[i][1], hi[i][2], hi[i][3], q[2], q[3]);
        Half<T>::mma(d[2 * j], lo[i][0], lo[i][1], lo[i][2], lo[i][3], q[0], q[1]);
        Half<T>::mma(d[2 * j + 1], lo[i][0], lo[i][1], lo[i][2], lo[i][3], q[2], q[3]);
      }
    }
    // y + update in place of y in the stage, by the warp whose 16 x 32 values they
    // are; then whole 16-byte pieces of out.
    unsigned char *ys = stage + 64 * S::kPitchB + wm * 16 * kPitch + wk * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t *p = reinterpret_cast<uint32_t *>(ys + g * kPitch + i * 16 + 4 * t);
      uint32_t *q = reinterpret_cast<uint32_t *>(ys + (g + 8) * kPitch + i * 16 + 4 * t);
      const float2 u = Half<T>::unpack(*p), w = Half<T>::unpack(*q);
      *p = Half<T>::pack(u.x + d[i][0] * f0, u.y + d[i][1] * f0);
      *q = Half<T>::pack(w.x + d[i][2] * f1, w.y + d[i][3] * f1);
    }
    __syncwarp();
#pragma unroll
    for (int i = lane; i < 64; i += 32) {
      const int row = i >> 2, e = (i & 3) * 8;
      if (wm * 16 + row >= n_rows) continue;
      const int64_t at_n = n + e;
      T *o = out + rows[wm * 16 + row] * a.out_stride + at_n;
      const unsigned char *p = ys + row * kPitch + e * 2;
      if (a.vec_y && at_n + 8 <= a.N) {
        *reinterpret_cast<uint4 *>(o) = *reinterpret_cast<const uint4 *>(p);
      } else {
        for (int j = 0; j < 8 && at_n + j < a.N; ++j) o[j] = reinterpret_cast<const T *>(p)[j];
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

int set_smem(const void *fn, int bytes) {
  if (bytes <= 48 * 1024) return XP_OK;
  cudaError_t err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  return err == cudaSuccess ? XP_OK : static_cast<int>(err);
}

int launch(const void *fn, unsigned ctas, unsigned cluster, int smem, const LowRankArgs &a,
           cudaStream_t s) {
  int rc = set_smem(fn, smem);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas * cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void *args[] = {const_cast<LowRankArgs *>(&a)};
  cudaError_t err = cudaLaunchKernelExC(&cfg, fn, args);
  return err == cudaSuccess ? launch_status() : static_cast<int>(err);
}

int64_t most_tiles(int64_t M, int64_t slots) {
  return (M + kTile - 1) / kTile + (slots + 1 < M ? slots + 1 : M);
}

int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// ntiles, the tiles, the rows by slot.
int64_t scratch_need(int64_t M, int64_t slots) {
  return M <= kRowsLimit ? 0 : 16 + 16 * most_tiles(M, slots) + round16(4 * M);
}

template <typename T, int kRB>
int run_sized(LowRankArgs &a, cudaStream_t s) {
  if (a.M <= kRowsLimit) {
    const unsigned cluster = a.M <= 16 ? 8 : 4;
    return launch((const void *)rows_kernel<T, kRB>, static_cast<unsigned>(a.M), cluster, 0, a, s);
  }
  const int bytes = 4 * (a.slots + 1);
  int rc = set_smem((const void *)plan_kernel, bytes);
  if (rc) return rc;
  plan_kernel<<<1, kPlanThreads, bytes, s>>>(a);
  rc = launch_status();
  if (rc) return rc;
  const int64_t tiles = most_tiles(a.M, a.slots);
  const int64_t full = (a.M + kTile - 1) / kTile;  // tiles of a batch with few adapters
  const unsigned cluster = full <= 40 ? 4 : (full <= 148 ? 2 : 1);
  return launch((const void *)tile_kernel<T, kRB>, static_cast<unsigned>(tiles), cluster,
                TileSmem<kRB>::kBytes, a, s);
}

template <typename T>
int run_typed(LowRankArgs &a, cudaStream_t s) {
  if (a.r <= 16) return run_sized<T, 1>(a, s);
  if (a.r <= 32) return run_sized<T, 2>(a, s);
  if (a.r <= 64) return run_sized<T, 4>(a, s);
  return run_sized<T, 8>(a, s);
}

}  // namespace
}  // namespace xp

using namespace xp;

extern "C" int64_t xp_low_rank_scratch_bytes(int64_t M, int64_t slots) {
  if (M < 0 || M > XP_MAX_TOKENS || slots < 1 || slots > XP_MAX_ADAPTER_SLOTS) return -1;
  return scratch_need(M, slots);
}

extern "C" int xp_add_low_rank(const void *x, int64_t x_stride, const void *y, int64_t y_stride,
                               void *out, int64_t out_stride, int dtype, int64_t M, int64_t H,
                               int64_t N, int64_t r, const void *a, const void *b, int64_t slots,
                               const float *scale, const void *ids, int ids_bytes,
                               const int32_t *slot_of, int64_t adapters, void *scratch,
                               int64_t scratch_bytes, void *stream) {
  if (dtype != XP_BF16 && dtype != XP_F16) return XP_EINVAL;
  if (M < 0 || H < 1 || N < 1 || r < 1 || slots < 1 || adapters < 0) return XP_EINVAL;
  if (M > XP_MAX_TOKENS || r > XP_MAX_RANK || slots > XP_MAX_ADAPTER_SLOTS || H > INT32_MAX ||
      N > INT32_MAX)
    return XP_ERANGE;
  if (ids_bytes != 4 && ids_bytes != 8) return XP_EINVAL;
  if (x_stride < 0 || y_stride < 0 || (M > 1 && out_stride < N)) return XP_EINVAL;
  if (M == 0) return XP_OK;
  if (!x || !y || !out || !a || !b || !ids) return XP_EINVAL;
  if (scratch_need(M, slots) > 0 &&
      (!scratch || !aligned(scratch, 16) || scratch_bytes < scratch_need(M, slots)))
    return XP_EINVAL;
  LowRankArgs p{x, y, out, x_stride, y_stride, out_stride, M, H, N,
                static_cast<int>(r), static_cast<int>(slots), a, b, scale, ids, ids_bytes, slot_of,
                adapters};
  p.vec_x = aligned(x, 16) && x_stride % 8 == 0;
  p.vec_a = aligned(a, 16) && H % 8 == 0;
  p.vec_b = aligned(b, 16) && r % 8 == 0;
  p.vec_y = aligned(y, 16) && aligned(out, 16) && y_stride % 8 == 0 && out_stride % 8 == 0;
  p.in_place = y == out && y_stride == out_stride;
  if (M > kRowsLimit) {
    unsigned char *at = static_cast<unsigned char *>(scratch);
    p.ntiles = reinterpret_cast<int32_t *>(at);
    p.tiles = reinterpret_cast<int4 *>(at + 16);
    p.perm = reinterpret_cast<int32_t *>(at + 16 + 16 * most_tiles(M, slots));
  }
  return dtype == XP_BF16 ? run_typed<__nv_bfloat16>(p, as_stream(stream))
                          : run_typed<__half>(p, as_stream(stream));
}
