// Low-rank adapters of many requests: out = y + scale_s (x A_s^T) B_s^T, the slot
// s of every row from its adapter id.
//
// Both products run on the tensor cores (16-bit operands, 32-bit sums).  Between
// them stands v = scale_s x A_s^T, r values a row, which enters the second product
// whole, as the sum of three 16-bit parts (8 or 11 bits each; two of bfloat16 would
// lose 2^-16 of v, which shows where v's terms cancel).  float16 parts are taken of v
// times the power of two that brings the row's largest magnitude to 2^14, so that
// neither end of the type's range is left; its least value then is 2^-38 of that magnitude,
// and bounds what values far below it keep.
//
// Two kernels, by the number of rows (see kRowsLimit):
//
//  * rows_kernel: short batches, most rows with adapters of their own.  Bound by
//    reading the adapters.  A cluster of CTAs takes up to 8 rows of one adapter
//    and splits both products' long axes, with the weights as a matrix
//    instruction's 16-row operand and the rows as its 8 columns (mma.sync: at 8
//    columns the tensor cores wait for memory in any form).  Which rows belong
//    together each cluster finds out by itself from the ids, so the call is one
//    launch.  B200, 256 rows of 100 adapters, rank 64, 2048 -> 1024: 15.8 us, of
//    which A comes at HBM's rate for 5.
//  * tile_kernel: long batches.  Bound by reading x and y and writing out.  A
//    small launch sorts the rows by slot; then a CTA (or a cluster, where there
//    are few tiles) takes up to 128 rows of one adapter: warps load x and A, then
//    B and y, through one ring of shared-memory stages, one thread issues tcgen05
//    instructions with the sums in tensor memory, and eight warps make v's parts
//    and write out.  The second product's operands are on their way while the
//    first one ends.  B200, 16384 rows, rank 64, 2048 -> 2048: 52 us against 32 of
//    HBM; a tile's chain of 64 blocks alone takes 45.  (mma.sync on 64-row tiles took
//    87: its instructions alone fill the tensor pipe for 29 us at that rank.)
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace xp {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
// rows_kernel up to here.  Measured at 2048 -> 2048, rank 16 (us, rows_kernel /
// tile_kernel): 512 rows of 4 adapters 9.5 / 18.7, of 256 adapters 26 / 72; 1024 rows
// 17.2 / 19.0 and 30 / 72; 1536 rows 23.2 / 19.3 and 35 / 72.  2048 -> 1024, rank 64: 1024
// rows 21 / 21 and 45 / 67; 1536 rows 32 / 21 and 50 / 67.  The bound knows the rows alone:
// right for few adapters, it gives 1536 rows of 256 adapters to the slower kernel.
constexpr int kRowsLimit = 1024;
constexpr int kGroup = 8;         // rows of a cluster of rows_kernel
constexpr int kRowStages = 3;     // its ring
constexpr int kTile = 128;        // rows of a tile
constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;      // one cluster

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
  const void *slot_of;  // NULL: ids are slots
  int slot_bytes;
  int64_t adapters;
  int vec_x, vec_a, vec_b, vec_y;  // 16-byte accesses to x, A, B, and y with out
  int in_place;
  int cluster_log2;  // CTAs of a cluster
  uint32_t wait_ns;  // after which a wait of tile_kernel gives up
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
  static constexpr float kLeast = 0x1p-133f;  // above 0
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
  }
  static __device__ __forceinline__ uint32_t cut(float lo, float hi) {
    uint32_t w;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
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
  static constexpr float kLeast = 0x1p-24f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
  }
  static __device__ __forceinline__ uint32_t cut(float lo, float hi) {
    uint32_t w;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
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

// The parts of two neighbouring values, cut and not rounded, so that each is exact and
// none leaves the range.  All have the value's sign and none is 0 unless the value is (the
// type's least value stands instead, below the last bit of any sum here), so that an
// infinity of B times the parts is the infinity that it is times the value, and no NaN.  Of
// an infinity or NaN the first part holds all.
template <typename T>
__device__ __forceinline__ void split(float u, float w, uint32_t (&part)[3]) {
  const uint32_t sign = (__float_as_uint(u) >> 16 & 0x8000u) | (__float_as_uint(w) & 0x80000000u);
  const float u0 = u == 0.0f ? 0.0f : Half<T>::kLeast, w0 = w == 0.0f ? 0.0f : Half<T>::kLeast;
  u = fabsf(u), w = fabsf(w);
  u = u < u0 ? u0 : u, w = w < w0 ? w0 : w;  // a NaN stays
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t q = Half<T>::cut(u, w);
    const float2 h = Half<T>::unpack(q);
    part[i] = q | sign;
    u = fmaxf(u - h.x, u0), w = fmaxf(w - h.y, w0);
  }
}

// The power of two that brings a row's largest magnitude (of the finite values) into
// [2^14, 2^15), 2^126 at most.
__device__ __forceinline__ float range_factor(float amax) {
  const int e = static_cast<int>(__float_as_uint(amax) >> 23);  // the biased exponent
  return __uint_as_float(static_cast<uint32_t>(min(268 - e, 253)) << 23);
}

__device__ __forceinline__ float finite_abs(float x) { return isfinite(x) ? fabsf(x) : 0.0f; }

// The slot of row m, -1 without an adapter.
__device__ __forceinline__ int slot_of_row(const LowRankArgs &a, int64_t m) {
  int64_t s = load_id(a.ids, a.ids_bytes, m);
  if (a.slot_of) s = s >= 0 && s < a.adapters ? load_id(a.slot_of, a.slot_bytes, s) : -1;
  return s >= 0 && s < a.slots ? static_cast<int>(s) : -1;
}

__device__ __forceinline__ int place_of(const void *p) {
  return static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
}

// Eight neighbouring values at any place, those from `valid` on as zeros (valid may
// be <= 0): the aligned 16-byte words around them (those two that hold at least one
// of the values), then shifts, which takes a quarter of the loads that single values
// would.  Two steps, so that several fetches can be under way.
struct Words {
  uint4 lo, hi;
};

template <typename T>
__device__ __forceinline__ Words fetch_words(const T *p, int64_t valid) {
  Words w = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (valid <= 0) return w;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  const int off = static_cast<int>(at & 15), n = valid < 8 ? static_cast<int>(valid) : 8;
  const uint4 *word = reinterpret_cast<const uint4 *>(at - off);
  w.lo = __ldg(word);
  if (off + 2 * n > 16) w.hi = __ldg(word + 1);
  return w;
}

// `off`: the first value's byte in the first word.
__device__ __forceinline__ uint4 join_words(const Words &v, int off, int64_t valid) {
  const int n = valid < 0 ? 0 : (valid < 8 ? static_cast<int>(valid) : 8);
  uint32_t w[8] = {v.lo.x, v.lo.y, v.lo.z, v.lo.w, v.hi.x, v.hi.y, v.hi.z, v.hi.w};
  if (off & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (off & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (off & 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (2 * i + 2 > n) w[i] &= 2 * i + 1 > n ? 0u : 0xffffu;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ uint4 load8(const T *p, int64_t valid, bool vec) {
  if (vec && valid >= 8) return __ldg(reinterpret_cast<const uint4 *>(p));
  return join_words(fetch_words(p, valid), place_of(p), valid);
}

// Eight neighbouring values of which `valid` exist, to any place.
template <typename T>
__device__ __forceinline__ void put8(T *p, const uint4 &q, int64_t valid, bool vec) {
  if (vec && valid >= 8) {
    *reinterpret_cast<uint4 *>(p) = q;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid)
        reinterpret_cast<uint16_t *>(p)[e] =
            static_cast<uint16_t>((&q.x)[e >> 1] >> (16 * (e & 1)));
  }
}

// out = y for n_rows rows (row(i): the i-th): part `part` of `parts`, by the whole
// block, four pieces of a thread under way.
template <typename T, typename Row>
__device__ __forceinline__ void copy_rows(const LowRankArgs &a, int n_rows, int part, int parts,
                                          Row row) {
  const int64_t pieces = (a.N + 7) / 8, all = n_rows * pieces;
  const int64_t step = static_cast<int64_t>(parts) * blockDim.x;
  for (int64_t i0 = static_cast<int64_t>(part) * blockDim.x + threadIdx.x; i0 < all;
       i0 += 4 * step) {
    uint4 q[4];
    int64_t m[4], n[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = i0 + j * step;
      if (i < all) {
        m[j] = row(static_cast<int>(i / pieces));
        n[j] = i % pieces * 8;
        q[j] = load8(static_cast<const T *>(a.y) + m[j] * a.y_stride + n[j], a.N - n[j], a.vec_y);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j * step < all)
        put8(static_cast<T *>(a.out) + m[j] * a.out_stride + n[j], q[j], a.N - n[j], a.vec_y);
  }
}

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes into shared memory, asynchronously; bytes from `bytes` on are zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}

__device__ __forceinline__ void store16(uint32_t dst, const uint4 &q) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(q.x), "r"(q.y), "r"(q.z),
               "r"(q.w)
               : "memory");
}

// ---- short batches ----

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void ldmatrix2(uint32_t (&r)[2], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
               : "=r"(r[0]), "=r"(r[1])
               : "r"(addr));
}

// Pitches are 16 bytes longer than the rows, so that eight rows' 16-byte pieces
// lie in different banks.
template <int kRB>
struct RowsSmem {
  static constexpr int kR = kRB * 16;
  static constexpr int kK = kRB <= 2 ? 256 : 8192 / kR;  // values of a row of A (and x) in a stage
  static constexpr int kN = (kRB <= 2 ? 4096 : 8192) / kR;  // rows of B in a stage, columns of y
  static constexpr int kPitchA = kK * 2 + 16, kPitchB = kR * 2 + 16, kPitchY = kN * 2 + 16;
  static constexpr int kFirst = (kR + kGroup) * kPitchA;
  static constexpr int kSecond = kN * kPitchB + kGroup * kPitchY;
  static constexpr int kStage = kFirst > kSecond ? kFirst : kSecond;
  static constexpr int kBytes = kRowStages * kStage;
};

// kRB: blocks of 16 ranks.  kVec: all rows allow 16-byte accesses.
template <typename T, int kRB, bool kVec>
__global__ void __launch_bounds__(kThreads, kVec && kRB <= 4 ? 3 : 2)
    rows_kernel(const __grid_constant__ LowRankArgs a) {
  using S = RowsSmem<kRB>;
  constexpr int kR = S::kR, kParts = kWarps / kRB;  // warps that share a block of ranks
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int kPitchV = kR + 4;
  // The warps' sums of v; when they have been added up, v's parts.
  constexpr int kRed = kParts * kGroup * kPitchV * 4, kSplit = 3 * kGroup * (kR + 8) * 2;
  __shared__ __align__(16) unsigned char room[kRed > kSplit ? kRed : kSplit];
  float(*red)[kGroup * kPitchV] = reinterpret_cast<float(*)[kGroup * kPitchV]>(room);
  uint16_t(*vs)[kGroup][kR + 8] = reinterpret_cast<uint16_t(*)[kGroup][kR + 8]>(room);
  __shared__ __align__(8) float part[kGroup * kPitchV];  // [row][rank]: this CTA's share of v
  __shared__ float factor[kGroup];
  static_assert(XP_MAX_ADAPTER_SLOTS <= INT16_MAX, "slots fit 16 bits");
  __shared__ int16_t slot[kRowsLimit];
  __shared__ uint16_t order[kRowsLimit], items[kRowsLimit];
  __shared__ int found[2];
  __shared__ int rows[kGroup];

  const bool vec_x = kVec || a.vec_x, vec_a = kVec || a.vec_a, vec_b = kVec || a.vec_b,
             vec_y = kVec || a.vec_y;
  cg::cluster_group cluster = cg::this_cluster();
  const int log2c = a.cluster_log2, C = 1 << log2c;
  const int rank = blockIdx.x & (C - 1), me = blockIdx.x >> log2c, clusters = gridDim.x >> log2c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int M = static_cast<int>(a.M);

  // The items of the batch: eight rows of an adapter at a time, each at the first
  // of them, then the rows without an adapter.  Every cluster finds them all (one
  // warp, 32 rows at a time, with the slots' rows so far in the ring) and takes
  // every so many-th.
  uint16_t *seen = reinterpret_cast<uint16_t *>(smem);
  for (int m0 = warp * 32; m0 < M; m0 += kThreads) {
    const int m = m0 + lane, s = m < M ? slot_of_row(a, m) : -2;
    const unsigned peers = __match_any_sync(kFull, s);
    if (m < M) slot[m] = static_cast<int16_t>(s);
    if (s >= 0) {  // the rows of the 32 before this one, and whether it is their last
      order[m] = static_cast<uint16_t>(__popc(peers & lanemask_lt()) | (peers >> lane == 1) << 15);
      seen[s] = 0;
    }
  }
  __syncthreads();
  if (warp == 0) {
    int leads = 0, alone = 0;
    constexpr int kAhead = 4;  // words of rows whose slots are read at once
    for (int m0 = 0; m0 < M; m0 += 32 * kAhead) {
      int s[kAhead], o[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int m = m0 + 32 * j + lane;
        s[j] = m < M ? slot[m] : -2;
        o[j] = m < M ? order[m] : 0;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int m = m0 + 32 * j + lane;
        int n = 0;  // rows of the same adapter before this one
        if (s[j] >= 0) {
          n = (o[j] & 0x7fff) + seen[s[j]];
          order[m] = static_cast<uint16_t>(n);
        }
        __syncwarp();
        if (s[j] >= 0 && o[j] >> 15) seen[s[j]] = static_cast<uint16_t>(n + 1);
        const unsigned lead = __ballot_sync(kFull, s[j] >= 0 && n % kGroup == 0);
        const unsigned none = __ballot_sync(kFull, s[j] == -1 && !a.in_place);
        if (lead >> lane & 1)
          items[leads + __popc(lead & lanemask_lt())] = static_cast<uint16_t>(m);
        if (none >> lane & 1)  // from the end
          items[kRowsLimit - 1 - alone - __popc(none & lanemask_lt())] = static_cast<uint16_t>(m);
        leads += __popc(lead);
        alone += __popc(none);
        __syncwarp();
      }
    }
    if (lane == 0) found[0] = leads, found[1] = alone;
  }
  __syncthreads();
  const int leads = found[0], n_items = leads + found[1];

  const uint32_t ring = smem_addr(smem);
  // This CTA's part of H and of N, in stages.
  const uint32_t kb = static_cast<uint32_t>((a.H + 63) / 64);
  const uint32_t nb = static_cast<uint32_t>((a.N + 15) / 16);
  const int64_t k0 = static_cast<int64_t>(kb * rank >> log2c) * 64;
  const int64_t k1 = min(a.H, static_cast<int64_t>(kb * (rank + 1) >> log2c) * 64);
  const int64_t n0 = static_cast<int64_t>(nb * rank >> log2c) * 16;
  const int64_t n1 = min(a.N, static_cast<int64_t>(nb * (rank + 1) >> log2c) * 16);
  const int first = static_cast<int>((k1 - k0 + S::kK - 1) / S::kK);
  const int chunks = first + static_cast<int>((n1 - n0 + S::kN - 1) / S::kN);
  // A thread's 16-byte pieces of a stage: a place along the rows, and every so
  // many-th row.
  constexpr int kPieces1 = S::kK / 8, kStep1 = kThreads / kPieces1;
  constexpr int kPieces2 = kRB * 2, kStep2 = kThreads / kPieces2;
  constexpr int kPiecesY = S::kN / 8;
  const int e1 = tid % kPieces1 * 8, row1 = tid / kPieces1;
  const int e2 = tid % kPieces2 * 8, row2 = tid / kPieces2;
  const int ey = tid % kPiecesY * 8, rowy = tid / kPiecesY;
  bool again = false;

  for (int item = me; item < n_items; item += clusters) {
    const int m = items[item < leads ? item : kRowsLimit - 1 - (item - leads)], s = slot[m];
    if (s < 0) {
      copy_rows<T>(a, 1, rank, C, [&](int) { return static_cast<int64_t>(m); });
      continue;  // every CTA of the cluster
    }
    if (again) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    again = true;
    int n_rows = 0;
    for (int j0 = m & ~31; j0 < M; j0 += kThreads) {
      const int j = j0 + tid;
      const int n = j < M && slot[j] == s ? order[j] - order[m] : -1;
      const bool in = n >= 0 && n < kGroup;
      if (in) rows[n] = j;
      n_rows += __syncthreads_count(in);
    }

    const T *A = static_cast<const T *>(a.a) + static_cast<int64_t>(s) * a.r * a.H;
    const T *B = static_cast<const T *>(a.b) + static_cast<int64_t>(s) * a.r * a.N;
    const T *xr = static_cast<const T *>(a.x) + rows[min(row1, n_rows - 1)] * a.x_stride + e1;
    const T *yr = static_cast<const T *>(a.y) + rows[min(rowy, n_rows - 1)] * a.y_stride + ey;
    auto clip = [](int64_t values) {
      return values >= 8 ? 16 : (values <= 0 ? 0 : static_cast<int>(values) * 2);
    };
    // kCount pieces of a thread, `step` rows apart: the first `left` rows exist, with
    // `valid` values from the piece on.
    auto fetch = [&](uint32_t at, int pitch, const T *src, int64_t stride, int left, int step,
                     int64_t valid, bool vec, auto count) {
      constexpr int kCount = decltype(count)::value;
      if (vec) {
        const int bytes = clip(valid);
#pragma unroll
        for (int j = 0; j < kCount; ++j) {
          const bool in = j * step < left;
          copy16(at + j * step * pitch, in ? src + j * step * stride : src, in ? bytes : 0);
        }
      } else {
        Words w[kCount];
#pragma unroll
        for (int j = 0; j < kCount; ++j)
          w[j] = fetch_words(src + j * step * stride, j * step < left ? valid : 0);
#pragma unroll
        for (int j = 0; j < kCount; ++j)
          store16(at + j * step * pitch,
                  join_words(w[j], place_of(src + j * step * stride),
                             j * step < left ? valid : 0));
      }
    };
    using One = std::integral_constant<int, 1>;
    auto issue = [&](int c) {
      if (c < chunks) {
        const uint32_t at = ring + (c % kRowStages) * S::kStage;
        if (c < first) {
          const int64_t k = k0 + static_cast<int64_t>(c) * S::kK;
          fetch(at + row1 * S::kPitchA + e1 * 2, S::kPitchA, A + row1 * a.H + k + e1, a.H,
                a.r - row1, kStep1, k1 - k - e1, vec_a,
                std::integral_constant<int, kR / kStep1>());
          if (row1 < kGroup)
            fetch(at + (kR + row1) * S::kPitchA + e1 * 2, 0, xr + k, 0, n_rows - row1, 1,
                  k1 - k - e1, vec_x, One());
        } else {
          const int64_t n = n0 + static_cast<int64_t>(c - first) * S::kN;
          fetch(at + row2 * S::kPitchB + e2 * 2, S::kPitchB, B + (n + row2) * a.r + e2, a.r,
                static_cast<int>(n1 - n) - row2, kStep2, a.r - e2, vec_b,
                std::integral_constant<int, S::kN / kStep2>());
          if (rowy < kGroup)
            fetch(at + S::kN * S::kPitchB + rowy * S::kPitchY + ey * 2, 0, yr + n, 0,
                  n_rows - rowy, 1, n1 - n - ey, vec_y, One());
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto arrived = [&]() {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRowStages - 2) : "memory");
      __syncthreads();
    };
#pragma unroll 1
    for (int c = 0; c < kRowStages - 1; ++c) issue(c);
    // The second product's weights come into the cache while the first one runs.
    {
      const char *p = reinterpret_cast<const char *>(B + n0 * a.r);
      const int64_t bytes = (n1 - n0) * a.r * 2;
      for (int64_t o = tid * 128; o < bytes; o += kThreads * 128)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p + o));
    }

    // v^T[rank, row]: A as the 16 rows of an instruction, x as its 8 columns.  A warp
    // has a block of 16 ranks and every kParts-th 16 values of H.
    const int block = warp % kRB, share = warp / kRB;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int c = 0; c < first; ++c) {
      arrived();
      issue(c + kRowStages - 1);
      const uint32_t at = ring + (c % kRowStages) * S::kStage;
      // A stage past the end of this CTA's part holds zeros.
#pragma unroll
      for (int i = share; i < S::kK / 16; i += kParts) {
        uint32_t p[4], q[2];
        ldmatrix4(p, at + (block * 16 + (lane & 15)) * S::kPitchA + i * 32 + (lane >> 4) * 16);
        ldmatrix2(q, at + (kR + (lane & 7)) * S::kPitchA + i * 32 + ((lane >> 3) & 1) * 16);
        Half<T>::mma(acc, p[0], p[1], p[2], p[3], q[0], q[1]);
      }
    }
    {
      float *p = red[share] + 2 * t * kPitchV + block * 16 + g;
      p[0] = acc[0], p[kPitchV] = acc[1];
      p[8] = acc[2], p[kPitchV + 8] = acc[3];
    }
    __syncthreads();
    for (int i = tid; i < kGroup * kPitchV; i += kThreads) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kParts; ++w) sum += red[w][i];
      part[i] = sum;
    }
    const float scale = a.scale ? a.scale[s] : 1.0f;
    cluster.sync();
    {
      // v, its range and its parts: a row for each warp, two neighbouring ranks a lane.
      constexpr int kEach = (kR + 63) / 64;
      float u[kEach][2], amax = 0.0f;
#pragma unroll
      for (int i = 0; i < kEach; ++i) u[i][0] = u[i][1] = 0.0f;
#pragma unroll 4
      for (int p = 0; p < C; ++p) {
        const float *q = cluster.map_shared_rank(part, p) + warp * kPitchV + 2 * lane;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if (i * 64 + 2 * lane < kR) {
            const float2 w = *reinterpret_cast<const float2 *>(q + i * 64);
            u[i][0] += w.x, u[i][1] += w.y;
          }
      }
      // The other CTAs have read this one's share when all have arrived; waited for
      // before the next item, or at the end.
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      float f = 1.0f;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        // Behind the last rank stands 0, whatever x is (an infinity times 0 is none).
        const int e = i * 64 + 2 * lane;
        u[i][0] = e < a.r ? u[i][0] * scale : 0.0f;
        u[i][1] = e + 1 < a.r ? u[i][1] * scale : 0.0f;
        if (Half<T>::kNarrowRange)
          amax = fmaxf(amax, fmaxf(finite_abs(u[i][0]), finite_abs(u[i][1])));
      }
      if constexpr (Half<T>::kNarrowRange)
        f = range_factor(__uint_as_float(__reduce_max_sync(kFull, __float_as_uint(amax))));
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (i * 64 + 2 * lane < kR) {
          uint32_t q[3];
          split<T>(u[i][0] * f, u[i][1] * f, q);
#pragma unroll
          for (int p = 0; p < 3; ++p)
            *reinterpret_cast<uint32_t *>(&vs[p][warp][i * 64 + 2 * lane]) = q[p];
        }
      if (lane == 0) factor[warp] = 1.0f / f;
    }
    __syncthreads();

    // out^T[n, row]: B as the 16 rows of an instruction, v's parts as its 8 columns.
    uint32_t v[kRB][3][2];
#pragma unroll
    for (int i = 0; i < kRB; ++i)
#pragma unroll
      for (int p = 0; p < 3; ++p)
        ldmatrix2(v[i][p], smem_addr(&vs[p][lane & 7][i * 16 + ((lane >> 3) & 1) * 8]));
    const float f0 = factor[2 * t], f1 = factor[2 * t + 1];
#pragma unroll 1
    for (int c = first; c < chunks; ++c) {
      arrived();
      issue(c + kRowStages - 1);
      unsigned char *stage = smem + (c % kRowStages) * S::kStage;
      const uint32_t at = smem_addr(stage);
      unsigned char *ys = stage + S::kN * S::kPitchB;
      const int64_t n = n0 + static_cast<int64_t>(c - first) * S::kN;
#pragma unroll 1
      for (int b = warp * 16; b < S::kN && n + b < n1; b += kWarps * 16) {
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kRB; ++i) {
          uint32_t p[4];
          ldmatrix4(p, at + (b + (lane & 15)) * S::kPitchB + i * 32 + (lane >> 4) * 16);
#pragma unroll
          for (int q = 0; q < 3; ++q)
            Half<T>::mma(d, p[0], p[1], p[2], p[3], v[i][q][0], v[i][q][1]);
        }
        // y + update in place of y in the stage, then 16-byte pieces of out.
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          T *p = reinterpret_cast<T *>(ys + (2 * t + (j & 1)) * S::kPitchY) + b + g + (j >> 1) * 8;
          if (2 * t + (j & 1) < n_rows) narrow(p, widen(*p) + d[j] * (j & 1 ? f1 : f0));
        }
        __syncwarp();
        const int row = lane >> 1, e = b + (lane & 1) * 8;
        if (row < n_rows)
          put8(static_cast<T *>(a.out) + rows[row] * a.out_stride + n + e,
               *reinterpret_cast<const uint4 *>(ys + row * S::kPitchY + e * 2), n1 - n - e, vec_y);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the ring and the rows are free for the next item
  }
  if (again) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- long batches ----

// Sorts the rows by slot and cuts each slot's rows into tiles: one cluster, a run of
// rows for each CTA; the CTAs' counts go through distributed shared memory.  The
// order of a slot's rows is free: a row's result does not depend on its tile.
__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads)
    plan_kernel(const __grid_constant__ LowRankArgs a) {
  // Each [slots + 1]: rows of this CTA; the next free place; rows of all CTAs.
  extern __shared__ int counts[];
  __shared__ int sum_rows[32], sum_tiles[32];
  // The tiles' kernel may be set up meanwhile (it waits for this one's end).
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = a.slots + 1, M = static_cast<int>(a.M);  // the last: rows without an adapter
  int *place = counts + n, *total = place + n;
  const int per = (M + kPlanCtas - 1) / kPlanCtas, first = min(rank * per, M),
            last = min(first + per, M);
  for (int i = tid; i < n; i += kPlanThreads) counts[i] = 0;
  // Four rows of a thread at a time: their ids (and map entries) come together.
  constexpr int kBatch = 4;
  auto slots_of = [&](int m0, int (&s)[kBatch]) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int m = m0 + j * kPlanThreads + lane;
      s[j] = -2;
      if (m < last) {
        s[j] = slot_of_row(a, m);
        if (s[j] < 0) s[j] = a.slots;
      }
    }
  };
  auto count = [&](const int (&s)[kBatch]) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const unsigned peers = __match_any_sync(kFull, s[j]);
      if (s[j] >= 0 && lane == __ffs(peers) - 1) atomicAdd(&counts[s[j]], __popc(peers));
    }
  };
  auto put = [&](int m0, const int (&s)[kBatch]) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const unsigned peers = __match_any_sync(kFull, s[j]);
      const int leader = __ffs(peers) - 1;
      int at = 0;
      if (s[j] >= 0 && lane == leader) at = atomicAdd(&place[s[j]], __popc(peers));
      at = __shfl_sync(kFull, at, leader) + __popc(peers & lanemask_lt());
      if (s[j] >= 0) a.perm[at] = m0 + j * kPlanThreads + lane;
    }
  };
  // The first batch's slots stay in registers; only longer runs are read again.
  const int mine = first + warp * 32;
  int s0[kBatch];
  slots_of(mine, s0);
  __syncthreads();
  count(s0);
  for (int m0 = mine + kBatch * kPlanThreads; m0 < last; m0 += kBatch * kPlanThreads) {
    int s[kBatch];
    slots_of(m0, s);
    count(s);
  }
  cluster.sync();
  // Exclusive sums over the slots, a run of slots per thread; every CTA has its own.
  const int run = (n + kPlanThreads - 1) / kPlanThreads, i0 = min(tid * run, n),
            i1 = min(i0 + run, n);
  int rows = 0, tiles = 0;
  for (int i = i0; i < i1; ++i) {
    int c[kPlanCtas], all = 0, before = 0;
#pragma unroll
    for (int b = 0; b < kPlanCtas; ++b) c[b] = cluster.map_shared_rank(counts, b)[i];
#pragma unroll
    for (int b = 0; b < kPlanCtas; ++b) {
      if (b == rank) before = all;
      all += c[b];
    }
    place[i] = before;  // of the slot's rows, those of the CTAs before this one
    total[i] = all;
    rows += all;
    if (i < a.slots || !a.in_place) tiles += (all + kTile - 1) / kTile;
  }
  // The counts stay until all have read them; waited for at the end.
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
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
    const int all = total[i];
    if (rank == 0 && (i < a.slots || !a.in_place))
      for (int o = 0; o < all; o += kTile)
        a.tiles[tiles_before++] =
            make_int4(i < a.slots ? i : -1, rows_before + o, min(kTile, all - o), 0);
    place[i] += rows_before;
    rows_before += all;
  }
  if (rank == 0 && tid == kPlanThreads - 1) *a.ntiles = tiles_before;
  __syncthreads();
  put(mine, s0);
  for (int m0 = mine + kBatch * kPlanThreads; m0 < last; m0 += kBatch * kPlanThreads) {
    int s[kBatch];
    slots_of(m0, s);
    put(m0, s);
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// mbarriers.  A wait gives up after its limit or when another one of the block has: it then
// sets *failed.  A block with such a wait adds 1 to wait_errors.
constexpr uint32_t kWaitNs = 2000000000u;
constexpr int kFreePolls = 16;        // tries before the time is looked at
constexpr uint32_t kTryNs = 1000000;  // a try may be suspended for

__device__ uint32_t wait_errors;
std::atomic<uint32_t> wait_limit{kWaitNs};

__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Arrives at the barrier at the same place in another CTA of the cluster.
__device__ __forceinline__ void bar_arrive_peer(uint32_t bar, int cta) {
  asm volatile(
      "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, %1;\n\t"
      "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n\t}" ::"r"(bar),
      "r"(cta)
      : "memory");
}

template <bool kCluster = false>
__device__ __forceinline__ bool bar_wait(uint32_t bar, int parity, uint32_t limit,
                                         volatile int *failed) {
  uint64_t since = 0;
  const uint32_t hint = min(limit, kTryNs);
  for (int i = limit ? 0 : kFreePolls;; ++i) {  // without a limit in time: a single try
    uint32_t done;
    if constexpr (kCluster)
      asm volatile(
          "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], "
          "%2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done)
          : "r"(bar), "r"(parity), "r"(hint)
          : "memory");
    else
      asm volatile(
          "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done)
          : "r"(bar), "r"(parity), "r"(hint)
          : "memory");
    if (done) return true;
    if (i < kFreePolls) continue;
    const uint64_t now = global_ns();
    if (i == kFreePolls) since = now;
    if (*failed || now - since >= limit) break;
  }
  *failed = 1;
  return false;
}

__device__ __forceinline__ void fence_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// The barrier completes when the matrix instructions issued so far have.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}

// Operand in shared memory: rows of 128 bytes along the summed axis, 16-byte pieces
// exchanged within 8 rows (128-byte swizzle), 1024 bytes from 8 rows to the next 8.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (1ull << 16) | (64ull << 32) |
         (1ull << 46) | (2ull << 61);
}

// d[128, N] (+)= a[128, 16] b[N, 16]^T, 32-bit sums in tensor memory, both operands in
// shared memory.
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t what,
                                       bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(what), "r"(static_cast<uint32_t>(add))
      : "memory");
}

// The same with a in tensor memory: a lane for each row, two neighbouring values a column.
__device__ __forceinline__ void tc_mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t what,
                                            bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(what), "r"(static_cast<uint32_t>(add))
      : "memory");
}

// Eight columns of this thread's row of tensor memory.
__device__ __forceinline__ void tc_store8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}

// This thread's row of tensor memory, 16 columns.
__device__ __forceinline__ void tc_load16(float (&v)[16], uint32_t addr) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Byte of 16-byte piece `piece` of row `row` in a swizzled block of 128-byte rows.
__device__ __forceinline__ int swizzled(int row, int piece) {
  return row * 128 + ((piece ^ (row & 7)) << 4);
}

constexpr int kOutWarps = 8;                 // half a row of the tile for each thread
constexpr int kMmaWarp = kOutWarps;          // issues the matrix instructions
constexpr int kLoadWarps = 4;
constexpr int kLoaders = kLoadWarps * 32;
constexpr int kShiftWarps = 4;               // where rows lie at any place
constexpr int kNBlock = 64;                  // columns of out in a stage
// Blocks of 64 of H that are not split.  Measured with 2048 columns, 6 adapters in 8 slots
// (us, whole / split): rank 16, 1100 rows, H 512 14.1 / 17.0, 768 15.3 / 17.4; 2048 rows, 256
// 15.6 / 17.0, 512 17.5 / 17.2, 768 19.0 / 17.4, 1024 20.6 / 18.0; 4096 rows, 256 22.9 / 23.7,
// 512 26.2 / 24.5, 768 29.4 / 25.2, 1024 33.1 / 25.9; rank 64, H 512, 1100 rows 15.9 / 21.3,
// 2048 20.3 / 21.8, 4096 29.7 / 27.5.  Few rows bear a longer whole H than many.
constexpr uint32_t kWholeBlocks = 12;
// Tensor memory: v's sums, and when they have been read two blocks of out in their place;
// behind them v's parts, two values a column.  All parts are there, none in shared memory:
// an instruction with an operand from tensor memory does not wait for one before it that
// takes both from shared memory, on the same sum (the product of the last of those was lost).
constexpr int kTmemV = 128;
constexpr int tmem_cols(int blocks) { return blocks <= 4 ? 256 : 512; }
constexpr int kWholeSm = 208 * 1024;         // shared memory that leaves no room for another CTA
constexpr int tile_threads(bool vec) {
  return (kOutWarps + 1 + kLoadWarps + (vec ? 0 : kShiftWarps)) * 32;
}

// kRB: blocks of 16 ranks.  kAtoms: 128-byte rows that hold a row of ranks.
template <int kRB, bool kVec, bool kDeep>
struct TileSmem {
  static constexpr int kR = kRB * 16;
  static constexpr int kAtoms = kR > 64 ? 2 : 1;
  static constexpr int kStages = kDeep ? (kRB <= 4 ? 6 : 4) : (kVec || kRB <= 4 ? 3 : 2);
  // A stage holds 128 rows x 64 values of x and kR x 64 of A, or 64 rows of B and 128 x 64 of y.
  static constexpr int kA = kTile * 128;
  static constexpr int kY = kAtoms * kNBlock * 128;
  static constexpr int kFirst = kA + kR * 128, kSecond = kY + kTile * 128;
  static constexpr int kStage = ((kFirst > kSecond ? kFirst : kSecond) + 1023) / 1024 * 1024;
  static constexpr int kShare = kR * kTile * 4;  // this CTA's share of v
  // Rows at any place come as the aligned 16-byte words around them, one more than
  // the stage's row has; shifting them fills the stage.
  static constexpr int kWords = kVec ? 0 : (kRB <= 4 ? 4 : 2);  // such stages
  static constexpr int kPitch = 128 + 16, kPitchB = kR * 2 + 16;
  static constexpr int kWordsA = kTile * kPitch, kWordsY = kNBlock * kPitchB;
  static constexpr int kWords1 = kWordsA + kR * kPitch, kWords2 = kWordsY + kTile * kPitch;
  static constexpr int kWordsStage = kWords1 > kWords2 ? kWords1 : kWords2;
  static constexpr int kBytes = 1024 + kStages * kStage + kShare + kWords * kWordsStage;
};

// kVec: all rows allow 16-byte accesses; else four more warps shift what the loading
// warps bring.  kDeep: twice the stages, one CTA on an SM.
template <typename T, int kRB, bool kVec, bool kDeep>
__global__ void __launch_bounds__(tile_threads(kVec), kVec && kRB <= 4 && !kDeep ? 2 : 1)
    tile_kernel(const __grid_constant__ LowRankArgs a) {
  using S = TileSmem<kRB, kVec, kDeep>;
  constexpr int kStages = S::kStages;
  const bool vec_y = kVec || a.vec_y;
  extern __shared__ unsigned char raw[];
  __shared__ int64_t rows[kTile];
  __shared__ __align__(8) uint64_t bars[3 * kStages + 8 + 2 * S::kWords];
  // Not kVec: where a row's first value lies in its words (bytes), and in the upper
  // half the bits to shift by; the rows' first values of out in this CTA's part.
  __shared__ uint32_t at_x[kVec ? 1 : kTile], at_y[kVec ? 1 : kTile], at_a[kVec ? 1 : S::kR],
      at_b[kVec ? 1 : kNBlock];
  __shared__ uint16_t *out_row[kVec ? 1 : kTile];
  __shared__ uint4 carry[kVec ? 1 : kTile];  // the last eight values of the block before
  __shared__ float amax[2][kTile];
  __shared__ uint32_t tmem_at;
  __shared__ int failed;

  cg::cluster_group cluster = cg::this_cluster();
  const int log2c = a.cluster_log2, C = 1 << log2c, rank = blockIdx.x & (C - 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = blockIdx.x >> log2c;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the plan's end
  if (tile >= *a.ntiles) return;
  const int4 job = a.tiles[tile];
  const int s = job.x, n_rows = job.z;
  unsigned char *smem =
      raw + ((1024 - (static_cast<uint32_t>(__cvta_generic_to_shared(raw)) & 1023)) & 1023);
  const uint32_t ring = smem_addr(smem);
  // Stage filled; stage free after the first / the second product; v in tensor
  // memory; v's parts there; a block of out there, and read from it; the cluster's
  // shares of v written; all matrix instructions over; words arrived, and shifted.
  const uint32_t full = smem_addr(bars), free1 = full + 8 * kStages, free2 = free1 + 8 * kStages;
  const uint32_t v_done = free2 + 8 * kStages, v_ready = v_done + 8, out_done = v_ready + 8,
                 out_read = out_done + 16, shares = out_read + 16, drained = shares + 8,
                 words_full = drained + 8, words_free = words_full + 8 * S::kWords;
  volatile int *fail = &failed;

  if (tid < kTile) rows[tid] = a.perm[job.y + min(tid, n_rows - 1)];
  if (s < 0) {
    __syncthreads();
    copy_rows<T>(a, n_rows, rank, C, [&](int i) { return rows[i]; });
    return;  // every CTA of the cluster
  }
  if (tid == 0) {
    failed = 0;
    for (int i = 0; i < kStages; ++i) {
      bar_init(full + 8 * i, kLoaders);
      bar_init(free1 + 8 * i, 1);
      bar_init(free2 + 8 * i, kOutWarps);
    }
    bar_init(v_done, 1);
    bar_init(v_ready, kOutWarps * 32);
    for (int i = 0; i < 2; ++i) {
      bar_init(out_done + 8 * i, 1);
      bar_init(out_read + 8 * i, kOutWarps * 32);
    }
    bar_init(shares, C);
    bar_init(drained, 1);
    for (int i = 0; i < S::kWords; ++i) {
      bar_init(words_full + 8 * i, kLoaders);
      bar_init(words_free + 8 * i, kLoaders);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&tmem_at)),
                 "n"(tmem_cols(kRB))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tc_fence_before();
  }
  // A short H is not worth the exchange of shares: every CTA sums all of it.
  const uint32_t kb_all = static_cast<uint32_t>((a.H + 63) / 64);
  const bool shared_v = C > 1 && kb_all > kWholeBlocks;
  if (shared_v)
    cluster.sync();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;

  const T *A = static_cast<const T *>(a.a) + static_cast<int64_t>(s) * a.r * a.H;
  const T *B = static_cast<const T *>(a.b) + static_cast<int64_t>(s) * a.r * a.N;
  // This CTA's blocks of 64 along H (where it is split there are more than CTAs) and along N
  // (there may be none).
  const uint32_t nb_all = static_cast<uint32_t>((a.N + kNBlock - 1) / kNBlock);
  const int k0 = shared_v ? kb_all * rank >> log2c : 0;
  const int k1 = shared_v ? kb_all * (rank + 1) >> log2c : kb_all;
  const int n0 = nb_all * rank >> log2c, n1 = nb_all * (rank + 1) >> log2c;
  const int first = k1 - k0, chunks = first + n1 - n0;
  const int k_steps = (a.r + 15) / 16;  // of the second product
  if constexpr (!kVec) {
    // Blocks are whole words apart, so these hold for every block.
    auto place = [](const T *row, int pitch, int i) {
      const int off = place_of(row);
      return static_cast<uint32_t>(i * pitch + (off & 12)) | (off & 2 ? 16u << 16 : 0u);
    };
    if (tid < kTile) {
      at_x[tid] = place(static_cast<const T *>(a.x) + rows[tid] * a.x_stride, S::kPitch, tid);
      at_y[tid] = place(static_cast<const T *>(a.y) + rows[tid] * a.y_stride, S::kPitch, tid);
      out_row[tid] = static_cast<uint16_t *>(a.out) + rows[tid] * a.out_stride +
                     static_cast<int64_t>(n0) * kNBlock;
    }
    if (tid < S::kR) at_a[tid] = place(A + tid * a.H, S::kPitch, tid);
    if (tid < kNBlock) at_b[tid] = place(B + tid * a.r, S::kPitchB, tid);
    __syncthreads();
  }

  if (warp > kMmaWarp) {
    // Loading: a thread has one 16-byte piece of every 16th row.
    const int p = (tid - (kMmaWarp + 1) * 32) % kLoaders, piece = p & 7, row0 = p >> 3;
    const int mine = (n_rows - row0 + 15) / 16;  // rows of the tile of this thread
    const int ranks = a.r - row0;                // rows of A from this thread's first on
    constexpr int kEach = kTile / 16;
    const int64_t k_at = static_cast<int64_t>(k0) * 64, n_at = static_cast<int64_t>(n0) * kNBlock;
    // Waits until the stage of chunk c is free; its place, 0 after a wait gave up.
    auto begin = [&](int c) {
      const int stage = c % kStages, use = c / kStages;
      if (use > 0) {
        const int before = (first + kStages - 1 - stage) / kStages;  // uses by the first product
        const bool ok = c - kStages < first
                            ? bar_wait(free1 + 8 * stage, (use - 1) & 1, a.wait_ns, fail)
                            : bar_wait(free2 + 8 * stage, (use - 1 - before) & 1, a.wait_ns, fail);
        if (!ok) return 0u;
      }
      return ring + stage * S::kStage;
    };
    auto arrive_async = [](uint32_t bar) {
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
    };
    if constexpr (kVec) {
      const uint32_t at0 = swizzled(row0, piece);
      auto clip = [](int64_t values) {  // bytes of a piece of which `values` are left
        return values >= 8 ? 16 : (values <= 0 ? 0 : static_cast<int>(values) * 2);
      };
      bool ok = true;
      {
        const T *src[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j)
          src[j] = static_cast<const T *>(a.x) + (j < mine ? rows[row0 + 16 * j] : 0) * a.x_stride +
                   k_at + piece * 8;
        const T *w = A + row0 * a.H + k_at + piece * 8;
        int64_t left = a.H - k_at - piece * 8;
        for (int c = 0; c < first; ++c, w += 64, left -= 64) {
          uint32_t at = begin(c);
          if (!at) {
            ok = false;
            break;
          }
          at += at0;
          const int bytes = clip(left);
#pragma unroll
          for (int j = 0; j < kEach; ++j) {
            if (j < mine) copy16(at + j * 2048, src[j], bytes);
            src[j] += 64;
          }
#pragma unroll
          for (int j = 0; j < kRB; ++j)
            copy16(at + S::kA + j * 2048, 16 * j < ranks ? w + j * 16 * a.H : A,
                   16 * j < ranks ? bytes : 0);
          arrive_async(full + 8 * (c % kStages));
        }
      }
      if (ok) {
        const T *src[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j)
          src[j] = static_cast<const T *>(a.y) + (j < mine ? rows[row0 + 16 * j] : 0) * a.y_stride +
                   n_at + piece * 8;
        for (int c = first; c < chunks; ++c) {
          uint32_t at = begin(c);
          if (!at) break;
          at += at0;
          const int64_t n = static_cast<int64_t>(n0 + c - first) * kNBlock;
#pragma unroll
          for (int q = 0; q < S::kAtoms; ++q) {
            const int e = q * 64 + piece * 8;
            if (e >= S::kR) continue;
            const T *w = B + (n + row0) * a.r + e;
            const int64_t left = a.N - n - row0;
            const int bytes = clip(a.r - e);
#pragma unroll
            for (int j = 0; j < kNBlock / 16; ++j)
              copy16(at + q * kNBlock * 128 + j * 2048, 16 * j < left ? w + j * 16 * a.r : B,
                     16 * j < left ? bytes : 0);
          }
          const int bytes = clip(a.N - n - piece * 8);
#pragma unroll
          for (int j = 0; j < kEach; ++j) {
            if (j < mine) copy16(at + S::kY + j * 2048, src[j], bytes);
            src[j] += kNBlock;
          }
          arrive_async(full + 8 * (c % kStages));
        }
      }
    } else if (warp <= kMmaWarp + kLoadWarps) {
      // Words: the eight of a thread's rows that begin at its piece, and the ninth of
      // one row.  A word is read where it holds a value of the row.
      const uint32_t words = ring + kStages * S::kStage + S::kShare;
      auto begin_words = [&](int c) {
        const int stage = c % S::kWords, use = c / S::kWords;
        if (use > 0 && !bar_wait(words_free + 8 * stage, (use - 1) & 1, a.wait_ns, fail)) return 0u;
        return words + stage * S::kWordsStage;
      };
      // `bytes`: of the row's values from the block on.
      auto word = [](uint32_t dst, const T *row, int i, int64_t bytes) {
        const int off = place_of(row);
        copy16(dst, reinterpret_cast<const char *>(row) - off + i * 16,
               i * 16 - off < bytes ? 16 : 0);
      };
      // The words of up to eight rows of x or y: kept as addresses, and the rows'
      // places in their first words (four bits each).
      const char *src[kEach], *ninth;
      uint32_t offs = 0;
      int off9 = 0;
      auto aim = [&](const T *base, int64_t stride) {
        offs = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          const T *row = base + (j < mine ? rows[row0 + 16 * j] : 0) * stride;
          offs |= static_cast<uint32_t>(place_of(row)) << (4 * j);
          src[j] = reinterpret_cast<const char *>(row) - place_of(row) + piece * 16;
        }
        const T *row = base + (p < n_rows ? rows[p] : 0) * stride;
        off9 = place_of(row);
        ninth = reinterpret_cast<const char *>(row) - off9 + 128;
      };
      auto fetch = [&](uint32_t at, int bytes) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          if (j < mine)
            copy16(at + (row0 + 16 * j) * S::kPitch + piece * 16, src[j],
                   piece * 16 - static_cast<int>(offs >> (4 * j) & 15) < bytes ? 16 : 0);
          src[j] += 128;
        }
        if (p < n_rows) copy16(at + p * S::kPitch + 128, ninth, 128 - off9 < bytes ? 16 : 0);
        ninth += 128;
      };
      bool ok = true;
      aim(static_cast<const T *>(a.x) + k_at, a.x_stride);
      for (int c = 0; c < first; ++c) {
        const uint32_t at = begin_words(c);
        ok = at != 0;
        if (!ok) break;
        const int64_t k = k_at + static_cast<int64_t>(c) * 64;
        const int bytes = static_cast<int>(min(a.H - k, static_cast<int64_t>(64))) * 2;
        fetch(at, bytes);
#pragma unroll
        for (int j = 0; j < kRB; ++j)
          if (16 * j < ranks)
            word(at + S::kWordsA + (row0 + 16 * j) * S::kPitch + piece * 16,
                 A + (row0 + 16 * j) * a.H + k, piece, bytes);
        if (p < a.r) word(at + S::kWordsA + p * S::kPitch + 128, A + p * a.H + k, 8, bytes);
        arrive_async(words_full + 8 * (c % S::kWords));
      }
      aim(static_cast<const T *>(a.y) + n_at, a.y_stride);
      for (int c = first; c < chunks && ok; ++c) {
        const uint32_t at = begin_words(c);
        if (!at) break;
        const int64_t n = n_at + static_cast<int64_t>(c - first) * kNBlock;
        constexpr int kEachB = kRB * 2 + 1;  // words of a row of B
        for (int i = p; i < kNBlock * kEachB; i += kLoaders) {
          const int row = i / kEachB, j = i % kEachB;
          if (n + row < a.N)
            word(at + row * S::kPitchB + j * 16, B + (n + row) * a.r, j, a.r * 2);
        }
        fetch(at + S::kWordsY,
              static_cast<int>(min(a.N - n, static_cast<int64_t>(kNBlock))) * 2);
        arrive_async(words_full + 8 * (c % S::kWords));
      }
    } else {
      // Shifting, from the words to a stage: two values a lane, a row of 64 for a warp
      // (whole rows of shared memory, no two lanes at one bank).
      const unsigned char *words = smem + kStages * S::kStage + S::kShare;
      const int sw = p >> 5;
      // Values 2 i and 2 i + 1 of the row at `place` (see above).
      auto two = [](const unsigned char *src, uint32_t place, int i) {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(src + (place & 0xffff)) + i;
        return __funnelshift_r(w[0], w[1], place >> 16);
      };
      // Of two values those of which `valid` from the first on exist.
      auto keep = [](int64_t valid) { return valid >= 2 ? ~0u : (valid == 1 ? 0xffffu : 0u); };
      auto put2 = [](uint32_t at, uint32_t v) {
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
      };
      // A lane's place in rows of this warp (row % 8 is sw or sw + 4).
      const uint32_t lane_at[2] = {
          static_cast<uint32_t>(swizzled(sw, lane >> 2) + (lane & 3) * 4),
          static_cast<uint32_t>(swizzled(sw + 4, lane >> 2) + (lane & 3) * 4 - 512)};
      // Rows sw, sw + 4, ... of x or y, eight at a time (the last eight may run past
      // n_rows: rows of the stage that nothing reads).
      auto shift_rows = [&](uint32_t at, const unsigned char *src, const uint32_t *place,
                            int count, uint32_t mask) {
#pragma unroll 1
        for (int j0 = 0; 4 * j0 < count; j0 += 8) {
          uint32_t v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = two(src, place[sw + 4 * (j0 + j)], lane) & mask;
#pragma unroll
          for (int j = 0; j < 8; ++j) put2(at + lane_at[j & 1] + (j0 + j) * 512, v[j]);
        }
      };
      for (int c = 0; c < chunks; ++c) {
        const int stage = c % S::kWords;
        if (!bar_wait(words_full + 8 * stage, (c / S::kWords) & 1, a.wait_ns, fail)) break;
        const uint32_t at = begin(c);
        if (!at) break;
        const unsigned char *from = words + stage * S::kWordsStage;
        if (c < first) {
          const uint32_t mask = keep(a.H - k_at - static_cast<int64_t>(c) * 64 - 2 * lane);
          shift_rows(at, from, at_x, n_rows, mask);
#pragma unroll
          for (int j0 = 0; j0 < S::kR / 4; j0 += 4) {
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int row = sw + 4 * (j0 + j);
              v[j] = row < a.r ? two(from + S::kWordsA, at_a[row], lane) & mask : 0u;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) put2(at + S::kA + lane_at[j & 1] + (j0 + j) * 512, v[j]);
          }
        } else {
          const int64_t n = n_at + static_cast<int64_t>(c - first) * kNBlock;
          constexpr int kTwos = kRB * 8;  // of a row of B
#pragma unroll 1
          for (int i0 = p; i0 < kNBlock * kTwos; i0 += 4 * kLoaders) {
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int row = (i0 + j * kLoaders) / kTwos, e = (i0 + j * kLoaders) % kTwos;
              v[j] = n + row < a.N ? two(from, at_b[row], e) & keep(a.r - 2 * e) : 0u;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int row = (i0 + j * kLoaders) / kTwos, e = (i0 + j * kLoaders) % kTwos;
              put2(at + e / 32 * kNBlock * 128 + swizzled(row, e % 32 >> 2) + (e & 3) * 4, v[j]);
            }
          }
          shift_rows(at + S::kY, from + S::kWordsY, at_y, n_rows, keep(a.N - n - 2 * lane));
        }
        fence_async_proxy();
        bar_arrive(full + 8 * (c % kStages));
        bar_arrive(words_free + 8 * stage);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kMmaWarp) {
    if (lane == 0) {
      constexpr uint32_t kType = Half<T>::kNarrowRange ? 0u : (1u << 7) | (1u << 10);
      constexpr uint32_t kWhat = (1u << 4) | kType | (8u << 24);  // 32-bit sums, 128 rows
      constexpr uint32_t kWhat1 = kWhat | (static_cast<uint32_t>(S::kR / 8) << 17);
      constexpr uint32_t kWhat2 = kWhat | (static_cast<uint32_t>(kNBlock / 8) << 17);
      bool ok = true;
      for (int c = 0; c < first && ok; ++c) {
        const int stage = c % kStages;
        ok = bar_wait(full + 8 * stage, (c / kStages) & 1, a.wait_ns, fail);
        if (!ok) break;
        fence_async_proxy();
        tc_fence_after();
        const uint32_t at = ring + stage * S::kStage;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tc_mma(tmem, operand(at + 32 * i), operand(at + S::kA + 32 * i), kWhat1, c > 0 || i > 0);
        tc_commit(free1 + 8 * stage);
      }
      if (ok) tc_commit(v_done);
      ok = ok && bar_wait(v_ready, 0, a.wait_ns, fail);
      for (int c = first; c < chunks && ok; ++c) {
        const int stage = c % kStages, i = c - first, half = i & 1;
        ok = bar_wait(full + 8 * stage, (c / kStages) & 1, a.wait_ns, fail) &&
             (i < 2 || bar_wait(out_read + 8 * half, (i / 2 - 1) & 1, a.wait_ns, fail));
        if (!ok) break;
        fence_async_proxy();
        tc_fence_after();
        const uint32_t at = ring + stage * S::kStage, d = tmem + half * kNBlock;
        // A lone thread issues these: places are constants added to one descriptor (with
        // each computed anew 16384 rows of rank 64 took 60 us, not 52).
        const uint64_t b_at = operand(at);
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
          for (int j = 0; j < kRB; ++j) {
            if (j >= k_steps) break;
            tc_mma_tmem(d, tmem + kTmemV + (part * kRB + j) * 8,
                        b_at + ((j / 4) * kNBlock * 128 + 32 * (j % 4)) / 16, kWhat2,
                        part + j > 0);
          }
        tc_commit(out_done + 8 * half);
      }
      // What has been issued reads and writes memory that is given back below, though the
      // warps that wait for its results may have given up.
      volatile int never = 0;
      tc_commit(drained);
      bar_wait(drained, 0, kWaitNs, &never);
    }
    __syncwarp();
  } else {
    // Half a row of the tile for each thread (a warp reaches the 32 rows of tensor
    // memory that its number gives).
    const int row = tid & 127, side = warp >> 2;
    const uint32_t my_tmem = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float scale = a.scale ? a.scale[s] : 1.0f;
    bool ok = __all_sync(kFull, bar_wait(v_done, 0, a.wait_ns, fail));
    tc_fence_after();
    constexpr int kMine = (kRB + 1) / 2;  // blocks of 16 ranks: every other one is this side's
    float u[kMine][16];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
#pragma unroll
      for (int j = 0; j < 16; ++j) u[i][j] = 0.0f;
      if (ok && 2 * i + side < kRB) tc_load16(u[i], my_tmem + (2 * i + side) * 16);
    }
    if (shared_v) {
      // The cluster's shares of v, added in the order of its CTAs.  Four ranks of all
      // rows together, so that a warp reads 512 bytes in a row.
      float4 *share = reinterpret_cast<float4 *>(smem + kStages * S::kStage) + row;
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        if (2 * i + side < kRB) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            share[((2 * i + side) * 4 + j) * kTile] =
                make_float4(u[i][4 * j], u[i][4 * j + 1], u[i][4 * j + 2], u[i][4 * j + 3]);
            u[i][4 * j] = u[i][4 * j + 1] = u[i][4 * j + 2] = u[i][4 * j + 3] = 0.0f;
          }
        }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (ok && tid < C) {
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        bar_arrive_peer(shares, tid);
      }
      ok = __all_sync(kFull, ok && bar_wait<true>(shares, 0, a.wait_ns, fail));
      if (ok) {
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if (2 * i + side < kRB) {
            for (int b = 0; b < C; b += 2) {  // C is even here
              float4 q[2][4];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float4 *p =
                    (b + h == rank ? share : cluster.map_shared_rank(share, b + h)) +
                    (2 * i + side) * 4 * kTile;
#pragma unroll
                for (int j = 0; j < 4; ++j) q[h][j] = p[j * kTile];
              }
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  u[i][4 * j] += q[h][j].x, u[i][4 * j + 1] += q[h][j].y;
                  u[i][4 * j + 2] += q[h][j].z, u[i][4 * j + 3] += q[h][j].w;
                }
            }
          }
      }
    }
    float f = 1.0f;
    // Behind the last rank stands 0, whatever x is (an infinity times 0 is none).
#pragma unroll
    for (int i = 0; i < kMine; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        u[i][j] = (2 * i + side) * 16 + j < a.r ? u[i][j] * scale : 0.0f;
    if constexpr (Half<T>::kNarrowRange) {
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < kMine; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) most = fmaxf(most, finite_abs(u[i][j]));
      amax[side][row] = most;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      f = range_factor(fmaxf(amax[0][row], amax[1][row]));
    }
    const float back = 1.0f / f;
    if (ok) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (2 * i + side >= kRB) continue;
        uint32_t q[3][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t w[3];
          split<T>(u[i][2 * j] * f, u[i][2 * j + 1] * f, w);
          q[0][j] = w[0], q[1][j] = w[1], q[2][j] = w[2];
        }
#pragma unroll
        for (int p = 0; p < 3; ++p)
          tc_store8(my_tmem + kTmemV + (p * kRB + 2 * i + side) * 8, q[p]);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      bar_arrive(v_ready);
    }
    // After a wait gave up, warps that meet others at a barrier still do.
    for (int c = first; c < chunks && (ok || !vec_y); ++c) {
      const int stage = c % kStages, i = c - first, half = i & 1;
      ok = __all_sync(kFull, ok && bar_wait(out_done + 8 * half, (i / 2) & 1, a.wait_ns, fail) &&
                                 bar_wait(full + 8 * stage, (c / kStages) & 1, a.wait_ns, fail));
      if (!ok && vec_y) break;
      tc_fence_after();
      unsigned char *ys = smem + stage * S::kStage + S::kY;
      // y + update in place of y in the stage, then whole 16-byte pieces of out.
#pragma unroll
      for (int j = 2 * side; j < 2 * side + 2; ++j) {
        if (!ok) continue;
        uint4 q[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          q[h] = *reinterpret_cast<const uint4 *>(ys + swizzled(row, 2 * j + h));
        float d[16];
        tc_load16(d, my_tmem + half * kNBlock + j * 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 w = Half<T>::unpack((&q[h].x)[e]);
            (&q[h].x)[e] = Half<T>::pack(w.x + d[h * 8 + 2 * e] * back,
                                         w.y + d[h * 8 + 2 * e + 1] * back);
          }
          *reinterpret_cast<uint4 *>(ys + swizzled(row, 2 * j + h)) = q[h];
        }
      }
      tc_fence_before();
      if (ok) bar_arrive(out_read + 8 * half);
      const int64_t n = static_cast<int64_t>(n0 + i) * kNBlock;
      if (vec_y) {
        __syncwarp();
        const int piece = side * 4 + (lane & 3);
        uint4 q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          q[j] = *reinterpret_cast<const uint4 *>(
              ys + swizzled((warp & 3) * 32 + j * 8 + (lane >> 2), piece));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = (warp & 3) * 32 + j * 8 + (lane >> 2);
          if (r < n_rows)
            put8(static_cast<T *>(a.out) + rows[r] * a.out_stride + n + piece * 8, q[j],
                 a.N - n - piece * 8, true);
        }
      } else {
        // Rows at any place: the aligned 16-byte words of out, each from two
        // neighbouring pieces of a row (the first from the end of the block before);
        // both sides' columns together.
        asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");
        const int left = static_cast<int>(min(a.N - n, static_cast<int64_t>(kNBlock)));
        const int piece = lane & 7, r0 = (warp & 3) * 32 + side * 16 + (lane >> 3);
        if (ok) {
          Words w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = r0 + 4 * j;
            w[j].hi = *reinterpret_cast<const uint4 *>(ys + swizzled(r, piece));
            w[j].lo = piece ? *reinterpret_cast<const uint4 *>(ys + swizzled(r, piece - 1 & 7))
                            : carry[r];
          }
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = r0 + 4 * j;
            if (r >= n_rows) break;
            if (piece == 7) carry[r] = w[j].hi;
            uint16_t *o = out_row[r] + static_cast<int64_t>(i) * kNBlock;
            const int off = place_of(o), e0 = piece * 8 - off / 2;  // the word's first value
            const uint4 q = off ? join_words(w[j], 16 - off, 8) : w[j].hi;
            if ((e0 >= 0 || i > 0) && e0 + 8 <= left) {
              *reinterpret_cast<uint4 *>(o + e0) = q;
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if ((e0 + e >= 0 || i > 0) && e0 + e < left)
                  o[e0 + e] = static_cast<uint16_t>((&q.x)[e >> 1] >> (16 * (e & 1)));
            }
            if (piece == 7 && c == chunks - 1) {  // what is left behind the last word
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (56 + e >= e0 + 8 && 56 + e < left)
                  o[56 + e] = static_cast<uint16_t>((&w[j].hi.x)[e >> 1] >> (16 * (e & 1)));
            }
          }
        }
        asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");
      }
      __syncwarp();
      if (ok && lane == 0) bar_arrive(free2 + 8 * stage);
    }
  }
  __syncwarp();  // lanes may have given up apart
  tc_fence_before();
  if (shared_v)
    cluster.sync();  // a CTA's barriers and its share stay until the cluster has used them
  else
    __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "n"(tmem_cols(kRB)));
  }
  if (failed) {  // a wait gave up: the rows must not pass for results
    if (tid == 0) atomicAdd(&wait_errors, 1u);
    for (int i = 0; i < n_rows; ++i)
      for (int64_t n = static_cast<int64_t>(n0) * kNBlock + tid;
           n < min(a.N, static_cast<int64_t>(n1) * kNBlock); n += blockDim.x)
        narrow(static_cast<T *>(a.out) + rows[i] * a.out_stride + n, NAN);
  }
}

// CTAs of a kind that a device holds at once, for each device (0: not looked up yet).
struct Fit {
  static constexpr int kDevices = 64;
  std::atomic<int> most[kDevices];
};

// `clusters` clusters of 2^log2c CTAs; where `fit` is not NULL no more than the device
// holds at once (looked up once for a kernel, cluster size and device).  `early`: the launch
// may begin before the kernel before it has ended (it waits for that end itself).
int launch(const void *fn, int64_t clusters, int log2c, int threads, int smem, int most_smem,
           Fit *fit, bool early, LowRankArgs &a, cudaStream_t s) {
  int rc = allow_smem(fn, smem, most_smem);
  if (rc) return rc;
  a.cluster_log2 = log2c;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1u << log2c);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1u << log2c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 2 : 1;
  if (fit) {
    int device = 0, most = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return static_cast<int>(err);
    const bool kept = device < Fit::kDevices;
    if (kept) most = fit->most[device].load(std::memory_order_relaxed);
    if (most == 0) {
      err = cudaOccupancyMaxActiveClusters(&most, fn, &cfg);
      if (err != cudaSuccess) return static_cast<int>(err);
      if (most < 1) return XP_ERANGE;
      if (kept) fit->most[device].store(most, std::memory_order_relaxed);
    }
    if (clusters > most) clusters = most;
  }
  cfg.gridDim = dim3(static_cast<unsigned>(clusters) << log2c);
  void *args[] = {&a};
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
  const bool vec = a.vec_x && a.vec_a && a.vec_b && a.vec_y;
  if (a.M <= kRowsLimit) {
    static Fit fit[2][2];
    // Measured with 64 adapters (us, clusters of 8 / 4 / 2, ranks 16 and 64): 1 row 5.6 / 6.3 /
    // 8.7 and 6.4 / 7.7 / 11.5; 32 rows 6.7 / 6.7 / 8.9 and 8.4 / 8.2 / 11.7; 64 rows
    // 11.4 / 8.2 / 9.0 and 14.8 / 10.3 / 11.8; 256 rows 12.6 / 9.4 / 10.2 and 16.0 / 11.6 / 13.4.
    const int log2c = a.M <= 16 ? 3 : 2;
    const void *fn = vec ? (const void *)rows_kernel<T, kRB, true>
                         : (const void *)rows_kernel<T, kRB, false>;
    constexpr int kBytes = RowsSmem<kRB>::kBytes;
    return launch(fn, a.M, log2c, kThreads, kBytes, kBytes, &fit[vec][log2c & 1], false, a, s);
  }
  const int bytes = 12 * (a.slots + 1);
  int rc = allow_smem((const void *)plan_kernel, bytes, 12 * (XP_MAX_ADAPTER_SLOTS + 1));
  if (rc) return rc;
  plan_kernel<<<kPlanCtas, kPlanThreads, bytes, s>>>(a);
  rc = launch_status();
  if (rc) return rc;
  const int64_t tiles = most_tiles(a.M, a.slots);
  // Where shares of v are exchanged, CTAs wait for one another while they hold tensor
  // memory.  With two CTAs on an SM, or another kernel's beside one, such clusters
  // could each hold what the other's next CTA waits for; so these launches take an
  // SM's shared memory whole, and nothing that uses tensor memory fits beside them.
  const bool shares = a.H > 64 * static_cast<int64_t>(kWholeBlocks);
  // As large a cluster for a tile as leaves all tiles on the device at once, if half
  // of the slots are in use (the host does not know).  Measured at 2048 -> 2048, 6 adapters
  // in 8 slots (us, clusters of 1 / 2 / 4): rank 16, 3000 rows 44 / 28 / 20, 4096 44 / 29 / 35
  // (more tiles than fit), 8192 45 / 31 / 43, 12000 46 / 63 / 62; rank 64, 8192 51 / 34 / 52.
  // At 512 -> 2048, nothing exchanged and two CTAs on an SM, 2048 rows take 18 in clusters of 8.
  const int64_t full = (a.M + kTile - 1) / kTile, guess = full + a.slots / 2;
  const bool two = vec && kRB <= 4;  // two CTAs fit on an SM
  int log2c = 0;
  if (shares)
    log2c = guess * 4 <= 132 ? 2 : (guess * 2 <= 144 ? 1 : 0);
  else
    for (log2c = 3; log2c > 0 && guess << log2c > (two ? 296 : 148);) --log2c;
  // One CTA on an SM with a deep ring up to as many tiles as SMs, then two (16384 rows, rank
  // 64, 2048 -> 2048: 52 / 62 us; 24000 rows: 97 / 82).
  const bool deep = vec && (!two || (shares && guess << log2c <= 148));
  const void *fn = deep ? (const void *)tile_kernel<T, kRB, true, true>
                        : (vec ? (const void *)tile_kernel<T, kRB, true, kRB == 8>
                               : (const void *)tile_kernel<T, kRB, false, false>);
  int smem = deep ? TileSmem<kRB, true, true>::kBytes
                  : (vec ? TileSmem<kRB, true, kRB == 8>::kBytes
                         : TileSmem<kRB, false, false>::kBytes);
  const int most = smem < kWholeSm ? kWholeSm : smem;
  if (shares && log2c > 0) smem = most;
  return launch(fn, tiles, log2c, tile_threads(vec), smem, most, nullptr, true, a, s);
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
                               const void *slot_of, int slot_bytes, int64_t adapters,
                               void *scratch, int64_t scratch_bytes, void *stream) {
  if (dtype != XP_BF16 && dtype != XP_F16) return XP_EINVAL;
  if (M < 0 || H < 1 || N < 1 || r < 1 || slots < 1 || adapters < 0) return XP_EINVAL;
  if (M > XP_MAX_TOKENS || r > XP_MAX_RANK || slots > XP_MAX_ADAPTER_SLOTS || H > INT32_MAX ||
      N > INT32_MAX)
    return XP_ERANGE;
  if (ids_bytes != 4 && ids_bytes != 8) return XP_EINVAL;
  if (slot_of && slot_bytes != 4 && slot_bytes != 8) return XP_EINVAL;
  if (x_stride < 0 || y_stride < 0 || (M > 1 && out_stride < N)) return XP_EINVAL;
  if (M == 0) return XP_OK;
  if (!x || !y || !out || !a || !b || !ids) return XP_EINVAL;
  if (scratch_need(M, slots) > 0 &&
      (!scratch || !aligned(scratch, 16) || scratch_bytes < scratch_need(M, slots)))
    return XP_EINVAL;
  LowRankArgs p{x, y, out, x_stride, y_stride, out_stride, M, H, N,
                static_cast<int>(r), static_cast<int>(slots), a, b, scale, ids, ids_bytes, slot_of,
                slot_bytes, adapters};
  p.vec_x = aligned(x, 16) && x_stride % 8 == 0;
  p.vec_a = aligned(a, 16) && H % 8 == 0;
  p.vec_b = aligned(b, 16) && r % 8 == 0;
  p.vec_y = aligned(y, 16) && aligned(out, 16) && y_stride % 8 == 0 && out_stride % 8 == 0;
  p.wait_ns = wait_limit.load(std::memory_order_relaxed);
  p.in_place = y == out && (y_stride == out_stride || M == 1);
  if (M > kRowsLimit) {
    unsigned char *at = static_cast<unsigned char *>(scratch);
    p.ntiles = reinterpret_cast<int32_t *>(at);
    p.tiles = reinterpret_cast<int4 *>(at + 16);
    p.perm = reinterpret_cast<int32_t *>(at + 16 + 16 * most_tiles(M, slots));
  }
  return dtype == XP_BF16 ? run_typed<__nv_bfloat16>(p, as_stream(stream))
                          : run_typed<__half>(p, as_stream(stream));
}

extern "C" int xp_low_rank_errors(uint32_t *count, void *stream) {
  if (!count) return XP_EINVAL;
  // A wait for a stream would end its capture.
  cudaStreamCaptureStatus capture;
  cudaError_t err = cudaStreamIsCapturing(as_stream(stream), &capture);
  if (err != cudaSuccess) return static_cast<int>(err);
  if (capture != cudaStreamCaptureStatusNone) return XP_EINVAL;
  err = cudaMemcpyFromSymbolAsync(count, wait_errors, sizeof(*count), 0,
                                              cudaMemcpyDeviceToHost, as_stream(stream));
  if (err == cudaSuccess) err = cudaStreamSynchronize(as_stream(stream));
  return err == cudaSuccess ? XP_OK : static_cast<int>(err);
}

extern "C" int64_t xp_low_rank_wait_limit(int64_t ns) {
  if (ns < 0) return wait_limit.load(std::memory_order_relaxed);
  return wait_limit.exchange(static_cast<uint32_t>(ns < kWaitNs ? ns : kWaitNs));
}
