// Low-rank adapters of many requests: out = y + scale_s (x A_s^T) B_s^T, the slot
// s of every row from its adapter id.
//
// One CTA owns a row: the low-rank vector v = scale_s x A_s^T goes through shared
// memory, sums are held in 32 bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace xp {
namespace {

constexpr int kThreads = 256;

struct LowRankArgs {
  const void *x, *y;
  void *out;
  int64_t x_stride, y_stride, out_stride;
  int64_t M, H, N, r, slots;
  const void *a, *b;
  const float *scale;
  const void *ids;
  int ids_bytes;
  const int32_t *slot_of;
  int64_t adapters;
};

__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ void narrow(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void narrow(__half *p, float x) { *p = __float2half_rn(x); }

// The slot of row m, -1 without an adapter.
__device__ __forceinline__ int64_t slot_of_row(const LowRankArgs &a, int64_t m) {
  int64_t s = load_id(a.ids, a.ids_bytes, m);
  if (a.slot_of) s = s >= 0 && s < a.adapters ? a.slot_of[s] : -1;
  return s >= 0 && s < a.slots ? s : -1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) rows_kernel(const __grid_constant__ LowRankArgs a) {
  __shared__ float v[XP_MAX_RANK];
  const int64_t m = blockIdx.x;
  const int64_t s = slot_of_row(a, m);
  const T *y = static_cast<const T *>(a.y) + m * a.y_stride;
  T *out = static_cast<T *>(a.out) + m * a.out_stride;
  if (s < 0) {
    if (y != out)
      for (int64_t n = threadIdx.x; n < a.N; n += kThreads) out[n] = y[n];
    return;
  }
  const T *x = static_cast<const T *>(a.x) + m * a.x_stride;
  const T *A = static_cast<const T *>(a.a) + s * a.r * a.H;
  const T *B = static_cast<const T *>(a.b) + s * a.r * a.N;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float scale = a.scale ? a.scale[s] : 1.0f;
  for (int64_t i = warp; i < a.r; i += kThreads / 32) {
    float sum = 0.0f;
    for (int64_t k = lane; k < a.H; k += 32) sum += widen(x[k]) * widen(A[i * a.H + k]);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) v[i] = sum * scale;
  }
  __syncthreads();
  for (int64_t n = threadIdx.x; n < a.N; n += kThreads) {
    float sum = 0.0f;
    for (int64_t i = 0; i < a.r; ++i) sum += v[i] * widen(B[n * a.r + i]);
    narrow(&out[n], widen(y[n]) + sum);
  }
}

template <typename T>
int launch_rows(const LowRankArgs &a, cudaStream_t s) {
  rows_kernel<T><<<static_cast<unsigned>(a.M), kThreads, 0, s>>>(a);
  return launch_status();
}

int64_t scratch_need(int64_t, int64_t) { return 0; }

}  // namespace
}  // namespace xp

using namespace xp;

extern "C" int64_t xp_low_rank_scratch_bytes(int64_t M, int64_t slots) {
  if (M < 0 || M > XP_MAX_TOKENS || slots < 1) return -1;
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
  if (M > XP_MAX_TOKENS || r > XP_MAX_RANK) return XP_ERANGE;
  if (ids_bytes != 4 && ids_bytes != 8) return XP_EINVAL;
  if (x_stride < 0 || y_stride < 0 || (M > 1 && out_stride < N)) return XP_EINVAL;
  if (M == 0) return XP_OK;
  if (!x || !y || !out || !a || !b || !ids) return XP_EINVAL;
  if (scratch_need(M, slots) > 0 &&
      (!scratch || !aligned(scratch, 16) || scratch_bytes < scratch_need(M, slots)))
    return XP_EINVAL;
  LowRankArgs p{x, y, out, x_stride, y_stride, out_stride, M, H, N, r, slots,
                a, b, scale, ids, ids_bytes, slot_of, adapters};
  return dtype == XP_BF16 ? launch_rows<__nv_bfloat16>(p, as_stream(stream))
                          : launch_rows<__half>(p, as_stream(stream));
}
