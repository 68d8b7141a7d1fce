// Device helpers of the session-cache attention kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cache_attn.h"
#include "dev_common.cuh"

namespace lfm {
namespace cache {

// What the kernels of the including file report. The kernels name the variable
// itself, so that a launch needs no address from the host.
static __device__ unsigned g_status;
__device__ __forceinline__ void report(unsigned bits) { atomicOr(&g_status, bits); }

// (static, like the variable: each file has its own)
static cudaError_t status_word(unsigned** at) { return cudaGetSymbolAddress((void**)at, g_status); }

// The element types of LFM_ATTN_*: q and out, and the caches.
template <int T>
struct Types;
template <>
struct Types<T_F32> {
  using Q = float;
  using C = __half;
};
template <>
struct Types<T_F16> {
  using Q = __half;
  using C = __half;
};
template <>
struct Types<T_BF16> {
  using Q = __nv_bfloat16;
  using C = __nv_bfloat16;
};

// Weights that enter a product in fp16 are taken relative to a row's reference of
// log2 m = its maximum - SHIFT, not to the maximum: the type's exponents above 1
// would lie idle, and below 2^-14 (low halves of a pair: 2^-3) its steps stop
// shrinking. With 2^15 the steps of a pair are relative down to 2^-18 of the
// largest weight and 2^-40 of it below; with 0 a key that takes all the weight
// over a small V row left 4e-5 (6 nats above the others) to 8e-2 (14) of error
// in fp32 outputs. Sums and outputs carry the same factor, which cancels; bf16
// has fp32's exponents.
template <int T>
constexpr float SHIFT = T == T_BF16 ? 0.f : 15.f;

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// fp32 queries enter a product as fp16 hi/lo pairs. A row whose largest value is
// `most` is multiplied by x, a power of two that brings it to [2^13, 2^14), and
// its scores by y = 1 / x: both exact, so rows of any size keep the pair's 22
// bits (without it queries of 1e-3 against keys of 1e3 lost 1e-4 of the output,
// and those of 65504 and above were infinite). 0, infinities and NaN stay.
__device__ __forceinline__ float2 row_scale(float most) {
  int e = __float_as_uint(most) >> 23 & 255;
  e = e == 255 ? 127 + 13 : max(e, 27);
  return make_float2(__uint_as_float((unsigned)(2 * 127 + 13 - e) << 23), __uint_as_float((unsigned)(e - 13) << 23));
}
template <int N>
__device__ __forceinline__ float max_abs(const float (&f)[N]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) m = max3(m, fabsf(f[i]), fabsf(f[i + 1]));
  return m;
}

__device__ __forceinline__ void from_f32(float x, float* o) { *o = x; }
__device__ __forceinline__ void from_f32(float x, __half* o) { *o = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16* o) { *o = __float2bfloat16_rn(x); }

// Bounded waits, false where they ran out. warp_wait is one for the warp: its lanes' limits end apart, and what follows
// (shuffles, tensor-memory loads) needs all lanes, so they leave it together. lane_wait is for code that one lane alone runs.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, dev::mbar_wait(bar, parity, nullptr));
}
__device__ __forceinline__ bool lane_wait(uint64_t* bar, uint32_t parity) { return dev::mbar_wait(bar, parity, nullptr); }

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(dev::smem_u32(p)), "r"(rank));
  return r;
}

// 2^x by the hardware's instruction, within 2^-22 of it; results under 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t two(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 one(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Four neighbouring outputs.
__device__ __forceinline__ void store4(float* dst, float4 v) { *(float4*)dst = v; }
template <class H>
__device__ __forceinline__ void store4(H* dst, float4 v) {
  __align__(8) H x[4];
  from_f32(v.x, x), from_f32(v.y, x + 1), from_f32(v.z, x + 2), from_f32(v.w, x + 3);
  *(uint2*)dst = *(const uint2*)x;
}

// 32 accumulators times `by`, as 32 neighbouring outputs at 16-byte aligned dst.
template <class Q>
__device__ __forceinline__ void store_row(Q* dst, const uint32_t (&v)[32], float by) {
  constexpr int PER = 16 / sizeof(Q);
#pragma unroll
  for (int e = 0; e < 32; e += PER) {
    __align__(16) Q x[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) from_f32(__uint_as_float(v[e + i]) * by, &x[i]);
    *(uint4*)(dst + e) = *(const uint4*)x;
  }
}

// The slot and the length of session b, checked: false leaves the session out.
__device__ __forceinline__ bool session(const int* slots, const int* lens, int b, int n_slots, int most, int* slot,
                                        int* len) {
  *slot = slots ? slots[b] : b;
  *len = lens[b];
  const unsigned bad = ((unsigned)*slot >= (unsigned)n_slots ? BAD_SLOT : 0u) |
                       ((unsigned)*len > (unsigned)most ? BAD_LEN : 0u);
  if (bad && threadIdx.x == 0) report(bad);
  return !bad;
}

// First position of the window of a query at position p (0: no window).
__host__ __device__ __forceinline__ int window_first(int p, int window) {
  return window > 0 && window <= p ? p - window + 1 : 0;
}

}  // namespace cache
}  // namespace lfm
