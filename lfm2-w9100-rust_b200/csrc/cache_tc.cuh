// Tensor-core helpers of the session-cache attention kernels (tcgen05 / TMEM / TMA).
#pragma once
#include <cuda.h>

#include "cache_common.cuh"
#include "tc_common.cuh"

namespace lfm {
namespace cache {
using namespace dev;
using namespace tc;

// The MMAs are issued by one elected lane of a converged warp: with the branch
// around the instruction alone, addresses and descriptors stay in uniform
// registers (under a branch around the whole loop an MMA took ~100 cycles to
// issue and 64 to run).
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t pack(__half, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t pack(__nv_bfloat16, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *(const uint32_t*)&h;
}
// what an fp16 pair leaves off, as the next fp16 pair
__device__ __forceinline__ uint32_t rest(uint32_t hi, float a, float b) {
  const float2 back = __half22float2(*(const __half2*)&hi);
  return pack(__half(), a - back.x, b - back.y);
}
// N values of a row that LANES neighbouring lanes of a converged warp share, as fp16 pairs of the row brought to size;
// returns what brings its scores back.
template <int LANES, int N>
__device__ __forceinline__ float pairs(const float (&f)[N], uint32_t (&h)[N / 2], uint32_t (&l)[N / 2]) {
  float most = max_abs(f);
#pragma unroll
  for (int o = 1; o < LANES; o *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  const float2 by = row_scale(most);
  const uint64_t by2 = two(by.x, by.x), minus = two(-1.f, -1.f);
#pragma unroll
  for (int e = 0; e < N / 2; e++) {
    const uint64_t x = mul2(two(f[2 * e], f[2 * e + 1]), by2);
    const float2 y = one(x);
    h[e] = pack(__half(), y.x, y.y);
    const float2 back = __half22float2(*(const __half2*)&h[e]), z = one(fma2(two(back.x, back.y), minus, x));
    l[e] = pack(__half(), z.x, z.y);
  }
  return by.y;
}
// 16 bytes at column block `piece` (of 8) of row r of a swizzled 64-wide chunk
__device__ __forceinline__ void st_piece(uint8_t* chunk, int r, int piece, uint4 v) {
  *(uint4*)(chunk + r * 128 + ((piece ^ (r & 7)) << 4)) = v;
}

// The n lowest bits.
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeFn)p;
  }();
  return fn;
}

// A cache slot [kv head][position][d] of 16-bit values, read in boxes of 64 values x `rows` positions of one head.
inline cudaError_t map_cache(CUtensorMap* map, const void* base, int kv_heads, int ctx, int d, int rows) {
  EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)ctx, (cuuint64_t)kv_heads};
  const cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)ctx * d * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)rows, 1}, step[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Query rows [token][head][d] of 16-bit values, read in boxes of 64 values x g heads x `tokens` tokens.
inline cudaError_t map_queries(CUtensorMap* map, const void* q, size_t q_stride, int n, int heads, int d, int g,
                               int tokens) {
  EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)n};
  const cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)q_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)g, (cuuint32_t)tokens}, step[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(q), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace cache
}  // namespace lfm
