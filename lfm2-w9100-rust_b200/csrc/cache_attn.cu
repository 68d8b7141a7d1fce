// A prompt's attention weights summed per position: one lane a key.
#include <type_traits>

#include "cache_attn.h"
#include "cache_common.cuh"

namespace lfm {
namespace cache {
namespace {
using namespace dev;

template <int D, class Q>
__device__ __forceinline__ void load_q(float* dst, const Q* q, float scale) {
  const int lane = threadIdx.x & 31;
  for (int c = lane; c < D; c += 32) dst[c] = to_f32(q[c]) * scale;
  __syncwarp();
}

template <int T, int D>
__global__ void __launch_bounds__(32) k_weights(Prompt a) {
  using Q = typename Types<T>::Q;
  using C = typename Types<T>::C;
  __shared__ float qs[D];
  const int kh = blockIdx.y, j = blockIdx.x * 32 + threadIdx.x;
  const int g = a.heads / a.kv_heads;
  const bool in = j < a.start + a.n;
  float kr[D];
#pragma unroll
  for (int c = 0; c < D; c++) kr[c] = in ? to_f32(((const C*)a.k)[((size_t)kh * a.ctx + j) * D + c]) : 0.f;
  float sum = 0.f;
  for (int t = max(0, (int)(blockIdx.x * 32) - a.start); t < a.n; t++) {
    const int p = a.start + t;
    const bool see = in && j <= p && (a.window == 0 || p - j < a.window || j < a.sinks);
    if (!__any_sync(0xffffffffu, see)) continue;
    for (int h = kh * g; h < (kh + 1) * g; h++) {
      __syncwarp();
      load_q<D>(qs, (const Q*)a.q + (size_t)t * a.q_stride + h * D, a.scale);
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < D; c++) s = fmaf(qs[c], kr[c], s);
      if (see) sum += expf(s - a.lse[(size_t)t * a.heads + h]);
    }
  }
  if (in) a.acc[(size_t)kh * a.ctx + j] += sum;
}

template <class F>
void by_type(int type, int d, F&& f) {
  auto with_d = [&](auto t) {
    if (d == 64)
      f(t, std::integral_constant<int, 64>());
    else
      f(t, std::integral_constant<int, 128>());
  };
  if (type == T_F32)
    with_d(std::integral_constant<int, T_F32>());
  else if (type == T_F16)
    with_d(std::integral_constant<int, T_F16>());
  else
    with_d(std::integral_constant<int, T_BF16>());
}
}  // namespace

cudaError_t weights(const Prompt& a, cudaStream_t s) {
  by_type(a.type, a.d, [&](auto t, auto d) {
    k_weights<decltype(t)::value, decltype(d)::value><<<dim3((a.start + a.n + 31) / 32, a.kv_heads), 32, 0, s>>>(a);
  });
  return cudaGetLastError();
}

}  // namespace cache
}  // namespace lfm
