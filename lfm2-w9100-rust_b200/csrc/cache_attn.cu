// Attention over session caches: one warp per query row and head, one lane per
// key for the scores, one lane per head_dim / 32 columns for the output.
#include <type_traits>

#include "cache_attn.h"
#include "cache_common.cuh"

namespace lfm {
namespace cache {
namespace {
using namespace dev;

// The running softmax of one query row.
template <int D>
struct Row {
  float m = -INFINITY, l = 0.f, o[D / 32] = {};
};

// Adds positions [j0, j1) of a cache to the row.
template <int D, class C>
__device__ __forceinline__ void attend(Row<D>& r, const float* q, const C* k, const C* v, int j0, int j1) {
  const int lane = threadIdx.x & 31;
  for (int base = j0; base < j1; base += 32) {
    const int j = base + lane;
    float s = -INFINITY;
    if (j < j1) {
      const C* kr = k + (size_t)j * D;
      s = 0.f;
      for (int c = 0; c < D; c += 8) {
        const uint4 raw = *(const uint4*)(kr + c);
        const C* e = (const C*)&raw;
#pragma unroll
        for (int i = 0; i < 8; i++) s = fmaf(q[c + i], to_f32(e[i]), s);
      }
    }
    float mx = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float m = fmaxf(r.m, mx);
    const float alpha = r.m == -INFINITY ? 0.f : expf(r.m - m);
    const float p = j < j1 ? expf(s - m) : 0.f;
    r.l = r.l * alpha + warp_sum(p);
    r.m = m;
#pragma unroll
    for (int i = 0; i < D / 32; i++) r.o[i] *= alpha;
    const int cnt = min(32, j1 - base);
    for (int t = 0; t < cnt; t++) {
      const float pt = __shfl_sync(0xffffffffu, p, t);
      const C* vr = v + (size_t)(base + t) * D + lane;
#pragma unroll
      for (int i = 0; i < D / 32; i++) r.o[i] = fmaf(pt, to_f32(vr[32 * i]), r.o[i]);
    }
  }
}

template <int D, class Q>
__device__ __forceinline__ void load_q(float* dst, const Q* q, float scale) {
  const int lane = threadIdx.x & 31;
  for (int c = lane; c < D; c += 32) dst[c] = to_f32(q[c]) * scale;
  __syncwarp();
}

template <int D, class Q>
__device__ __forceinline__ void store(const Row<D>& r, Q* out) {
  const int lane = threadIdx.x & 31;
  const float inv = r.l > 0.f || r.l != r.l ? 1.f / r.l : 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; i++) from_f32(r.o[i] * inv, out + lane + 32 * i);
}

template <int T, int D>
__global__ void __launch_bounds__(128) k_window(Prompt a) {
  using Q = typename Types<T>::Q;
  using C = typename Types<T>::C;
  __shared__ float qs[4][D];
  const int w = threadIdx.x >> 5;
  const int h = blockIdx.y;
  const int t = blockIdx.x * 4 + w;
  if (t >= a.n) return;
  const int kh = h / (a.heads / a.kv_heads);
  const C* k = (const C*)a.k + (size_t)kh * a.ctx * D;
  const C* v = (const C*)a.v + (size_t)kh * a.ctx * D;
  load_q<D>(qs[w], (const Q*)a.q + (size_t)t * a.q_stride + h * D, a.scale);
  const int p = a.start + t, lo = window_first(p, a.window);
  Row<D> r;
  attend<D>(r, qs[w], k, v, 0, min(a.sinks, lo));
  attend<D>(r, qs[w], k, v, lo, p + 1);
  store<D>(r, (Q*)a.out + (size_t)t * a.out_stride + h * D);
  if (a.lse && (threadIdx.x & 31) == 0) a.lse[(size_t)t * a.heads + h] = r.m + logf(r.l);
}

// One warp per query head of a KV head; the weights of a position are summed
// over the heads by one thread, so the sum comes out the same on every run.
template <int T, int D>
__global__ void __launch_bounds__(256) k_decode(Decode a) {
  using Q = typename Types<T>::Q;
  using C = typename Types<T>::C;
  __shared__ float qs[8][D], s_m[8], s_inv[8];
  const int kh = blockIdx.x, b = blockIdx.y, w = threadIdx.x >> 5;
  const int g = a.heads / a.kv_heads, h = kh * g + w;
  int slot, len;
  Row<D> r;
  Q* out = (Q*)a.out + (size_t)b * a.out_stride + h * D;
  if (!session(a.slots, a.lens, b, a.n_slots, a.max_len, &slot, &len)) {
    store<D>(r, out);
    return;
  }
  const size_t at = (size_t)slot * a.slot_stride + (size_t)kh * a.ctx * D;
  const C *k = (const C*)a.k + at, *v = (const C*)a.v + at;
  load_q<D>(qs[w], (const Q*)a.q + (size_t)b * a.q_stride + h * D, a.scale);
  if (a.prefix_len) {
    const size_t pat = (size_t)kh * a.prefix_ctx * D;
    attend<D>(r, qs[w], (const C*)a.pk + pat, (const C*)a.pv + pat, 0, a.prefix_len);
  }
  const int lo = window_first(len - 1, a.window), hi = min(a.sinks, lo);
  attend<D>(r, qs[w], k, v, 0, hi);
  attend<D>(r, qs[w], k, v, lo, len);
  store<D>(r, out);
  if (!a.acc) return;
  s_m[w] = r.m;
  s_inv[w] = 1.f / r.l;
  __syncthreads();
  float* acc = a.acc + ((size_t)slot * a.kv_heads + kh) * a.ctx;
  for (int i = threadIdx.x; i < hi + len - lo; i += blockDim.x) {
    const int j = i < hi ? i : lo + i - hi;
    float sum = 0.f;
    for (int x = 0; x < g; x++) {
      float s = 0.f;
      for (int c = 0; c < D; c++) s = fmaf(qs[x][c], to_f32(k[(size_t)j * D + c]), s);
      sum += expf(s - s_m[x]) * s_inv[x];
    }
    acc[j] += sum;
  }
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

cudaError_t window(const Prompt& a, cudaStream_t s) {
  by_type(a.type, a.d, [&](auto t, auto d) {
    k_window<decltype(t)::value, decltype(d)::value><<<dim3((a.n + 3) / 4, a.heads), 128, 0, s>>>(a);
  });
  return cudaGetLastError();
}

cudaError_t weights(const Prompt& a, cudaStream_t s) {
  by_type(a.type, a.d, [&](auto t, auto d) {
    k_weights<decltype(t)::value, decltype(d)::value><<<dim3((a.start + a.n + 31) / 32, a.kv_heads), 32, 0, s>>>(a);
  });
  return cudaGetLastError();
}

cudaError_t shared(const Decode& a, cudaStream_t s) {
  by_type(a.type, a.d, [&](auto t, auto d) {
    k_decode<decltype(t)::value, decltype(d)::value><<<dim3(a.kv_heads, a.batch), 32 * (a.heads / a.kv_heads), 0, s>>>(a);
  });
  return cudaGetLastError();
}

cudaError_t take_status_attn(unsigned* bits, cudaStream_t s) { return take_status(bits, s); }

size_t shared_workspace(const Decode&) { return 16; }

}  // namespace cache
}  // namespace lfm
