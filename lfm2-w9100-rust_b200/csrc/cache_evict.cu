// Eviction from session caches by accumulated attention weight.
#include "cache_attn.h"
#include "cache_common.cuh"

namespace lfm {
namespace cache {
namespace {
using namespace dev;

constexpr int THREADS = 256;

// A float's order as an unsigned: larger weights have larger keys, NaN the smallest.
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned u = __float_as_uint(x + 0.f);  // -0 counts as 0
  if (x != x) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(THREADS) k_evict(Evict a) {
  __shared__ int s_cnt[THREADS / 32], s_dup;
  const int b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int slot, len;
  if (!session(a.slots, a.lens, b, a.n_slots, a.max_len, &slot, &len)) return;
  if (a.slots) {
    if (tid == 0) s_dup = 0;
    __syncthreads();
    for (int i = tid; i < b; i += THREADS)
      if (a.slots[i] == slot) s_dup = 1;
    __syncthreads();
    if (s_dup) {
      if (tid == 0) report(BAD_SLOT);
      return;
    }
  }
  if (h == 0 && tid == 0) a.lens_out[b] = min(len, a.budget);
  const size_t row0 = ((size_t)slot * a.kv_heads + h) * a.ctx;
  const float* acc = a.acc + row0;
  auto block_sum = [&](int v) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) s_cnt[warp] = v;
    __syncthreads();
    int t = 0;
    for (int i = 0; i < THREADS / 32; i++) t += s_cnt[i];
    return t;
  };
  const bool all = len <= a.budget;
  const int lo = all ? len : a.keep_first, hi = all ? len : len - a.keep_last;
  const int want = all ? 0 : a.budget - a.keep_first - a.keep_last;
  // the largest key T that at least `want` middle positions reach
  unsigned T = 0;
  int above = 0;  // keys above T
  if (want > 0) {
    for (int bit = 31; bit >= 0; bit--) {
      const unsigned c = T | 1u << bit;
      int n = 0;
      for (int i = lo + tid; i < hi; i += THREADS) n += order_key(acc[i]) >= c;
      if (block_sum(n) >= want) T = c;
    }
    int n = 0;
    for (int i = lo + tid; i < hi; i += THREADS) n += order_key(acc[i]) > T;
    above = block_sum(n);
  }
  int ties = want - above;  // of those at T, the earliest
  int to = 0;
  const size_t src0 = (size_t)slot * a.slot_stride + (size_t)h * a.ctx * a.d;
  const int pieces = a.d / 8;
  for (int base = 0; base < len; base += THREADS) {
    const int i = base + tid;
    float w = 0.f;
    int ps = 0;
    unsigned key = 0;
    const bool in = i < len;
    if (in) {
      w = acc[i];
      if (a.pos) ps = a.pos[row0 + i];
      key = order_key(w);
    }
    const bool middle = in && i >= lo && i < hi;
    const bool tie = middle && want > 0 && key == T;
    // rank among this block's ties, then among its kept
    const unsigned tb = __ballot_sync(0xffffffffu, tie);
    __syncthreads();
    if (lane == 0) s_cnt[warp] = __popc(tb);
    __syncthreads();
    int before = __popc(tb & ((1u << lane) - 1)), total = 0;
    for (int k = 0; k < THREADS / 32; k++) {
      if (k < warp) before += s_cnt[k];
      total += s_cnt[k];
    }
    const bool keep = in && (!middle || (want > 0 && (key > T || (tie && before < ties))));
    ties -= min(total, ties);
    const unsigned kb = __ballot_sync(0xffffffffu, keep);
    __syncthreads();
    if (lane == 0) s_cnt[warp] = __popc(kb);
    __syncthreads();
    int rank = __popc(kb & ((1u << lane) - 1)), kept = 0;
    for (int k = 0; k < THREADS / 32; k++) {
      if (k < warp) rank += s_cnt[k];
      kept += s_cnt[k];
    }
    // a chunk's rows are read before any is written; later chunks lie behind all that is written here
    __syncthreads();
    if (keep) {
      a.acc_out[row0 + to + rank] = w;
      if (a.pos) a.pos_out[row0 + to + rank] = ps;
    }
    for (int c = 0; c < pieces; c++) {
      uint4 kk = {}, vv = {};
      if (keep) {
        kk = *(const uint4*)((const char*)a.k + 2 * (src0 + (size_t)i * a.d + 8 * c));
        vv = *(const uint4*)((const char*)a.v + 2 * (src0 + (size_t)i * a.d + 8 * c));
      }
      __syncthreads();
      if (keep) {
        *(uint4*)((char*)a.k_out + 2 * (src0 + (size_t)(to + rank) * a.d + 8 * c)) = kk;
        *(uint4*)((char*)a.v_out + 2 * (src0 + (size_t)(to + rank) * a.d + 8 * c)) = vv;
      }
    }
    to += kept;
  }
}
}  // namespace

cudaError_t take_status_evict(unsigned* bits, cudaStream_t s) { return take_status(bits, s); }

cudaError_t evict(const Evict& a, cudaStream_t s) {
  k_evict<<<dim3(a.kv_heads, a.batch), THREADS, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace cache
}  // namespace lfm
