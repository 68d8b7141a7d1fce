// Eviction from session caches by accumulated attention weight.
//
// A cluster of CTAs takes one KV head of one session. Each CTA finds the weight T
// of the last position to keep by itself (three passes over the weights with
// histograms of 11, 11 and 10 bits of their order-preserving keys), and then
// walks the positions once, 1024 at a time: two counts before each position, of
// those above T and of those at T, give its place. The list of kept positions is moved
// in rounds: a round's rows are shared out among the CTAs, 32 KB to each, 128 bytes of
// loads in flight to a thread, and written behind the ones before. In place, a
// round's rows are all read before any is written (one cluster barrier); what is
// written lies in front of everything that later rounds and passes read, since
// the row that becomes the r-th comes from position r or behind.
// Bound by memory, of which it reaches 83%: every kept row is read and written
// once, but a CTA's loads wait for its stores to be issued.
#include <algorithm>

#include "cache_attn.h"
#include "cache_common.cuh"

namespace lfm {
namespace cache {
namespace {
using namespace dev;

constexpr int THREADS = 256, WARPS = THREADS / 32, EACH = 4, UNIT = THREADS * EACH, BINS = 2048;
constexpr int LIST = 2048;  // positions that are listed and not yet moved: fewer than a round's 1024 and a unit's 1024
// Up to so many positions' keys are read from memory once and kept: what static shared memory holds beside the lists.
// Longer sessions read their weights in every pass (all of them: 172 instead of 151 us for 48 sessions of up to 8192).
constexpr int KEYS = 8192;

// A weight's order as an unsigned: larger weights have larger keys, NaN the smallest.
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned u = __float_as_uint(x + 0.f);  // -0 counts as 0
  if (x != x) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int warp_before(int v, int lane, int* all) {
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  *all = __shfl_sync(0xffffffffu, s, 31);
  return s - v;
}

template <int D>
__global__ void __launch_bounds__(THREADS, 4) k_evict(Evict a, bool in_place) {
  constexpr int ROWS = 8192 / D, PIECES = D / 8;  // rows of a round for one CTA; 16-byte pieces of a row
  __shared__ union {
    int hist[BINS];
    int list[LIST];
  } u;
  __shared__ unsigned s_key[KEYS];
  __shared__ int s_warp[WARPS], s_found[2], s_dup;
  const int rank = blockIdx.x, nranks = gridDim.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();  // up to here the kernel may run beside the one before it
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
  if (h == 0 && rank == 0 && tid == 0) a.lens_out[b] = min(len, a.budget);
  const bool all = len <= a.budget;
  if (all && in_place) return;
  const size_t row0 = ((size_t)slot * a.kv_heads + h) * a.ctx;
  const float* acc = a.acc + row0;
  const int lo = all ? len : a.keep_first, hi = all ? len : len - a.keep_last;
  const int want = all ? 0 : a.budget - a.keep_first - a.keep_last;

  const bool kept_keys = len <= KEYS && want > 0;
  if (kept_keys) {
#pragma unroll 8
    for (int i = tid; i < len; i += THREADS) s_key[i] = order_key(acc[i]);
    __syncthreads();
  }
  auto key_of = [&](int i) { return kept_keys ? s_key[i] : order_key(acc[i]); };

  // T: the largest key that at least `want` of the middle positions reach; `ties` of those at T are kept
  unsigned T = 0;
  int ties = want;
  if (want > 0) {
    unsigned known = 0;  // the bits of T that are found
    for (int pass = 0; pass < 3; pass++) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < BINS; i += THREADS) u.hist[i] = 0;
      __syncthreads();
      // a warp's 32 neighbours together, those behind the last too: every lane takes part in the warp's votes
#pragma unroll 8
      for (int first = lo + tid - lane; first < hi; first += THREADS) {
        const int i = first + lane;
        const unsigned k = i < hi ? key_of(i) : 0u;
        const int bin = k >> shift & ((1 << bits) - 1);
        const bool counts = i < hi && (k & known) == T;
        // equal weights are common (positions never looked at): one addition for those of a warp
        const unsigned members = __ballot_sync(0xffffffffu, counts);
        if (counts) {
          int same;
          __match_all_sync(members, bin, &same);
          if (!same)
            atomicAdd(&u.hist[bin], 1);
          else if (lane == __ffs(members) - 1)
            atomicAdd(&u.hist[bin], __popc(members));
        }
      }
      __syncthreads();
      // from the highest bin down: the one with the `ties`-th key
      int c[BINS / THREADS], sum = 0, total;
#pragma unroll
      for (int i = 0; i < BINS / THREADS; i++) {
        c[i] = u.hist[BINS - 1 - (tid * (BINS / THREADS) + i)];
        sum += c[i];
      }
      int before = warp_before(sum, lane, &total);
      if (lane == 0) s_warp[warp] = total;
      __syncthreads();
      for (int i = 0; i < warp; i++) before += s_warp[i];
      if (before < ties && before + sum >= ties) {
        int i = 0;
        while (before + c[i] < ties) before += c[i++];
        s_found[0] = BINS - 1 - (tid * (BINS / THREADS) + i);
        s_found[1] = before;
      }
      __syncthreads();
      T |= (unsigned)s_found[0] << shift;
      ties -= s_found[1];
      known |= ((1u << bits) - 1) << shift;
    }
  }
  __syncthreads();

  const size_t src0 = (size_t)slot * a.slot_stride + (size_t)h * a.ctx * D;
  const int keep = min(len, a.budget), each = ROWS * nranks;
  int listed = 0, moved = 0, tied = 0;  // kept so far, of them moved; positions at T so far
  for (int base = 0; base < len; base += UNIT) {
    // this thread's positions: above T (or kept in any case), at T
    unsigned sure = 0, tie = 0;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const int i = base + tid * EACH + e;
      if (i >= len) continue;
      if (i < lo || i >= hi) {
        sure |= 1u << e;
      } else if (want > 0) {
        const unsigned k = key_of(i);
        if (k > T) sure |= 1u << e;
        if (k == T) tie |= 1u << e;
      }
    }
    int total;
    int before = warp_before(__popc(sure) << 16 | __popc(tie), lane, &total);
    __syncthreads();  // s_warp has been read, and the list's places that come round
    if (lane == 0) s_warp[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int i = 0; i < WARPS; i++) {
      if (i < warp) before += s_warp[i];
      total += s_warp[i];
    }
    int ns = before >> 16, nt = tied + (before & 0xffff);
    const int kept_ties = min(tied, ties);
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const bool is_tie = tie >> e & 1, is_sure = sure >> e & 1;
      if (is_sure || (is_tie && nt < ties))
        u.list[(listed + ns + min(nt, ties) - kept_ties) % LIST] = base + tid * EACH + e;
      ns += is_sure, nt += is_tie;
    }
    tied += total & 0xffff;
    listed += (total >> 16) + min(tied, ties) - kept_ties;
    __syncthreads();
    // whole rounds, and at the end what is left
    while (listed - moved >= each || (base + UNIT >= len && moved < keep)) {
      const int first = moved + rank * ROWS, have = min(ROWS, listed - first);  // this CTA's rows, may be none
      uint4 v[8];
      int to[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int x = tid + THREADS * (i & 3), r = x / PIECES;
        to[i] = -1;
        if (r < have) {
          const int from = u.list[(first + r) % LIST];
          if (!in_place || from != first + r) {
            to[i] = first + r;
            v[i] = *(const uint4*)((const char*)(i < 4 ? a.k : a.v) + 2 * (src0 + (size_t)from * D) + 16 * (x % PIECES));
          }
        }
      }
      float w = 0.f;
      int ps = 0;
      if (tid < have) {
        const int from = u.list[(first + tid) % LIST];
        w = acc[from];
        if (a.pos) ps = a.pos[row0 + from];
      }
      if (in_place) {
        __syncwarp();
        if (nranks > 1)
          cluster_sync();
        else
          __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (to[i] >= 0)
          *(uint4*)((char*)(i < 4 ? a.k_out : a.v_out) + 2 * (src0 + (size_t)to[i] * D) +
                    16 * ((tid + THREADS * (i & 3)) % PIECES)) = v[i];
      if (tid < have) {
        a.acc_out[row0 + first + tid] = w;
        if (a.pos) a.pos_out[row0 + first + tid] = ps;
      }
      moved = min(moved + each, listed);
    }
  }
}
}  // namespace

cudaError_t status_word_evict(unsigned** at) { return status_word(at); }

cudaError_t evict(const Evict& a, cudaStream_t s) {
  // As many CTAs to a head as give every SM two, each with a round of its own at least. More repeat the selection for
  // less work each, fewer leave SMs idle. Rules of one, two and four to an SM: 16 sessions of 8 heads, 8192 to 2045
  // positions, 66, 66 and 90 us; 24 of up to 8192 95, 82 and 101; 48 153, 153 and 163; 37 of 4 heads, 3000 to 1000,
  // 25, 21 and 32; one of 4096 to 1024 13.8 each.
  const int rows = 8192 / a.d, most = std::min(a.max_len, a.budget);
  int nranks = 1;
  while (nranks < 8 && (long long)a.batch * a.kv_heads * nranks < 2 * 148 && rows * nranks < most) nranks *= 2;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(nranks, a.kv_heads, a.batch);
  c.blockDim = dim3(THREADS);
  c.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = nranks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits for what is before it (pdl_wait)
  at[1].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = 2;
  return a.d == 64 ? cudaLaunchKernelEx(&c, k_evict<64>, a, a.k == a.k_out)
                   : cudaLaunchKernelEx(&c, k_evict<128>, a, a.k == a.k_out);
}

}  // namespace cache
}  // namespace lfm
