// A prompt's attention weights summed per cache position
// (lfm_attention_weights): acc[j] += sum over the rows that see j of
// exp(scale q.k_j - lse), given each row's lse.
//
// With the statistics given, one product is enough, and it is taken transposed:
// S^T = K Q^T has a key to a tensor-memory lane, so a thread adds up its key's
// row in registers and nothing is reduced across lanes. A CTA keeps one tile of
// 128 keys and streams the rows that see any of them past it, up to 256 rows (all query
// heads of a KV head, token by token) at a time:
//   warp 0      16-bit queries: the tiles by TMA
//   warp 1      TMEM and the MMAs, into two buffers of S^T
//   warps 2-17  the sums; a key is shared by four threads, each for a quarter of the columns
//   from 18 on  the rows' lse, and for fp32 queries the tiles: fp16 hi/lo pairs, two MMAs
// 16-bit queries are bound by the exponentials: 16 a cycle and SM, 2048 cycles for
// a tile of 128 keys and 256 rows. 8191 bf16 tokens of 32 heads and 128 values:
// 353 us with the inputs in L2, 378 us from memory, the special-function units
// busy for 75% of it. A third of the exponentials through the fma units (range
// reduction and a polynomial of degree 5) took the units' time down to 55% and
// left the total: the issuing warp and the sums' start on each tile are what is
// left. Tiles of 128 rows in four buffers were 2% slower, eight warps for the sums
// 25%. fp32 queries are bound by making their pairs, once for each tile of keys:
// 3840 tokens of 32 heads and 64 values 177 us, with eight warps at it (four took
// twice that).
// A key is summed by one thread, in the order of the rows, tile by tile, and the
// CTAs of a cluster that splits the rows are added up in their order: the
// result is the same on every run.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "cache_tc.cuh"
#include "host_once.h"

namespace lfm {
namespace cache {
namespace {

constexpr int KEYS = 128, EPI = 16, PARTS = EPI / 4, LSE_RING = 4;
constexpr float LOG2E = 1.4426950408889634f;

template <int T, int D>
struct Cfg {
  static constexpr bool PAIR = T == T_F32;
  static constexpr int N = PAIR && D == 128 ? 128 : 256;  // rows of a tile at most: two tiles have to fit
  static constexpr int FEED = PAIR ? 8 : 2;               // warps that write lse, and fp32 queries
  static constexpr int THREADS = 32 * (2 + EPI + FEED);
  static constexpr int K_CHUNK = KEYS * 128, K_TILE = K_CHUNK * (D / 64);
  static constexpr int Q_CHUNK = N * 128, Q_TILE = Q_CHUNK * (D / 64), STAGE = (PAIR ? 2 : 1) * Q_TILE;
  static constexpr int RING = std::min(4, (200 * 1024 - K_TILE) / STAGE);
  static constexpr int SMEM = K_TILE + RING * STAGE;
  static_assert(RING >= 2, "shared memory");
};

struct Args {
  int heads, kv_heads, g, ctx, nranks;
  float scale2;  // scale * log2 e
  const float* q;  // fp32 queries
  size_t q_stride;
  int start, n, window, sinks;
  int tokens;  // of a tile
  const float* lse;
  float* acc;
};

template <int T, int D>
__global__ void __launch_bounds__((Cfg<T, D>::THREADS), 1)
    k_weights(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q, const Args a) {
  using F = Cfg<T, D>;
  using C = typename Types<T>::C;
  constexpr bool PAIR = F::PAIR;
  constexpr uint32_t BF = std::is_same<C, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
  extern __shared__ __align__(1024) uint8_t smem[];  // K, then the ring of query tiles
  __shared__ uint64_t k_full, full[F::RING], empty[F::RING], s_full[2], s_free[2], lse_full[LSE_RING], lse_free[LSE_RING], drained;
  __shared__ uint32_t tmem_at;
  __shared__ __align__(16) float s_lse[LSE_RING][F::N];  // -lse in log2 units
  __shared__ __align__(16) float s_row[LSE_RING][PAIR ? F::N : 4];  // fp32 queries: what makes a row's scores powers of two
  __shared__ float s_sum[8][KEYS];                      // the quarters' sums, then those of the cluster's CTAs
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // blockIdx.x counts ranks, then KV heads, then tiles: the first keys, which most rows see, come first
  const int nranks = a.nranks, rank = blockIdx.x % nranks, kh = blockIdx.x / nranks % a.kv_heads;
  const int j0 = blockIdx.x / nranks / a.kv_heads * KEYS;
  const int cols = a.tokens * a.g;
  // the tokens that see a key of this tile, in whole tiles, and this CTA's share of them
  const int first = max(0, j0 - a.start) / a.tokens;
  const int end_tok = a.window && j0 >= a.sinks ? min((long long)a.n, (long long)j0 + KEYS - 1 + a.window - a.start) : a.n;
  const int total = max(0, (end_tok + a.tokens - 1) / a.tokens - first);
  const int i0 = first + (int)((long long)total * rank / nranks), i1 = first + (int)((long long)total * (rank + 1) / nranks);
  const int count = i1 - i0;

  if (tid == 0) {
    mbar_init(&k_full, 1);
    mbar_init(&drained, 1);
    for (int i = 0; i < F::RING; i++) {
      mbar_init(&full[i], PAIR ? F::FEED : 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < LSE_RING; i++) {
      mbar_init(&lse_full[i], F::FEED);
      mbar_init(&lse_free[i], EPI);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], EPI);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&tmem_at, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  pdl_wait();  // up to here the kernel may run beside the one before it
  if (nranks > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  bool ok = true;
  float sum = 0.f;

  if (warp == 0) {
    if (lane == 0 && count > 0) {
      mbar_expect_tx(&k_full, F::K_TILE);
#pragma unroll
      for (int c = 0; c < D / 64; c++) tma_load_3d(smem + c * F::K_CHUNK, &map_k, 64 * c, j0, kh, &k_full);
      int k = 0;
      if (!PAIR)
        for (; k < count; k++) {
          const int st = k % F::RING;
          if (k >= F::RING && !(ok = lane_wait(&empty[st], (k / F::RING - 1) & 1))) break;
          mbar_expect_tx(&full[st], cols * 2 * D);
#pragma unroll
          for (int c = 0; c < D / 64; c++)
            tma_load_3d(smem + F::K_TILE + st * F::STAGE + c * F::Q_CHUNK, &map_q, 64 * c, kh * a.g, (i0 + k) * a.tokens,
                        &full[st]);
        }
      // the copies land before the CTA ends
      lane_wait(&k_full, 0);
      for (int i = max(0, k - F::RING); i < k; i++) lane_wait(&full[i % F::RING], (i / F::RING) & 1);
    }
  } else if (warp == 1) {
    if (count > 0) {
      const uint32_t tm = uniform(tmem), kb = uniform(smem_u32(smem));
      const uint32_t idesc = idesc_f16(KEYS, cols, false) | BF;
      ok = warp_wait(&k_full, 0);
      for (int k = 0; k < count && ok; k++) {
        const int st = k % F::RING;
        if (!(ok = warp_wait(&full[st], (k / F::RING) & 1))) break;
        if (k >= 2 && !(ok = warp_wait(&s_free[k & 1], (k / 2 - 1) & 1))) break;
        tc_fence_after();
        const uint64_t kd = smem_desc_sw128(kb), qd = smem_desc_sw128(kb + F::K_TILE + st * F::STAGE);
#pragma unroll
        for (int h = 0; h < (PAIR ? 2 : 1); h++)  // the low parts first
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++)
            mma_ss(tm + 256 * (k & 1), kd + (((kk >> 2) * F::K_CHUNK + (kk & 3) * 32) >> 4),
                   qd + (((PAIR ? 1 - h : 0) * F::Q_TILE + (kk >> 2) * F::Q_CHUNK + (kk & 3) * 32) >> 4), idesc, h || kk);
        commit(&s_full[k & 1]);
        commit(&empty[st]);
      }
      if (!ok) {
        commit(&drained);  // no product is left in flight when the tensor memory goes
        warp_wait(&drained, 0);
      }
    }
  } else if (warp < 2 + EPI) {
    // --------------------------------------------------------------- sums
    constexpr int COLS = F::N / PARTS;
    const int part = (warp - 2) >> 2, quarter = warp & 3, key = quarter * 32 + lane, j = j0 + key;
    const uint64_t sc2 = two(a.scale2, a.scale2);
    for (int k = 0; k < count; k++) {
      if (!(ok = warp_wait(&lse_full[k % LSE_RING], (k / LSE_RING) & 1) && warp_wait(&s_full[k & 1], (k >> 1) & 1)))
        break;
      __syncwarp();
      tc_fence_after();
      const int t0 = (i0 + k) * a.tokens, p0 = a.start + t0, p1 = p0 + a.tokens - 1;
      const bool all = p0 >= j0 + KEYS - 1 && t0 + a.tokens <= a.n &&
                       (a.window == 0 || p1 - j0 < a.window || j0 + KEYS <= a.sinks);
      // the columns of this key's queries
      int lo = 0, hi = cols;
      if (!all) {
        lo = max(0, j - p0) * a.g;
        hi = min(a.tokens, a.n - t0) * a.g;
        if (a.window && j >= a.sinks) hi = min(hi, max(0, j + a.window - p0) * a.g);
      }
      const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16) + 256 * (k & 1) + part * COLS;
      const float* nl = s_lse[k % LSE_RING] + part * COLS;
      const float* rs = s_row[k % LSE_RING] + (PAIR ? part * COLS : 0);
      uint64_t s2[2] = {0, 0};  // pairs of 0.f
#pragma unroll
      for (int c = 0; c < COLS / 32; c++) {
        uint32_t w[32];
        tmem_ld32(at + 32 * c, w);
        const int c0 = part * COLS + 32 * c;
        if (!all || c0 + 32 > cols) {
          const uint32_t see = low_bits(hi - c0) & ~low_bits(lo - c0);
          if (__any_sync(0xffffffffu, see != 0)) {
#pragma unroll
            for (int e = 0; e < 32; e++) {
              const float x = exp2_fast(fmaf(__uint_as_float(w[e]), PAIR ? rs[32 * c + e] : a.scale2, nl[32 * c + e]));
              if (see >> e & 1) sum += x;
            }
          }
          continue;
        }
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const float4 n4 = ((const float4*)(nl + 32 * c))[e / 2];
          uint64_t by = sc2;
          if constexpr (PAIR) {
            const float4 r4 = ((const float4*)(rs + 32 * c))[e / 2];
            by = e & 1 ? two(r4.z, r4.w) : two(r4.x, r4.y);
          }
          const uint64_t x = fma2(two(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1])), by,
                                  e & 1 ? two(n4.z, n4.w) : two(n4.x, n4.y));
          const float2 y = one(x);
          s2[e & 1] = add2(s2[e & 1], two(exp2_fast(y.x), exp2_fast(y.y)));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s_free[k & 1]);
        mbar_arrive(&lse_free[k % LSE_RING]);
      }
      const float2 s = one(add2(s2[0], s2[1]));
      sum += s.x + s.y;
    }
    s_sum[part][key] = sum;
  } else {
    // ---------------------------------------------------------- lse, fp32 queries
    const int ft = tid - 32 * (2 + EPI);
    const int per_row = 65536 / a.g + 1;  // row / g = row * per_row >> 16 for rows of a tile
    constexpr int PER = (F::N + 32 * F::FEED - 1) / (32 * F::FEED), AHEAD = 4;
    float pre[AHEAD][PER];  // loaded AHEAD tiles before they are stored: under the tiles' traffic a load takes ~2700 cycles
    int off[PER];           // of a row's lse from that of its tile's first token
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int c = ft + 32 * F::FEED * i;
      off[i] = c / a.g * a.heads + c % a.g;
    }
    auto fetch = [&](int k, float(&e)[PER]) {
      const int t0 = (i0 + k) * a.tokens, have = min(a.tokens, a.n - t0) * a.g;  // rows that exist
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const int c = ft + 32 * F::FEED * i;
        e[i] = INFINITY;
        if (k < count && c < have) e[i] = a.lse[(size_t)t0 * a.heads + kh * a.g + off[i]];
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) fetch(i, pre[i]);
    auto feed = [&](int k, float(&e)[PER]) {
      const int st = k % F::RING, t0 = (i0 + k) * a.tokens, have = min(a.tokens, a.n - t0) * a.g;
      if (k >= LSE_RING && !(ok = warp_wait(&lse_free[k % LSE_RING], (k / LSE_RING - 1) & 1))) return;
#pragma unroll
      for (int i = 0; i < PER; i++)
        if (ft + 32 * F::FEED * i < F::N) s_lse[k % LSE_RING][ft + 32 * F::FEED * i] = -LOG2E * e[i];
      fetch(k + AHEAD, e);
      if constexpr (PAIR) {
        if (k >= F::RING && !(ok = warp_wait(&empty[st], (k / F::RING - 1) & 1))) return;
        uint8_t* dst = smem + F::K_TILE + st * F::STAGE;
        constexpr int LANES = D / 16;  // to a row, each with the 8-value pieces c and c + LANES
#pragma unroll 1
        for (int i = ft; i < cols * LANES; i += 32 * F::FEED) {
          const int row = i / LANES, c = i % LANES;
          float f[16] = {};
          if (row < have) {
            const int t = row * per_row >> 16;
            const float* q = a.q + (size_t)(t0 + t) * a.q_stride + (size_t)(kh * a.g + row - t * a.g) * D + 8 * c;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float4 u = *(const float4*)(q + (e >> 1) * 8 * LANES + (e & 1) * 4);
              f[4 * e] = u.x, f[4 * e + 1] = u.y, f[4 * e + 2] = u.z, f[4 * e + 3] = u.w;
            }
          }
          uint32_t h[8], l[8];
          const float back = pairs<LANES>(f, h, l);
          if (c == 0) s_row[k % LSE_RING][row] = back * a.scale2;
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int piece = c + e * LANES;
            uint8_t* chunk = dst + (piece >> 3) * F::Q_CHUNK;
            st_piece(chunk, row, piece & 7, make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]));
            st_piece(chunk + F::Q_TILE, row, piece & 7, make_uint4(l[4 * e], l[4 * e + 1], l[4 * e + 2], l[4 * e + 3]));
          }
        }
        fence_async_smem();
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&lse_full[k % LSE_RING]);
        if (PAIR) mbar_arrive(&full[st]);
      }
    };
    for (int k = 0; k < count && ok; k += AHEAD)
#pragma unroll
      for (int i = 0; i < AHEAD; i++)
        if (k + i < count && ok) feed(k + i, pre[i]);
  }
  if (!ok && lane == 0) report(BAD_WAIT);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (tid < KEYS) sum = (s_sum[0][tid] + s_sum[1][tid]) + (s_sum[2][tid] + s_sum[3][tid]);
  if (nranks > 1) {
    // to the first CTA, which adds them up in the order of the ranks
    __syncthreads();
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire;\nbarrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    if (tid < KEYS)
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(peer(&s_sum[rank][tid], 0)), "f"(sum) : "memory");
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    if (rank) return;
    if (tid < KEYS) {
      sum = 0.f;
      for (int r = 0; r < nranks; r++) sum += s_sum[r][tid];
    }
  }
  // the record of a position that no row sees is another's
  const int j = j0 + tid;
  if (tid < KEYS && j < a.start + a.n && (a.window == 0 || j < a.sinks || a.start - j < a.window))
    a.acc[(size_t)kh * a.ctx + j] += sum;
}

template <int T, int D>
cudaError_t launch(const Prompt& p, cudaStream_t s) {
  using F = Cfg<T, D>;
  Args a = {};
  a.heads = p.heads, a.kv_heads = p.kv_heads, a.g = p.heads / p.kv_heads, a.ctx = p.ctx;
  a.scale2 = p.scale * LOG2E;
  a.q = (const float*)p.q, a.q_stride = p.q_stride;
  a.start = p.start, a.n = p.n, a.window = p.window, a.sinks = p.sinks;
  a.lse = p.lse, a.acc = p.acc;
  // as many tokens as give whole groups of 16 columns and at most N of them
  int unit = 16;
  while (unit > 1 && (unit / 2) * a.g % 16 == 0) unit /= 2;
  a.tokens = F::N / a.g / unit * unit;
  CUtensorMap mk, mq;
  cudaError_t e = map_cache(&mk, p.k, p.kv_heads, p.ctx, D, KEYS);
  if (e == cudaSuccess && !F::PAIR)
    e = map_queries(&mq, p.q, p.q_stride, p.n, p.heads, D, a.g, a.tokens);
  else
    mq = mk;
  if (e != cudaSuccess) return e;
  auto* f = k_weights<T, D>;
  static unsigned long long done = 0;
  static std::mutex mu;
  once_per_device(done, mu, [f] { cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM); });
  const int tiles = (p.start + p.n + KEYS - 1) / KEYS, most = (p.n + a.tokens - 1) / a.tokens;
  int nranks = 1;
  while (nranks < 8 && 2ll * nranks * tiles * p.kv_heads <= 148 && 2 * nranks <= most) nranks *= 2;
  cudaLaunchConfig_t c = {};
  a.nranks = nranks;
  c.gridDim = dim3((unsigned)nranks * p.kv_heads * tiles);
  c.blockDim = dim3(F::THREADS);
  c.dynamicSmemBytes = F::SMEM;
  c.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = nranks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits for what is before it (pdl_wait)
  at[1].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = 2;
  return cudaLaunchKernelEx(&c, f, mk, mq, a);
}
}  // namespace

cudaError_t weights(const Prompt& a, cudaStream_t s) {
  if (a.type == T_F32) return a.d == 64 ? launch<T_F32, 64>(a, s) : launch<T_F32, 128>(a, s);
  if (a.type == T_F16) return a.d == 64 ? launch<T_F16, 64>(a, s) : launch<T_F16, 128>(a, s);
  return a.d == 64 ? launch<T_BF16, 64>(a, s) : launch<T_BF16, 128>(a, s);
}

cudaError_t status_word_weights(unsigned** at) { return status_word(at); }

}  // namespace cache
}  // namespace lfm
