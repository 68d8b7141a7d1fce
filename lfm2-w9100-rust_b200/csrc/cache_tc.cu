// Attention of many query rows over one cache on the tensor cores (tcgen05 /
// TMEM): a prompt's rows under a causal window with sinks
// (lfm_attention_window), and the rows of all sessions over their shared
// prefix (the prefix half of lfm_attention_shared).
//
// Rows are packed: row R of a KV head is query head R % g of token (or session)
// R / g, so every group size fills the 128-row tiles. A CTA holds one tile of
// rows and walks the positions in tiles of 64; two CTAs share an SM, so that one
// fills the other's waits, its start and its end. In a CTA
//   warp 0     TMA: K and V tiles into a ring each
//   warp 1     TMEM and the MMAs: S = Q K^T, O += P V
//   warps 2-5  the softmax, one thread a row
// S has two buffers: the next tile's scores are computed while this one's are in
// the softmax. The weights P take the place of S in tensor memory and enter the
// second product from there.
// (Two tiles of rows and 128 positions with one S each, an SM to a CTA: the chain
// softmax - P V - Q K^T took 4400 cycles for 128 positions of bf16, 128 values,
// of which either unit was busy for half: 282 us for 8192 tokens, window 1500.)
//
// 16-bit queries: O stays in tensor memory, and a row's maximum is raised, and O
// rescaled, only when it grows by more than 2^8; over long rows it is moved every
// FOLD tiles into a running output. Weights are relative to the maximum less TOP,
// which keeps them inside fp16's range up to that growth and their roundings
// relative (fp16: down to 2^-21 of the largest). They are rounded to the caches'
// type, half a step each (fp16 2^-11, bf16 2^-8), as the caller's V and output
// are; the sums l are of the weights as they were. With the output's own rounding
// that is 2.2e-3 of error in bf16 and 2.8e-4 in fp16. (Pairs of weights and two
// MMAs: 1.6e-3 and 2.1e-4, what the output's rounding alone leaves, for 252
// instead of 207 us on 8192 bf16 tokens of 128 values behind a window of 1500,
// 130 instead of 115 us on 256 bf16 sessions behind a prefix, 73 instead of 67 us
// on 3840 fp16 tokens of 64 values: not taken.)
// fp32 queries: q, brought to size row by row, and P are fp16 hi/lo pairs, two
// MMAs each, the low parts first; the tensor core cuts its sums off instead of
// rounding them, a loss that grows with their number (2.2e-6 over 1024
// positions), so O of each tile starts from zero and is added to the running
// output in registers. A score of s nats still loses up to head_dim / 16 * 2^-23 s.
// Few row tiles leave SMs idle, so a cluster of CTAs may split the positions of
// one tile; each sends its part of a row to the CTA that finishes the row.
// Every wait is bounded; one that runs out is reported and the CTA releases
// its tensor memory.
#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "cache_tc.cuh"
#include "host_once.h"

namespace lfm {
namespace cache {
namespace {
using namespace dev;
using namespace tc;

constexpr int THREADS = 192, KT = 64, ROWS = 128;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float GROWTH = 8.f;  // log2 of what a row may grow before its maximum is raised
// log2 of the largest weight when the maximum has just been raised: fp16 keeps room for GROWTH
template <int T>
constexpr float TOP = T == T_F16 ? SHIFT<T> - GROWTH : SHIFT<T>;
constexpr uint32_t COLS = 256, COL_O = 2 * KT;  // tensor memory: two buffers of S, then those of O

template <int T, int D>
struct Cfg {
  static constexpr bool PAIR = T == T_F32;
  static constexpr int Q_CHUNK = ROWS * 128, KV_CHUNK = KT * 128;  // rows x 64 16-bit values, swizzled
  static constexpr int Q_TILE = Q_CHUNK * (D / 64), TILE = KV_CHUNK * (D / 64);
  static constexpr int Q_BYTES = (PAIR ? 2 : 1) * Q_TILE;
  static constexpr int STATIC = 2048, RESERVED = 1024;  // of the kernel's static arrays, of the system
  // two CTAs to an SM, except for fp32 queries of 128 values, whose pairs leave no room for the second one's ring
  static constexpr int CTAS = PAIR && D == 128 ? 1 : 2;
  static constexpr int RING = std::min(4, (228 * 1024 / CTAS - STATIC - RESERVED - Q_BYTES) / (2 * TILE));  // K and V tiles each
  static constexpr int SMEM = Q_BYTES + 2 * RING * TILE;
  // O buffers: fp32 queries fold one while the next product fills the other, where there is room
  static constexpr int OBUF = PAIR && D == 64 ? 2 : 1;
  static constexpr int STRIDE = D + 4;  // floats of a row in the join: rows of one column start in different banks
  static_assert(RING >= 2 && COL_O + OBUF * D <= COLS, "memories");
  static_assert(ROWS * (STRIDE * 4 + 8) <= SMEM, "the join takes the place of queries and ring");
};

struct Rows {
  int heads, kv_heads, g, rows;  // rows of one KV head
  int nranks;                    // CTAs that split a tile's positions
  float scale2;                  // scale * log2 e
  const void* q;
  size_t q_stride;
  // prompt: positions start + R / g under window and sinks; prefix: len positions
  bool prefix;
  int start, window, sinks, len;
  void* out;
  size_t out_stride;
  float* lse;
  float* part;     // prefix: O [kv head][row][D], not divided
  float2* part_ml; // prefix: (m in log2 units, l)
};

// ln of 2^m l; the sum without its factor, so that the logarithm is of a number near 1 or above.
template <int T>
__device__ __forceinline__ float log_sum(float m, float l) {
  return ((m + TOP<T>) + log2f(l * exp2f(-TOP<T>))) * LN2;
}

// Tiles whose output 16-bit queries add up in tensor memory, which cuts the sums off: 256 sums lose at most 3e-5, 1/16
// of fp16's half step. Without the fold a row of 2^20 positions came out smaller by 8e-4.
constexpr int FOLD = 64;

// The position tiles of a block of rows: the sinks in front of the window, then
// the positions from the first row's window to the last row. A tile has `width`
// columns (32 or 64) of which the first `valid` exist. Every row sees all of the
// tiles [all0, all1).
struct Tiles {
  int hi, lo, end, ns, n, all0, all1;
  __device__ __forceinline__ Tiles(const Rows& a, int r0, int nrows) {
    int p0 = 0, p1 = 0;
    lo = hi = 0, end = a.len;
    if (!a.prefix) {
      p0 = a.start + r0 / a.g, p1 = a.start + (r0 + nrows - 1) / a.g;
      lo = window_first(p0, a.window), hi = min(a.sinks, lo), end = p1 + 1;
    }
    ns = (hi + KT - 1) / KT;
    n = ns + (end - lo + KT - 1) / KT;
    // behind the start of the last row's window, and not past the first row
    all0 = ns + (a.window > 0 ? (max(window_first(p1, a.window) - lo, 0) + KT - 1) / KT : 0);
    all1 = ns + ((a.prefix ? end : p0 + 1) - lo) / KT;
  }
  __device__ __forceinline__ bool all(int i) const { return i >= all0 && i < all1; }
  __device__ __forceinline__ int first(int i) const { return i < ns ? i * KT : lo + (i - ns) * KT; }
  __device__ __forceinline__ int valid(int i) const { return min(KT, (i < ns ? hi : end) - first(i)); }
  __device__ __forceinline__ int width(int i) const { return all(i) || valid(i) > 32 ? 64 : 32; }
};

template <int T, int D, bool LONG>
__global__ void __launch_bounds__(THREADS, (Cfg<T, D>::CTAS))
    k_rows(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Rows a) {
  using F = Cfg<T, D>;
  using Q = typename Types<T>::Q;
  using C = typename Types<T>::C;
  constexpr bool PAIR = F::PAIR;
  static_assert(!(PAIR && LONG), "fp32 queries fold every tile");
  constexpr uint32_t BF = std::is_same<C, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem + F::Q_BYTES;  // K and V of ring place 0, of place 1, ...
  // s_full: scores computed, and with them the K tile free again; o_full: output added, and with it the V tile. One of
  // each for every ring place, because a parity must not come round before its last reader has come by: a softmax warp
  // may wait for a product when the next one is done too.
  __shared__ uint64_t q_full, k_full[F::RING], v_full[F::RING], s_full[F::RING], o_full[F::RING], p_full[2], drained;
  __shared__ uint32_t tmem_at;
  __shared__ float s_row[PAIR ? ROWS : 1];  // fp32 queries: what makes a row's scores powers of two
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // blockIdx.x counts ranks, then KV heads, then row tiles, the longest rows first
  const int nranks = a.nranks, rank = blockIdx.x % nranks, kh = blockIdx.x / nranks % a.kv_heads;
  const int r0 = (int)((gridDim.x - 1 - blockIdx.x) / nranks / a.kv_heads) * ROWS;
  const int nrows = min(ROWS, a.rows - r0);
  const Tiles tiles(a, r0, nrows);
  const int i0 = (int)((long long)tiles.n * rank / nranks), i1 = (int)((long long)tiles.n * (rank + 1) / nranks);
  const int count = i1 - i0;

  auto fresh = [](int k) { return LONG ? k % FOLD == 0 : k == 0; };  // 16-bit queries: O starts from zero at the k-th tile

  if (tid == 0) {
    mbar_init(&q_full, 4);
    for (int i = 0; i < F::RING; i++) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < 2; i++) mbar_init(&p_full[i], 4);
    mbar_init(&drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&tmem_at, COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  pdl_wait();  // up to here the kernel may run beside the one before it
  if (nranks > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");

  if (warp < 2) {
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- producer
      bool ok = true;
      int nk = 0, nv = 0;
      auto load = [&](const CUtensorMap* map, int& k, uint64_t* full, uint64_t* free, int at) {
        const int st = k % F::RING;
        if (!ok || (k >= F::RING && !(ok = lane_wait(&free[st], (k / F::RING - 1) & 1)))) return;
        mbar_expect_tx(&full[st], F::TILE);
#pragma unroll
        for (int c = 0; c < D / 64; c++)
          tma_load_3d(ring + 2 * st * F::TILE + at + c * F::KV_CHUNK, map, 64 * c, tiles.first(i0 + k), kh, &full[st]);
        k++;
      };
      // in the order in which the places come free: the scores of tile k + 1 are computed before the output of tile k - 1
      while (ok && nv < count) {
        if (nk < count) load(&map_k, nk, k_full, s_full, 0);
        if (nk > nv + 1 || nk == count) load(&map_v, nv, v_full, o_full, F::TILE);
      }
      if (!ok) report(BAD_WAIT);
      // the copies land before the CTA's shared memory is used for anything else
      for (int k = max(0, nk - F::RING); k < nk; k++) lane_wait(&k_full[k % F::RING], (k / F::RING) & 1);
      for (int k = max(0, nv - F::RING); k < nv; k++) lane_wait(&v_full[k % F::RING], (k / F::RING) & 1);
    } else if (warp == 1 && count > 0) {
      // -------------------------------------------------------------- MMAs
      constexpr uint32_t IDESC_PV = idesc_f16(ROWS, D, true) | BF;
      const uint32_t tm = uniform(tmem), q0 = uniform(smem_u32(smem)), ring0 = uniform(smem_u32(ring));
      bool ok = warp_wait(&q_full, 0);
      auto qk = [&](int k) {  // this CTA's k-th tile
        const int st = k % F::RING;
        if (k >= count || !ok || !(ok = warp_wait(&k_full[st], (k / F::RING) & 1))) return;
        tc_fence_after();
        const uint32_t idesc = idesc_f16(ROWS, tiles.width(i0 + k), false) | BF;
        const uint32_t d = tm + KT * (k & 1);
        const uint64_t kb = smem_desc_sw128(ring0 + 2 * st * F::TILE), qb = smem_desc_sw128(q0);
#pragma unroll
        for (int h = 0; h < (PAIR ? 2 : 1); h++)
#pragma unroll
          for (int kk = 0; kk < D / 16; kk++)
            mma_ss(d, qb + (((PAIR ? 1 - h : 0) * F::Q_TILE + (kk >> 2) * F::Q_CHUNK + (kk & 3) * 32) >> 4),
                   kb + (((kk >> 2) * F::KV_CHUNK + (kk & 3) * 32) >> 4), idesc, h || kk);
        commit(&s_full[st]);
      };
      qk(0);
      qk(1);
      for (int k = 0; k < count && ok; k++) {
        const int st = k % F::RING;
        if (!(ok = warp_wait(&v_full[st], (k / F::RING) & 1))) break;
        const uint32_t vb = ring0 + (2 * st + 1) * F::TILE;
        const int width = tiles.width(i0 + k), valid = tiles.all(i0 + k) ? KT : tiles.valid(i0 + k);
        if (valid < width) {  // rows that no query sees: their weights are 0, so they must be finite
          uint8_t* v = ring + (2 * st + 1) * F::TILE;
#pragma unroll
          for (int c = 0; c < D / 64; c++)
            for (int o = valid * 128 + 16 * lane; o < width * 128; o += 512)
              *(uint4*)(v + c * F::KV_CHUNK + o) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
          __syncwarp();
        }
        if (!(ok = warp_wait(&p_full[k & 1], (k >> 1) & 1))) break;
        tc_fence_after();
        const uint32_t d = tm + COL_O + D * (k & (F::OBUF - 1)), p = tm + KT * (k & 1);
        const uint64_t v = smem_desc_mn_sw128(vb, F::KV_CHUNK);
#pragma unroll
        for (int h = 0; h < (PAIR ? 2 : 1); h++)  // 32 columns of S hold 16 columns of weights, and behind them their low parts
#pragma unroll
          for (int kk = 0; kk < KT / 16; kk++)
            if (kk < 2 || 16 * kk < width)
              mma_ts(d, p + 32 * (kk >> 1) + 8 * (kk & 1) + (PAIR && h == 0 ? 16 : 0), v + kk * (2048 >> 4), IDESC_PV,
                     h || kk ? 1u : (!PAIR && !fresh(k)));
        // The scores of the tile after next take the place of these weights: MMAs run in order. Its commit goes first
        // where O is rarely waited for (a commit costs the issuing warp ~200 cycles).
        if (PAIR) commit(&o_full[st]);
        qk(k + 2);
        if (!PAIR) commit(&o_full[st]);
      }
      if (!ok) {
        commit(&drained);  // no product is left in flight when the tensor memory goes
        warp_wait(&drained, 0);
        if (lane == 0) report(BAD_WAIT);
      }
    }
  } else {
    // -------------------------------------------------------------- softmax
    const int quarter = warp & 3, row = quarter * 32 + lane;  // TMEM lanes by warp % 4
    const int R = r0 + min(row, nrows - 1), tok = R / a.g, head = kh * a.g + R % a.g;
    const bool live = row < nrows;
    {
      // Rows behind the last are copies of it. fp32: a row's 8-value pieces go to neighbouring threads (3840 tokens 98.8
      // -> 96.9 us). 16 bits: a thread loads its own row; the other way took 238 instead of 232 us for 8192 tokens of 128
      // values, and 114 instead of 115 us for 256 sessions behind a prefix.
#pragma unroll
      for (int k = 0; k < D / 8; k++) {
        const int i = tid - 64 + 128 * k, qr = PAIR ? i / (D / 8) : row, c = PAIR ? i % (D / 8) : k;
        const int QR = r0 + min(qr, nrows - 1), qt = QR / a.g;
        const Q* q = (const Q*)a.q + (size_t)qt * a.q_stride + (size_t)(kh * a.g + QR - qt * a.g) * D + 8 * c;
        uint8_t* chunk = smem + (c >> 3) * F::Q_CHUNK;
        if constexpr (PAIR) {
          const float4 u = *(const float4*)q, v = *(const float4*)(q + 4);
          const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
          uint32_t h[4], l[4];
          const float back = pairs<D / 8>(f, h, l);
          if (c == 0) s_row[qr] = fmaxf(back * a.scale2, 0x1p-126f);  // > 0: masked scores are -inf times it
          st_piece(chunk, qr, c & 7, make_uint4(h[0], h[1], h[2], h[3]));
          st_piece(chunk + F::Q_TILE, qr, c & 7, make_uint4(l[0], l[1], l[2], l[3]));
        } else {
          st_piece(chunk, qr, c & 7, *(const uint4*)q);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      if (PAIR) asm volatile("bar.sync 1, 128;" ::: "memory");  // s_row
    }
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t obase = mine + COL_O;
    const float sc = PAIR ? s_row[PAIR ? row : 0] : a.scale2;
    const int p = a.start + tok;
    const int wlo = a.window > 0 ? p - a.window + 1 : -0x40000000;
    float m = -INFINITY, l = 0.f, alpha_last = 0.f;
    float o[PAIR ? D : 1] = {};  // fp32 queries: the running output
    bool ok = true;
    auto wait_o = [&](int k) {  // the k-th product has been added
      if (ok) ok = warp_wait(&o_full[k % F::RING], (k / F::RING) & 1);
      tc_fence_after();
    };
    auto fold = [&](int k) {  // O of the k-th tile, whose maximum came with alpha_last
      if constexpr (PAIR) {
        wait_o(k);
        __syncwarp();
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
          uint32_t v[32];
          tmem_ld32(obase + D * (k & (F::OBUF - 1)) + 32 * c, v);
#pragma unroll
          for (int e = 0; e < 32; e++) o[32 * c + e] = fmaf(o[32 * c + e], alpha_last, __uint_as_float(v[e]));
        }
      }
    };
    // LONG: every FOLD tiles O moves, before it starts from zero again, into the running output of the tiles
    // before, which is rarely touched and lies in local memory, with the maximum that it is relative to behind it
    float far[LONG ? D + 1 : 1];
    far[LONG ? D : 0] = -INFINITY;
    auto move_far = [&](bool empty) {
      const float by = far[D] == -INFINITY ? 0.f : exp2_fast(far[D] - m);
#pragma unroll 1
      for (int c = 0; c < D / 32; c++) {
        uint32_t v[32];
        tmem_ld32(obase + 32 * c, v);
#pragma unroll
        for (int e = 0; e < 32; e++)
          far[32 * c + e] = empty ? __uint_as_float(v[e]) : fmaf(far[32 * c + e], by, __uint_as_float(v[e]));
      }
      far[D] = m;
    };
    auto add_far = [&](int c, uint32_t(&v)[32]) {
      if constexpr (LONG)
        if (count > FOLD) {
          const float by = far[D] == -INFINITY ? 0.f : exp2_fast(far[D] - m);
#pragma unroll
          for (int e = 0; e < 32; e++) v[e] = __float_as_uint(fmaf(far[32 * c + e], by, __uint_as_float(v[e])));
        }
    };
    for (int k = 0; k < count; k++) {
      const int i = i0 + k;
      if (ok) ok = warp_wait(&s_full[k % F::RING], (k / F::RING) & 1);
      if (!ok) break;
      __syncwarp();
      tc_fence_after();
      const uint32_t sbase = mine + KT * (k & 1);
      bool upper = true;  // the tile has its second 32 columns
      uint32_t v[2][32];
      float mx = -INFINITY;
      auto load = [&](int c) { tmem_ld32_nowait(sbase + 32 * c, v[c]); };
      auto most = [&](int c) {
        float mx = -INFINITY, my = -INFINITY;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          mx = max3(mx, __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
          my = max3(my, __uint_as_float(v[c][e + 2]), __uint_as_float(v[c][e + 3]));
        }
        return fmaxf(mx, my);
      };
      // the loads stand in both branches, so that the selects of one are not executed for the other
      if (tiles.all(i)) {
        load(0);
        load(1);
        tmem_wait_ld();
        mx = fmaxf(most(0), most(1));
      } else {
        const int valid = tiles.valid(i);
        upper = valid > 32;
        load(0);
        if (upper) load(1);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 2; c++)
          if (c == 0 || upper) {
            uint32_t see = low_bits(valid - 32 * c);  // of these columns, those that the row sees
            if (!a.prefix && i >= tiles.ns) {
              const int j0 = tiles.first(i) + 32 * c;
              see &= low_bits(p + 1 - j0) & (~low_bits(wlo - j0) | low_bits(a.sinks - j0));
            }
#pragma unroll
            for (int e = 0; e < 32; e++) v[c][e] = see >> e & 1 ? v[c][e] : 0xff800000u;
            mx = fmaxf(mx, most(c));
          }
      }
      mx = mx * sc - TOP<T>;
      if constexpr (LONG)
        if (k > 0 && fresh(k)) {
          wait_o(k - 1);
          __syncwarp();
          move_far(k == FOLD);
        }
      float alpha = 1.f;
      if (PAIR || __any_sync(0xffffffffu, mx > m + GROWTH)) {
        const float mn = fmaxf(m, mx);
        alpha = m == -INFINITY ? 0.f : exp2_fast(m - mn);
        if (!PAIR && !fresh(k)) {
          wait_o(k - 1);
          __syncwarp();
#pragma unroll
          for (int c = 0; c < D / 32; c++) {
            uint32_t w[32];
            tmem_ld32(obase + 32 * c, w);
#pragma unroll
            for (int e = 0; e < 32; e++) w[e] = __float_as_uint(__uint_as_float(w[e]) * alpha);
            tmem_st16(obase + 32 * c, w);
            tmem_st16(obase + 32 * c + 16, w + 16);
          }
        }
        l *= alpha;
        m = mn;
      }
      if (F::OBUF == 1 && k > 0) fold(k - 1);
      const float ms = m == -INFINITY ? 0.f : m;  // a row that has seen nothing yet: its weights are all 0
      const uint64_t sc2 = two(sc, sc), ms2 = two(-ms, -ms);
      uint64_t la = 0, lb = 0;  // pairs of 0.f
#pragma unroll
      for (int c = 0; c < 2; c++)
        if (c == 0 || upper) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const float2 z = one(fma2(two(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1])), sc2, ms2));
            const float u = exp2_fast(z.x), w = exp2_fast(z.y);
            if (e & 1)
              lb = add2(lb, two(u, w));
            else
              la = add2(la, two(u, w));
            hi[e] = pack(C(), u, w);
            if constexpr (PAIR) lo[e] = rest(hi[e], u, w);
          }
          tmem_st16(sbase + 32 * c, hi);
          if constexpr (PAIR) tmem_st16(sbase + 32 * c + 16, lo);
        }
      const float2 sum = one(add2(la, lb));
      l += sum.x + sum.y;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[k & 1]);
      if (F::OBUF == 2 && k > 0) fold(k - 1);
      alpha_last = alpha;
    }
    const bool has = count > 0;
    if (has) {
      if constexpr (PAIR)
        fold(count - 1);
      else
        wait_o(count - 1);
    }
    if (!ok && lane == 0) report(BAD_WAIT);
    // ------------------------------------------------------------ epilogue
    if (nranks == 1) {
      const float inv = l == 0.f && m == -INFINITY ? 0.f : 1.f / l;
      const size_t at = (size_t)kh * a.rows + R;
      if (has) {
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
          uint32_t v[32];
          __syncwarp();
          if constexpr (PAIR) {
#pragma unroll
            for (int e = 0; e < 32; e++) v[e] = __float_as_uint(o[32 * c + e]);
          } else {
            tmem_ld32(obase + 32 * c, v);
            add_far(c, v);
          }
          const int col = 32 * c;
          if (live) {
            if (a.prefix)
              store_row<float>(a.part + at * D + col, v, 1.f);
            else
              store_row<Q>((Q*)a.out + (size_t)tok * a.out_stride + (size_t)head * D + col, v, inv);
          }
        }
        if (live) {
          if (a.prefix)
            a.part_ml[at] = make_float2(m, l);
          else if (a.lse)
            a.lse[(size_t)tok * a.heads + head] = log_sum<T>(m, l);
        }
      }
    } else {
      // every CTA of the cluster is past its ring and its queries: row r goes to CTA r % nranks, behind the parts of lower ranks
      asm volatile("bar.sync 1, 128;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;\nbarrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
      const int each = (ROWS + nranks - 1) / nranks;  // rows of a CTA
      float* so = (float*)smem;
      float2* s_ml = (float2*)(smem + ROWS * F::STRIDE * 4);
      const int at = rank * each + row / nranks;
      if (row < nrows) {
        const uint32_t ml_at = peer(&s_ml[at], row % nranks);
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(ml_at), "f"(has ? m : -INFINITY), "f"(has ? l : 0.f)
                     : "memory");
      }
      if (has) {
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
          uint32_t v[32];
          __syncwarp();
          if constexpr (PAIR) {
#pragma unroll
            for (int e = 0; e < 32; e++) v[e] = __float_as_uint(o[32 * c + e]);
          } else {
            tmem_ld32(obase + 32 * c, v);
            add_far(c, v);
          }
          if (row < nrows) {
            const uint32_t to = peer(&so[at * F::STRIDE + 32 * c], row % nranks);
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + 4 * e), "r"(v[e]), "r"(v[e + 1]),
                           "r"(v[e + 2]), "r"(v[e + 3])
                           : "memory");
          }
        }
      }
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
      // this CTA's rows, 4 columns to a thread
      constexpr int PER = D / 4;
      const int c = tid % PER * 4;
      for (int k = (tid - 64) / PER; k * nranks + rank < nrows; k += 128 / PER) {
        float M = -INFINITY, L = 0.f;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int y = 0; y < nranks; y++) M = fmaxf(M, s_ml[y * each + k].x);
        for (int y = 0; y < nranks; y++) {
          const float2 ml = s_ml[y * each + k];
          // that CTA has no part, and sent no output (one whose scores are all NaN has: its sum is NaN)
          if (ml.x == -INFINITY && ml.y == 0.f) continue;
          const float wt = exp2f(ml.x - M);
          const float4 q4 = *(const float4*)(so + (y * each + k) * F::STRIDE + c);
          L = fmaf(wt, ml.y, L);
          f.x = fmaf(wt, q4.x, f.x), f.y = fmaf(wt, q4.y, f.y), f.z = fmaf(wt, q4.z, f.z), f.w = fmaf(wt, q4.w, f.w);
        }
        const int R2 = r0 + k * nranks + rank, tok2 = R2 / a.g, head2 = kh * a.g + R2 % a.g;
        const size_t at2 = (size_t)kh * a.rows + R2;
        if (a.prefix) {
          *(float4*)(a.part + at2 * D + c) = f;
          if (c == 0) a.part_ml[at2] = make_float2(M, L);
        } else {
          const float inv = 1.f / L;
          store4((Q*)a.out + (size_t)tok2 * a.out_stride + (size_t)head2 * D + c,
                 make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv));
          if (c == 0 && a.lse) a.lse[(size_t)tok2 * a.heads + head2] = log_sum<T>(M, L);
        }
      }
    }
    __syncwarp();
  }
  if (nranks > 1 && warp < 2) {
    // the issuing warps' part in the softmax warps' three cluster barriers; their copies and products are done
    __syncwarp();
    asm volatile(
        "barrier.cluster.wait.acquire;\nbarrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n"
        "barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
}

// CTAs that split one block's positions: as many as fill the SMs, each with a tile of its own at least.
int split(int blocks, int tiles) {
  int n = 1;
  while (n < 8 && 2ll * n * blocks <= 2 * 148 && 2 * n <= tiles) n *= 2;
  return n;
}

template <int T, int D, bool LONG>
cudaError_t launch(const Rows& a, const void* k, const void* v, int ctx, cudaStream_t s) {
  using F = Cfg<T, D>;
  CUtensorMap mk, mv;
  cudaError_t e = map_cache(&mk, k, a.kv_heads, ctx, D, KT);
  if (e == cudaSuccess) e = map_cache(&mv, v, a.kv_heads, ctx, D, KT);
  if (e != cudaSuccess) return e;
  auto* f = k_rows<T, D, LONG>;
  static unsigned long long done = 0;
  static std::mutex mu;
  once_per_device(done, mu, [f] { cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM); });
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3((unsigned)a.nranks * a.kv_heads * ((a.rows + ROWS - 1) / ROWS));
  c.blockDim = dim3(THREADS);
  c.dynamicSmemBytes = F::SMEM;
  c.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.nranks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits for what is before it (pdl_wait)
  at[1].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = 2;
  return cudaLaunchKernelEx(&c, f, mk, mv, a);
}

// `tiles` is the number of position tiles of the last block of rows, which has the most. The fold's own instructions
// cost 3% where nothing is folded (8192 tokens behind a window of 1500: 209 instead of 203 us).
cudaError_t by_type(int type, int d, Rows a, const void* k, const void* v, int ctx, int tiles, cudaStream_t s) {
  a.nranks = split((a.rows + ROWS - 1) / ROWS * a.kv_heads, tiles);
  const bool lng = (tiles + a.nranks - 1) / a.nranks > FOLD;
  auto with = [&](auto t, auto d) {
    constexpr int T = decltype(t)::value, D = decltype(d)::value;
    if constexpr (T == T_F32)
      return launch<T, D, false>(a, k, v, ctx, s);
    else
      return lng ? launch<T, D, true>(a, k, v, ctx, s) : launch<T, D, false>(a, k, v, ctx, s);
  };
  using I = std::integral_constant<int, 64>;
  using J = std::integral_constant<int, 128>;
  auto with_d = [&](auto t) { return d == 64 ? with(t, I()) : with(t, J()); };
  return type == T_F32   ? with_d(std::integral_constant<int, T_F32>())
         : type == T_F16 ? with_d(std::integral_constant<int, T_F16>())
                         : with_d(std::integral_constant<int, T_BF16>());
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }
}  // namespace

cudaError_t window(const Prompt& a, cudaStream_t s) {
  Rows r = {};
  r.heads = a.heads, r.kv_heads = a.kv_heads, r.g = a.heads / a.kv_heads, r.rows = a.n * r.g;
  r.scale2 = a.scale * LOG2E;
  r.q = a.q, r.q_stride = a.q_stride;
  r.start = a.start, r.window = a.window, r.sinks = a.sinks;
  r.out = a.out, r.out_stride = a.out_stride, r.lse = a.lse;
  const int last = a.start + a.n - 1, tok = std::min(a.n, ROWS / r.g);
  const int lo = window_first(last - tok + 1, a.window), hi = std::min(a.sinks, lo);
  return by_type(a.type, a.d, r, a.k, a.v, a.ctx, (hi + KT - 1) / KT + (last - lo + KT) / KT, s);
}

// Partial outputs and statistics of the prefix, one of each row.
size_t shared_workspace(const Decode& a) {
  const size_t rows = (size_t)a.batch * a.heads;
  return a.prefix_len ? up16(rows * a.d * 4) + rows * 8 : 16;
}

cudaError_t shared(const Decode& a, cudaStream_t s) {
  if (!a.prefix_len) return decode(a, s);
  Rows r = {};
  r.heads = a.heads, r.kv_heads = a.kv_heads, r.g = a.heads / a.kv_heads, r.rows = a.batch * r.g;
  r.scale2 = a.scale * LOG2E;
  r.q = a.q, r.q_stride = a.q_stride;
  r.prefix = true, r.len = a.prefix_len;
  r.part = (float*)a.work;
  r.part_ml = (float2*)((char*)a.work + up16((size_t)a.batch * a.heads * a.d * 4));
  cudaError_t e = by_type(a.type, a.d, r, a.pk, a.pv, a.prefix_ctx, (a.prefix_len + KT - 1) / KT, s);
  if (e != cudaSuccess) return e;
  return decode_joined(a, r.part, r.part_ml, s);
}

cudaError_t status_word_tc(unsigned** at) { return status_word(at); }

}  // namespace cache
}  // namespace lfm
