// One token of each session over its own cache (lfm_attention_decode), and the
// own-cache half of lfm_attention_shared with the join of both halves.
//
// A cluster of C CTAs takes one KV head of one session and splits the positions
// that its query sees; each of a CTA's warps walks its own chunks of 4 KB of
// K and 4 KB of V (32 positions of 64 values, 16 of 128). A chunk's rows lie
// one behind the other in memory, so a warp's lane 0 fetches it with one bulk
// copy each (two where it spans the end of the sinks) into the warp's private
// ring; nothing but the ring's own mbarriers is waited for until the end.
//
// Products on m16n8k16 matrix instructions: rows are the KV head's up to 8
// query heads. For fp32 queries the row r + 8 holds what the fp16 row r leaves
// off (hi/lo pairs of q and of the weights), so one instruction does both halves
// and the sum of the two accumulator rows, which one thread holds, has ~22 bits.
//   A chunk's output is added to the running one in fp32: accumulated in the
//       matrix unit, which cuts its sums off, outputs came out smaller by 1.6e-5
//       of themselves over 2048 positions of a warp and by 6.6e-5 over 8192.
//   S = Q K^T: a lane reads 16 bytes of one key's row; the order of the
//       head_dim terms that this gives the instruction's k index is the same
//       for q, whose fragments are laid out to match. No transposed load.
//   O = P V: the scores' accumulator layout is the weights' operand layout; a
//       lane reads the same 16 bytes of 4 positions and pairs them by byte
//       permutes; output column n of tile e is head_dim index 8 n + e.
// Statistics and outputs stay in fp32; exponentials are of powers of two (the
// scores carry scale * log2 e), relative to the maximum less SHIFT
// (cache_common.cuh). 16-bit queries: the weights are rounded to the caches'
// type, half a step each (fp16 2^-11, bf16 2^-8), as the caller's V and output
// are; the sums l are of the weights as they were. (Pairs in the rows that 16-bit
// queries leave free take the error from 2.3e-4 to 2.1e-4 in fp16 and from 2.1e-3
// to 1.6e-3 in bf16, and 24 long fp16 sessions with weights from 361 to 390 us,
// 64 bf16 sessions of up to 4096 positions from 124 to 135 us: not taken.)
// The warps join through shared memory, the CTAs through the cluster's: each
// sends its part of the columns to the CTA that finishes them, so a call is one
// launch without workspace. Accumulated weights need the joined statistics: a CTA
// keeps its scores in shared memory until the join, or, where they would not fit,
// reads K once more.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "cache_attn.h"
#include "cache_common.cuh"
#include "host_once.h"

namespace lfm {
namespace cache {
namespace {
using namespace dev;

constexpr int STAGES = 2, HALF = 4096, STAGE = 2 * HALF;
constexpr float LOG2E = 1.4426950408889634f;
enum Acc { NO_ACC = 0, STORED = 1, AGAIN = 2 };
// Warps of a CTA. 4: three CTAs to an SM. 3: four, where that saves a second round, from 3 x 148 + 1 to 4 x 148 CTAs
// without weights (64 windowed sessions of 8 heads, 512 CTAs: 24 instead of 30 us; 56 of 4096 positions, 448 CTAs: 74
// instead of 90; 74 of 1000, 592 CTAs: 54 instead of 64; 64 of 64 positions: 11.1 instead of 10.7; 64 of 100 to 3000
// positions, where rounds end apart anyway: 90 instead of 82). 7: where the scores are kept, one CTA with what its ring
// leaves of shared memory (24 sessions of up to 32768 positions, 6 heads of 128 values to a KV head, with weights: 361 us;
// before this, reading K again 487 us; without weights 295 us).
constexpr int warps_of(int acc) { return acc == STORED ? 7 : 4; }
constexpr int ctas_of(int warps) { return warps == 3 ? 4 : warps == 4 ? 3 : 1; }  // to an SM, by their rings
constexpr int ring_of(int warps) { return warps * STAGES * STAGE; }
constexpr int SCORE_BYTES = 227 * 1024 - ring_of(warps_of(STORED)) - 6 * 1024;

template <class C>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<C, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The weight of a part whose maximum is m under the joint maximum M (no part: 0).
__device__ __forceinline__ float part_weight(float m, float M) { return m == -INFINITY ? 0.f : exp2f(m - M); }

struct Joint {
  const float* o;    // the prefix's part [kv head][row][D], not divided by l; null: none
  const float2* ml;  // its (m in log2 units, l) [kv head][row]
};

template <int T, int D, int ACC, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, ctas_of(WARPS)) k_decode(Decode a, Joint pre, int cap) {
  using Q = typename Types<T>::Q;
  using C = typename Types<T>::C;
  constexpr int RING = ring_of(WARPS);
  constexpr int KC = HALF / (2 * D);  // positions of a chunk
  constexpr int NU = D / 64, TILES = KC / 8;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* scores = (float*)(smem + RING);  // STORED: [head][cap]
  __shared__ uint64_t full[WARPS][STAGES];
  __shared__ __align__(16) float4 s_o[8 * D / 4 + 16];  // this CTA's share of the columns, from every CTA: [CTA][item]
  __shared__ float2 s_ml[8][8];                    // every CTA's statistics
  __shared__ float w_m[WARPS][8], w_l[WARPS][8], f_m[8], f_inv[8], f_pre[8];
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, r = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x, nranks = gridDim.x, kh = blockIdx.y, b = blockIdx.z;
  const int g = a.heads / a.kv_heads;

  // what is before this kernel, or, behind the prefix's kernel, which has waited for that, later: that kernel's part
  if (!pre.o) pdl_wait();
  int slot, len;
  const bool good = session(a.slots, a.lens, b, a.n_slots, a.max_len, &slot, &len);
  if (!good) slot = len = 0;
  const int lo = window_first(len - 1, a.window), hi = min(a.sinks, lo);
  const int n = hi + len - lo;  // positions seen, counted through
  const int chunks = (n + KC - 1) / KC;
  const int c0 = (int)((long long)chunks * rank / nranks), c1 = (int)((long long)chunks * (rank + 1) / nranks);
  const size_t base = (size_t)slot * a.slot_stride + (size_t)kh * a.ctx * D;
  const C *kg = (const C*)a.k + base, *vg = (const C*)a.v + base;
  uint8_t* ring = smem + w * STAGES * STAGE;
  if (nranks > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");

  if (lane < STAGES) mbar_init(&full[w][lane], 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncwarp();
  const int mine = c1 - c0 > w ? (c1 - c0 - w + WARPS - 1) / WARPS : 0;  // this warp's chunks
  auto fetch = [&](int i, int st, bool with_v) {
    const int i0 = (c0 + w + i * WARPS) * KC, i1 = min(i0 + KC, n);
    uint8_t* dst = ring + st * STAGE;
    mbar_expect_tx(&full[w][st], (with_v ? 2 : 1) * (i1 - i0) * 2 * D);
    const int ns = max(0, min(i1, hi) - i0), nw = i1 - i0 - ns;  // of the sinks, of the window
    const int jw = lo + i0 + ns - hi;
    if (ns) {
      bulk_g2s(dst, kg + (size_t)i0 * D, ns * 2 * D, &full[w][st]);
      if (with_v) bulk_g2s(dst + HALF, vg + (size_t)i0 * D, ns * 2 * D, &full[w][st]);
    }
    if (nw) {
      bulk_g2s(dst + ns * 2 * D, kg + (size_t)jw * D, nw * 2 * D, &full[w][st]);
      if (with_v) bulk_g2s(dst + HALF + ns * 2 * D, vg + (size_t)jw * D, nw * 2 * D, &full[w][st]);
    }
  };
  if (lane == 0)
    for (int i = 0; i < min(mine, STAGES); i++) fetch(i, i, true);

  // the query fragments: k step 2 s of head_dim segment [32 s, 32 s + 32) takes a lane's values 0-3 of 8, step 2 s + 1 the others
  constexpr bool PAIR = T == T_F32;
  uint32_t qf[D / 16][4];
  float post = a.scale * LOG2E;
  {
    const Q* q = (const Q*)a.q + (size_t)b * a.q_stride + (size_t)(kh * g + min(r, g - 1)) * D + 8 * t;
    if constexpr (PAIR) {
      float f[D / 32][8], most = 0.f;
#pragma unroll
      for (int s = 0; s < D / 32; s++) {
        const float4 x = *(const float4*)(q + 32 * s), y = *(const float4*)(q + 32 * s + 4);
        f[s][0] = x.x, f[s][1] = x.y, f[s][2] = x.z, f[s][3] = x.w;
        f[s][4] = y.x, f[s][5] = y.y, f[s][6] = y.z, f[s][7] = y.w;
        most = fmaxf(most, max_abs(f[s]));
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const float2 by = row_scale(most);
      post *= by.y;
#pragma unroll
      for (int s = 0; s < D / 32; s++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float u = f[s][2 * i] * by.x, v = f[s][2 * i + 1] * by.x;
          const __half2 h = __floats2half2_rn(u, v);
          const float2 back = __half22float2(h);
          const __half2 l = __floats2half2_rn(u - back.x, v - back.y);
          qf[2 * s + (i >> 1)][(i & 1) * 2] = *(const uint32_t*)&h;
          qf[2 * s + (i >> 1)][(i & 1) * 2 + 1] = *(const uint32_t*)&l;
        }
    } else {
#pragma unroll
      for (int s = 0; s < D / 32; s++) {
        const uint4 x = *(const uint4*)(q + 32 * s);
        const uint32_t f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          qf[2 * s + (i >> 1)][(i & 1) * 2] = f[i];
          qf[2 * s + (i >> 1)][(i & 1) * 2 + 1] = 0u;
        }
      }
    }
  }

  // a chunk's scores in log2 units: s[tile][0..1], head r, positions 8 tile + 2 t + {0, 1}; -inf behind the last
  auto score = [&](const uint8_t* kb, int i0, float (&s)[TILES][2]) {
#pragma unroll
    for (int kt = 0; kt < TILES; kt++) {
      float c[4] = {};
#pragma unroll
      for (int x = 0; x < D / 32; x++) {
        const uint4 k = *(const uint4*)(kb + (kt * 8 + r) * 2 * D + 64 * x + 16 * t);
        mma16816<C>(c, qf[2 * x], k.x, k.y);
        mma16816<C>(c, qf[2 * x + 1], k.z, k.w);
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const float v = (PAIR ? c[e] + c[e + 2] : c[e]) * post;
        s[kt][e] = i0 + kt * 8 + 2 * t + e < n ? v : -INFINITY;
      }
    }
  };

  float m = -INFINITY, l = 0.f, o[NU][8][2] = {};  // o: head r, column 64 u + 8 (2 t + x) + e
  bool ok = true;
  // the k-th fetch has landed; if it does not, the ones behind it are waited for too before their place is given up
  auto landed = [&](int k, int end) {
    if (warp_wait(&full[w][k % STAGES], (k / STAGES) & 1)) return true;
    for (int j = k; j < min(k + STAGES, end); j++) warp_wait(&full[w][j % STAGES], (j / STAGES) & 1);
    return false;
  };
  for (int i = 0; i < mine && ok; i++) {
    const int st = i % STAGES, i0 = (c0 + w + i * WARPS) * KC;
    if (!(ok = landed(i, mine))) break;
    uint8_t* kb = ring + st * STAGE;
    uint8_t* vb = kb + HALF;
    if (i0 + KC > n) {  // the rows behind the last hold what was there before: their weights are 0, so they must be finite
      for (int x = (n - i0) * 2 * D + 16 * lane; x < HALF; x += 512) *(uint4*)(vb + x) = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
    float s[TILES][2];
    score(kb, i0, s);
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < TILES; kt++) mx = fmaxf(mx, fmaxf(s[kt][0], s[kt][1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) - SHIFT<T>;
    if constexpr (ACC == STORED) {
      if (r < g) {
        float* dst = scores + r * cap + (i0 - c0 * KC) + 2 * t;
#pragma unroll
        for (int kt = 0; kt < TILES; kt++) *(float2*)(dst + 8 * kt) = make_float2(s[kt][0], s[kt][1]);
      }
    }
    float alpha = 1.f;
    if (__any_sync(0xffffffffu, mx > m)) {
      const float mn = fmaxf(m, mx);
      alpha = part_weight(m, mn);
      m = mn;
      l *= alpha;
    }
    uint32_t p[TILES][2];  // [tile][hi, lo]
#pragma unroll
    for (int kt = 0; kt < TILES; kt++) {
      const float x = exp2_fast(s[kt][0] - m), y = exp2_fast(s[kt][1] - m);
      l += x + y;
      if constexpr (std::is_same<C, __half>::value) {
        const __half2 h = __floats2half2_rn(x, y);
        p[kt][0] = *(const uint32_t*)&h;
        if constexpr (PAIR) {
          const float2 back = __half22float2(h);
          const __half2 lo2 = __floats2half2_rn(x - back.x, y - back.y);
          p[kt][1] = *(const uint32_t*)&lo2;
        } else {
          p[kt][1] = 0u;
        }
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        p[kt][0] = *(const uint32_t*)&h;
        p[kt][1] = 0u;
      }
    }
    // a chunk's output starts from zero and is added in fp32: the matrix unit cuts its sums off
#pragma unroll
    for (int u = 0; u < NU; u++) {
      float c[8][4] = {};
#pragma unroll
      for (int kk = 0; kk < TILES / 2; kk++) {
        const uint32_t pa[4] = {p[2 * kk][0], p[2 * kk][1], p[2 * kk + 1][0], p[2 * kk + 1][1]};
        uint32_t v[4][4];
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const uint4 q4 = *(const uint4*)(vb + (kk * 16 + (x >> 1) * 8 + 2 * t + (x & 1)) * 2 * D + 128 * u + 16 * r);
          v[x][0] = q4.x, v[x][1] = q4.y, v[x][2] = q4.z, v[x][3] = q4.w;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const uint32_t sel = e & 1 ? 0x7632u : 0x5410u;
          mma16816<C>(c[e], pa, __byte_perm(v[0][e >> 1], v[1][e >> 1], sel),
                      __byte_perm(v[2][e >> 1], v[3][e >> 1], sel));
        }
      }
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int x = 0; x < 2; x++) o[u][e][x] = fmaf(o[u][e][x], alpha, PAIR ? c[e][x] + c[e][x + 2] : c[e][x]);
    }
    __syncwarp();
    if (lane == 0 && i + STAGES < mine) fetch(i + STAGES, st, true);
  }

  // join the warps: each leaves its output in its own ring
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (t == 0) {
    w_m[w][r] = m;
    w_l[w][r] = l;
  }
  float* wo = (float*)ring;  // [head][D]
  __syncwarp();
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int x = 0; x < 2; x++) {
      float* dst = wo + r * D + 64 * u + 8 * (2 * t + x);
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const float4 f = make_float4(o[u][e][x], o[u][e + 1][x], o[u][e + 2][x], o[u][e + 3][x]);
        *(float4*)(dst + e) = f;
      }
    }
  if (!ok && lane == 0) report(BAD_WAIT);
  __syncthreads();
  // join the CTAs: item i (head, 4 columns) goes to CTA i % nranks, the statistics to all
  if (nranks > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // they have started
  const int items = g * (D / 4), share = (items + nranks - 1) / nranks;
  for (int i = tid; i < items; i += WARPS * 32) {
    const int h = i / (D / 4);
    float M = -INFINITY;
#pragma unroll
    for (int x = 0; x < WARPS; x++) M = fmaxf(M, w_m[x][h]);
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < WARPS; x++) {
      const float c = part_weight(w_m[x][h], M);
      const float4 y = ((const float4*)(smem + x * STAGES * STAGE))[i];
      f.x = fmaf(c, y.x, f.x), f.y = fmaf(c, y.y, f.y), f.z = fmaf(c, y.z, f.z), f.w = fmaf(c, y.w, f.w);
    }
    if (nranks == 1)
      s_o[i] = f;
    else
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(peer(&s_o[rank * share + i / nranks], i % nranks)),
                   "f"(f.x), "f"(f.y), "f"(f.z), "f"(f.w)
                   : "memory");
  }
  for (int i = tid; i < g * nranks; i += WARPS * 32) {
    const int h = i % g;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int x = 0; x < WARPS; x++) M = fmaxf(M, w_m[x][h]);
#pragma unroll
    for (int x = 0; x < WARPS; x++) L = fmaf(part_weight(w_m[x][h], M), w_l[x][h], L);
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(peer(&s_ml[rank][h], i / g)), "f"(M), "f"(L) : "memory");
  }
  if (nranks > 1) {
    __syncwarp();
    cluster_sync();
  } else {
    __syncthreads();
  }
  if (pre.o) pdl_wait();
  const size_t row0 = ((size_t)kh * a.batch + b) * g;  // of the prefix's part
  if (tid < g) {
    float M = -INFINITY, L = 0.f;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (pre.o) ml = pre.ml[row0 + tid];
    for (int x = 0; x < nranks; x++) M = fmaxf(M, s_ml[x][tid].x);
    M = fmaxf(M, ml.x);
    for (int x = 0; x < nranks; x++) L = fmaf(part_weight(s_ml[x][tid].x, M), s_ml[x][tid].y, L);
    L = fmaf(part_weight(ml.x, M), ml.y, L);
    f_pre[tid] = part_weight(ml.x, M);
    f_m[tid] = M;
    f_inv[tid] = M == -INFINITY && L == 0.f ? 0.f : 1.f / L;  // nothing seen: zeros
  }
  __syncthreads();
  for (int k = tid; k * nranks + rank < items; k += WARPS * 32) {
    const int i = k * nranks + rank, h = i / (D / 4), c = i % (D / 4) * 4;
    const float M = f_m[h], inv = f_inv[h];
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = 0; x < nranks; x++) {
      const float wt = part_weight(s_ml[x][h].x, M);
      const float4 y = s_o[x * share + k];
      f.x = fmaf(wt, y.x, f.x), f.y = fmaf(wt, y.y, f.y), f.z = fmaf(wt, y.z, f.z), f.w = fmaf(wt, y.w, f.w);
    }
    if (pre.o) {
      const float wt = f_pre[h];
      const float4 y = *(const float4*)(pre.o + (row0 + h) * D + c);
      f.x = fmaf(wt, y.x, f.x), f.y = fmaf(wt, y.y, f.y), f.z = fmaf(wt, y.z, f.z), f.w = fmaf(wt, y.w, f.w);
    }
    store4((Q*)a.out + (size_t)b * a.out_stride + (size_t)(kh * g + h) * D + c,
           good ? make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f));
  }
  if constexpr (ACC != NO_ACC) {
    if (good) {
      float* acc = a.acc + ((size_t)slot * a.kv_heads + kh) * a.ctx;
      const int first = c0 * KC, count = min(c1 * KC, n) - first;
      if constexpr (ACC == STORED) {
        for (int i = tid; i < count; i += WARPS * 32) {
          float sum = 0.f;
          for (int h = 0; h < g; h++)
            sum = fmaf(exp2_fast(scores[h * cap + i] - (f_m[h] + SHIFT<T>)), f_inv[h] * exp2f(SHIFT<T>), sum);
          const int j = first + i;
          atomicAdd(acc + (j < hi ? j : lo + j - hi), sum);
        }
      } else {
        // K once more: the ring's barriers go on from the phases that the first walk left
        const float M = f_m[min(r, g - 1)] + SHIFT<T>, inv = r < g ? f_inv[r] * exp2f(SHIFT<T>) : 0.f;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the ring was written by this warp's stores
        __syncthreads();
        if (lane == 0 && ok)
          for (int i = 0; i < min(mine, STAGES); i++) fetch(i, (mine + i) % STAGES, false);
        for (int i = 0; i < mine && ok; i++) {
          const int at = mine + i, st = at % STAGES, i0 = (c0 + w + i * WARPS) * KC;
          if (!(ok = landed(at, 2 * mine))) break;
          float s[TILES][2];
          score(ring + st * STAGE, i0, s);
#pragma unroll
          for (int kt = 0; kt < TILES; kt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float x = exp2_fast(s[kt][e] - M) * inv;
              x += __shfl_xor_sync(0xffffffffu, x, 4);
              x += __shfl_xor_sync(0xffffffffu, x, 8);
              x += __shfl_xor_sync(0xffffffffu, x, 16);
              const int j = i0 + kt * 8 + 2 * t + e;
              if (r == 0 && j < n) atomicAdd(acc + (j < hi ? j : lo + j - hi), x);
            }
          __syncwarp();
          if (lane == 0 && i + STAGES < mine) fetch(i + STAGES, st, false);
        }
        if (!ok && lane == 0) report(BAD_WAIT);
      }
    }
  }
}

template <int T, int D, int ACC, int WARPS = warps_of(ACC)>
cudaError_t launch(const Decode& a, const Joint& pre, int nranks, int cap, cudaStream_t s) {
  const int smem = ring_of(WARPS) + (ACC == STORED ? a.heads / a.kv_heads * cap * 4 : 0);
  auto* f = k_decode<T, D, ACC, WARPS>;
  static unsigned long long done = 0;
  static std::mutex mu;
  once_per_device(done, mu, [f] {
    cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, ring_of(WARPS) + (ACC == STORED ? SCORE_BYTES : 0));
  });
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(nranks, a.kv_heads, a.batch);
  c.blockDim = dim3(WARPS * 32);
  c.dynamicSmemBytes = smem;
  c.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = nranks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel waits for what is before it (pdl_wait)
  at[1].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = 2;
  return cudaLaunchKernelEx(&c, f, a, pre, cap);
}

cudaError_t run(const Decode& a, const Joint& pre, cudaStream_t s) {
  const int kc = HALF / (2 * a.d);
  const long long most = a.window ? std::min<long long>(a.max_len, (long long)a.window + a.sinks) : a.max_len;
  const int chunks = (int)((most + kc - 1) / kc);
  // As many CTAs to a KV head as fill three to an SM, each with chunks for its warps; more where that lets the scores
  // be kept. At most 8: clusters of 16 left most SMs without a second CTA (625 instead of 487 us where K was read again).
  const int g = a.heads / a.kv_heads;
  int nranks = 1;
  // the most positions that one CTA may get, in whole chunks
  auto cap = [&] { return (long long)((chunks + nranks - 1) / nranks) * kc; };
  while (nranks < 8 && chunks > 4 * nranks &&
         ((long long)a.batch * a.kv_heads * nranks < 3 * 148 || (a.acc && cap() * g * 4 > SCORE_BYTES)))
    nranks *= 2;
  const int acc = !a.acc ? NO_ACC : cap() * g * 4 <= SCORE_BYTES ? STORED : AGAIN;
  auto with = [&](auto t, auto d) {
    constexpr int T = decltype(t)::value, D = decltype(d)::value;
    const long long ctas = (long long)a.batch * a.kv_heads * nranks;
    if (acc == NO_ACC && ctas > 3 * 148 && ctas <= 4 * 148) return launch<T, D, NO_ACC, 3>(a, pre, nranks, (int)cap(), s);
    return acc == NO_ACC   ? launch<T, D, NO_ACC>(a, pre, nranks, (int)cap(), s)
           : acc == STORED ? launch<T, D, STORED>(a, pre, nranks, (int)cap(), s)
                           : launch<T, D, AGAIN>(a, pre, nranks, (int)cap(), s);
  };
  using I = std::integral_constant<int, 64>;
  using J = std::integral_constant<int, 128>;
  auto with_d = [&](auto t) { return a.d == 64 ? with(t, I()) : with(t, J()); };
  return a.type == T_F32   ? with_d(std::integral_constant<int, T_F32>())
         : a.type == T_F16 ? with_d(std::integral_constant<int, T_F16>())
                           : with_d(std::integral_constant<int, T_BF16>());
}
}  // namespace

cudaError_t decode(const Decode& a, cudaStream_t s) { return run(a, Joint{nullptr, nullptr}, s); }

cudaError_t decode_joined(const Decode& a, const float* o, const float2* ml, cudaStream_t s) {
  return run(a, Joint{o, ml}, s);
}

cudaError_t status_word_decode(unsigned** at) { return status_word(at); }

}  // namespace cache
}  // namespace lfm
