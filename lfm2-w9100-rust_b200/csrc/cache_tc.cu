// Attention of many query rows over one cache on the tensor cores (tcgen05 /
// TMEM): a prompt's rows under a causal window with sinks
// (lfm_attention_window), and the rows of all sessions over their shared
// prefix (the prefix half of lfm_attention_shared).
//
// Rows are packed: row R of a KV head is query head R % g of token (or session)
// R / g, so every group size fills the 128-row tiles. A CTA holds two tiles of
// rows and walks the positions in tiles of 128, with
//   warp 0      TMA: K and V tiles into one ring of slots
//   warp 1      TMEM and the MMAs: S_x = Q_x K^T, O_x += P_x V for tile x
//   warps 4-7   the softmax of tile 0, warps 8-11 that of tile 1: one thread a row
// While one tile is in its softmax, the products of the other run. The weights
// P take the place of S in tensor memory (a 16-bit operand of half its width)
// and enter the second product from there. For fp32 queries q and P are fp16
// hi/lo pairs, two MMAs each; the pair of weights fills the whole of S.
// O stays in tensor memory; a row's maximum is raised, and O rescaled, only
// when it grows by more than 2^8, which keeps every weight inside fp16's range
// and every rounding relative.
// Few row blocks leave SMs idle, so a cluster of CTAs may split the positions of
// one block and join through distributed shared memory.
// Every wait is bounded; one that runs out is reported and the CTA releases
// its tensor memory.
#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "cache_attn.h"
#include "cache_common.cuh"
#include "host_once.h"
#include "tc_common.cuh"

namespace lfm {
namespace cache {
namespace {
using namespace dev;
using namespace tc;

constexpr int THREADS = 384, KT = 128, ROWS = 256;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Registers of a thread: at launch, after the split between the two kinds of warps.
constexpr int REGS = 168, REGS_ISSUE = 72, REGS_SOFTMAX = 216;
static_assert(128 * REGS_ISSUE + 256 * REGS_SOFTMAX <= THREADS * REGS, "the split asks for more than the launch has");
constexpr float GROWTH = 8.f;  // log2 of what a row may grow before its maximum is raised
constexpr uint32_t COLS = 512, COL_O = 256;  // S_x: [128 x, 128 x + 128); O_x: [256 + D x, + D)

template <int T, int D>
struct Cfg {
  static constexpr bool PAIR = T == T_F32;
  static constexpr int CHUNK = 128 * 128;             // 128 rows x 64 16-bit values, swizzled
  static constexpr int TILE = CHUNK * (D / 64);       // 128 rows x D
  static constexpr int Q_BYTES = 2 * (PAIR ? 2 : 1) * TILE;
  static constexpr int SLOTS = std::min(6, (226 * 1024 - Q_BYTES) / TILE);
  static constexpr int SMEM = Q_BYTES + SLOTS * TILE + 1024;
  static constexpr int STRIDE = D + 4;  // floats of a row in the join: rows of one column start in different banks
  static_assert(SLOTS >= 3 && ROWS * (STRIDE * 4 + 8) <= Q_BYTES + SLOTS * TILE, "shared memory");
};

struct Rows {
  int heads, kv_heads, g, rows;  // rows of one KV head
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

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(
          d),
      "r"(a), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
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
// 16 bytes at column block `piece` (of 8) of row r of a swizzled 64-wide chunk
__device__ __forceinline__ void st_piece(uint8_t* chunk, int r, int piece, uint4 v) {
  *(uint4*)(chunk + r * 128 + ((piece ^ (r & 7)) << 4)) = v;
}

// The position tiles of a block of rows: the sinks in front of the window, then
// the positions from the first row's window to the last row. A tile has `width`
// columns (a multiple of 32) of which the first `valid` exist.
struct Tiles {
  int hi, lo, end, ns, n;
  __device__ __forceinline__ Tiles(int hi_, int lo_, int end_) : hi(hi_), lo(lo_), end(end_) {
    ns = (hi + KT - 1) / KT;
    n = ns + (end - lo + KT - 1) / KT;
  }
  __device__ __forceinline__ int first(int i) const { return i < ns ? i * KT : lo + (i - ns) * KT; }
  __device__ __forceinline__ int valid(int i) const { return min(KT, (i < ns ? hi : end) - first(i)); }
  __device__ __forceinline__ int width(int i) const { return (valid(i) + 31) & ~31; }
};

template <int T, int D>
__global__ void __launch_bounds__(THREADS, 1)
    k_rows(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Rows a) {
  using F = Cfg<T, D>;
  using Q = typename Types<T>::Q;
  using C = typename Types<T>::C;
  constexpr bool PAIR = F::PAIR;
  constexpr uint32_t BF = std::is_same<C, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* slots = smem + F::Q_BYTES;
  __shared__ uint64_t q_full, full[F::SLOTS], empty[F::SLOTS], s_full[2], p_full[2];
  __shared__ uint32_t tmem_at;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, nranks = gridDim.x, kh = blockIdx.y;
  const int r0 = (int)(gridDim.z - 1 - blockIdx.z) * ROWS;  // the longest rows first
  const int nrows = min(ROWS, a.rows - r0);
  const int ntiles_x = nrows > 128 ? 2 : 1;
  const int p0 = a.prefix ? 0 : a.start + r0 / a.g, p1 = a.prefix ? 0 : a.start + (r0 + nrows - 1) / a.g;
  const int lo0 = a.prefix ? 0 : window_first(p0, a.window);
  const Tiles tiles(a.prefix ? 0 : min(a.sinks, lo0), lo0, a.prefix ? a.len : p1 + 1);
  const int i0 = (int)((long long)tiles.n * rank / nranks), i1 = (int)((long long)tiles.n * (rank + 1) / nranks);

  if (tid == 0) {
    mbar_init(&q_full, 8);
    for (int i = 0; i < F::SLOTS; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int x = 0; x < 2; x++) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x], 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&tmem_at, COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  const int count = i1 - i0;
  float2 ml = make_float2(-INFINITY, 0.f);  // this thread's row

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ISSUE));
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- producer
      int n = 0;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, int j) {
        const int st = n % F::SLOTS;
        if (n >= F::SLOTS && !(ok = mbar_wait(&empty[st], (n / F::SLOTS - 1) & 1, nullptr))) return;
        mbar_expect_tx(&full[st], F::TILE);
#pragma unroll
        for (int c = 0; c < D / 64; c++)
          tma_load_3d(slots + st * F::TILE + c * F::CHUNK, map, 64 * c, j, kh, &full[st]);
        n++;
      };
      for (int i = i0; i < i1 && ok; i++) {
        load(&map_k, tiles.first(i));
        if (ok) load(&map_v, tiles.first(i));
      }
      if (!ok) report(BAD_WAIT);
      // the copies land before the CTA's shared memory is used for anything else
      for (int i = max(0, n - F::SLOTS); i < n; i++) mbar_wait(&full[i % F::SLOTS], (i / F::SLOTS) & 1, nullptr);
    } else if (warp == 1 && count > 0) {
      // -------------------------------------------------------------- MMAs
      constexpr uint32_t IDESC_PV = idesc_f16(128, D, true) | BF;
      bool ok = mbar_wait(&q_full, 0, nullptr);
      const bool one = lane == 0;
      auto qk = [&](int x, int i) {  // tile i of the block, slot 2 (i - i0)
        const int n = 2 * (i - i0), st = n % F::SLOTS;
        if (!ok || !(ok = mbar_wait(&full[st], (n / F::SLOTS) & 1, nullptr))) return;
        tc_fence_after();
        if (one) {
          const uint32_t idesc = idesc_f16(128, tiles.width(i), false) | BF;
          const uint32_t d = tmem + 128 * x, kb = smem_u32(slots + st * F::TILE);
          const uint32_t qb = smem_u32(smem) + x * (F::Q_BYTES / 2);
#pragma unroll
          for (int h = 0; h < (PAIR ? 2 : 1); h++)
#pragma unroll
            for (int kk = 0; kk < D / 16; kk++) {
              const uint32_t off = (kk >> 2) * F::CHUNK + (kk & 3) * 32;
              mma_f16(d, smem_desc_sw128(qb + h * F::TILE + off), smem_desc_sw128(kb + off), idesc, h || kk);
            }
        }
      };
      auto pv = [&](int x, int i) {
        const int n = 2 * (i - i0) + 1, st = n % F::SLOTS;
        if (!ok || !(ok = mbar_wait(&full[st], (n / F::SLOTS) & 1, nullptr))) return;
        uint8_t* vb = slots + st * F::TILE;
        const int width = tiles.width(i), valid = tiles.valid(i);
        if (x == 0 && valid < width) {  // rows that no query sees: their weights are 0, so they must be finite
#pragma unroll
          for (int c = 0; c < D / 64; c++)
            for (int o = valid * 128 + 16 * lane; o < width * 128; o += 512)
              *(uint4*)(vb + c * F::CHUNK + o) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
          __syncwarp();
        }
        tc_fence_after();
        if (one) {
          const uint32_t d = tmem + COL_O + D * x, p = tmem + 128 * x, v = smem_u32(vb);
          for (int h = 0; h < (PAIR ? 2 : 1); h++)
            for (int kk = 0; kk < width / 16; kk++)
              mma_ts(d, p + 64 * h + 8 * kk, smem_desc_mn_sw128(v + kk * 2048, F::CHUNK), IDESC_PV, i > i0 || h || kk);
        }
      };
      for (int x = 0; x < ntiles_x; x++) {
        qk(x, i0);
        if (one && ok) mma_commit(&s_full[x]);
      }
      if (one && ok) mma_commit(&empty[0]);
      for (int i = i0; i < i1 && ok; i++) {
        for (int x = 0; x < ntiles_x && ok; x++) {
          if (!(ok = mbar_wait(&p_full[x], (i - i0) & 1, nullptr))) break;
          tc_fence_after();
          pv(x, i);
          if (i + 1 < i1) qk(x, i + 1);
          if (one && ok) mma_commit(&s_full[x]);  // S of the next tile, and O of this one
        }
        if (one && ok) {
          mma_commit(&empty[(2 * (i - i0) + 1) % F::SLOTS]);
          if (i + 1 < i1) mma_commit(&empty[(2 * (i - i0) + 2) % F::SLOTS]);
        }
        __syncwarp();
      }
      if (!ok && one) report(BAD_WAIT);
    }
  } else {
    // -------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    const int x = (warp - 4) >> 2, quarter = warp & 3, rt = quarter * 32 + lane, row = x * 128 + rt;
    const int R = r0 + min(row, nrows - 1), tok = R / a.g, head = kh * a.g + R % a.g;
    const bool live = row < nrows;
    {
      const Q* q = (const Q*)a.q + (size_t)tok * a.q_stride + (size_t)head * D;
      uint8_t* dst = smem + x * (F::Q_BYTES / 2);
#pragma unroll
      for (int c = 0; c < D / 8; c++) {
        uint8_t* chunk = dst + (c >> 3) * F::CHUNK;
        if constexpr (PAIR) {
          const float4 u = *(const float4*)(q + 8 * c), v = *(const float4*)(q + 8 * c + 4);
          const float f[8] = {u.x * a.scale2, u.y * a.scale2, u.z * a.scale2, u.w * a.scale2,
                              v.x * a.scale2, v.y * a.scale2, v.z * a.scale2, v.w * a.scale2};
          uint32_t h[4], l[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            h[e] = pack(__half(), f[2 * e], f[2 * e + 1]);
            l[e] = rest(h[e], f[2 * e], f[2 * e + 1]);
          }
          st_piece(chunk, rt, c & 7, make_uint4(h[0], h[1], h[2], h[3]));
          st_piece(chunk + F::TILE, rt, c & 7, make_uint4(l[0], l[1], l[2], l[3]));
        } else {
          st_piece(chunk, rt, c & 7, *(const uint4*)(q + 8 * c));
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    }
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t sbase = mine + 128 * x, obase = mine + COL_O + D * x;
    const float sc = PAIR ? 1.f : a.scale2;
    const int p = a.start + tok;
    const int wlo = a.window > 0 ? p - a.window + 1 : -0x40000000;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    if (x < ntiles_x) {
      for (int i = i0; i < i1; i++) {
        if (!(ok = mbar_wait(&s_full[x], (i - i0) & 1, nullptr))) break;
        tc_fence_after();
        const int j0 = tiles.first(i), width = tiles.width(i), valid = tiles.valid(i);
        uint32_t s[KT];
#pragma unroll
        for (int c = 0; c < 4; c++) {
          uint32_t v[32];
          if (32 * c < width) {
            tmem_ld32_nowait(sbase + 32 * c, v);
#pragma unroll
            for (int e = 0; e < 32; e++) s[32 * c + e] = v[e];
          }
        }
        tmem_wait_ld();
        // the tile is masked for some row of the block, or ends early
        const bool full_tile =
            valid == KT && (a.prefix || i < tiles.ns ||
                            (j0 + KT - 1 <= p0 && (a.window == 0 || j0 > p1 - a.window || j0 + KT <= a.sinks)));
        if (!full_tile) {
          int cmax = valid - 1, cmin = -1, csink = 0;
          if (!a.prefix && i >= tiles.ns) cmax = min(cmax, p - j0), cmin = wlo - j0, csink = a.sinks - j0;
#pragma unroll
          for (int e = 0; e < KT; e++)
            if (!(e <= cmax && (e >= cmin || e < csink))) s[e] = 0xff800000u;
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; c++)
          if (32 * c < width) {
#pragma unroll
            for (int e = 0; e < 32; e++) mx4[e & 3] = fmaxf(mx4[e & 3], __uint_as_float(s[32 * c + e]));
          }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc;
        if (__any_sync(0xffffffffu, mx > m + GROWTH)) {
          const float mn = fmaxf(m, mx);
          const float alpha = m == -INFINITY ? 0.f : exp2f(m - mn);
          if (i > i0) {
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
              uint32_t v[32];
              tmem_ld32(obase + 32 * c, v);
#pragma unroll
              for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
              tmem_st32(obase + 32 * c, v);
            }
          }
          l *= alpha;
          m = mn;
        }
        const float ms = m == -INFINITY ? 0.f : m;  // a row that has seen nothing yet: its weights are all 0
        float l4[4] = {};
#pragma unroll
        for (int c = 0; c < 4; c++)
          if (32 * c < width) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int e = 0; e < 16; e++) {
              const float u = exp2_fast(fmaf(__uint_as_float(s[32 * c + 2 * e]), sc, -ms));
              const float v = exp2_fast(fmaf(__uint_as_float(s[32 * c + 2 * e + 1]), sc, -ms));
              l4[(2 * e) & 3] += u;
              l4[(2 * e + 1) & 3] += v;
              hi[e] = pack(C(), u, v);
              if constexpr (PAIR) lo[e] = rest(hi[e], u, v);
            }
            tmem_st16(sbase + 16 * c, hi);
            if constexpr (PAIR) tmem_st16(sbase + 64 + 16 * c, lo);
          }
        l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
      }
      if (ok && count > 0) ok = mbar_wait(&s_full[x], count & 1, nullptr);  // the last product
      tc_fence_after();
      if (!ok && lane == 0) report(BAD_WAIT);
    }
    const bool has = x < ntiles_x && count > 0;
    if (has) ml = make_float2(m, l);
    if (nranks == 1 && has) {
      const float inv = l == 0.f && m == -INFINITY ? 0.f : 1.f / l;
      const size_t at = (size_t)kh * a.rows + R;
#pragma unroll
      for (int c = 0; c < D / 32; c++) {
        uint32_t v[32];
        __syncwarp();
        tmem_ld32(obase + 32 * c, v);
        if (live) {
          if (a.prefix) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *(uint4*)(a.part + at * D + 32 * c + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          } else {
            store_row<Q>((Q*)a.out + (size_t)tok * a.out_stride + (size_t)head * D + 32 * c, v, inv);
          }
        }
      }
      if (live) {
        if (a.prefix)
          a.part_ml[at] = ml;
        else if (a.lse)
          a.lse[(size_t)tok * a.heads + head] = (m + log2f(l)) * LN2;
      }
    }
    __syncwarp();
  }
  if (nranks > 1) {
    // the ring and the queries are no longer read: every product and every copy is done
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    float* so = (float*)smem;
    float2* s_ml = (float2*)(smem + ROWS * F::STRIDE * 4);
    if (warp >= 4) {
      const int x = (warp - 4) >> 2, quarter = warp & 3, row = x * 128 + quarter * 32 + lane;
      if (x < ntiles_x && count > 0) {
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
          uint32_t v[32];
          tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + COL_O + D * x + 32 * c, v);
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *(uint4*)(so + row * F::STRIDE + 32 * c + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
      }
      s_ml[row] = ml;
    }
    __syncwarp();
    cluster_sync();
    if (warp >= 4) {
      // each CTA finishes a share of the rows, 4 columns to a thread
      constexpr int PER = D / 4;
      const int c = tid % PER * 4;
      for (int row = rank + (tid - 128) / PER * nranks; row < nrows; row += 256 / PER * nranks) {
        float M = -INFINITY, L = 0.f;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int y = 0; y < nranks; y++) M = fmaxf(M, ld_peer(peer(&s_ml[row].x, y)));
        for (int y = 0; y < nranks; y++) {
          const float mp = ld_peer(peer(&s_ml[row].x, y));
          if (mp == -INFINITY) continue;  // that CTA has no part, and its shared memory no output
          const float wt = exp2f(mp - M);
          const float4 o = ld_peer4(peer(&so[row * F::STRIDE + c], y));
          L = fmaf(wt, ld_peer(peer(&s_ml[row].y, y)), L);
          f.x = fmaf(wt, o.x, f.x), f.y = fmaf(wt, o.y, f.y), f.z = fmaf(wt, o.z, f.z), f.w = fmaf(wt, o.w, f.w);
        }
        const int R = r0 + row, tok = R / a.g, head = kh * a.g + R % a.g;
        const size_t at = (size_t)kh * a.rows + R;
        if (a.prefix) {
          *(float4*)(a.part + at * D + c) = f;
          if (c == 0) a.part_ml[at] = make_float2(M, L);
        } else {
          const float inv = 1.f / L;
          Q* dst = (Q*)a.out + (size_t)tok * a.out_stride + (size_t)head * D + c;
          from_f32(f.x * inv, dst);
          from_f32(f.y * inv, dst + 1);
          from_f32(f.z * inv, dst + 2);
          from_f32(f.w * inv, dst + 3);
          if (c == 0 && a.lse) a.lse[(size_t)tok * a.heads + head] = (M + log2f(L)) * LN2;
        }
      }
    }
    __syncwarp();
    cluster_sync();  // the peers have read this CTA's part
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
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

// A cache slot [kv head][position][d] of 16-bit values, read in boxes of 64 values x 128 positions of one head.
cudaError_t map_cache(CUtensorMap* map, const void* base, int kv_heads, int ctx, int d) {
  EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)ctx, (cuuint64_t)kv_heads};
  const cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)ctx * d * 2};
  const cuuint32_t box[3] = {64, KT, 1}, step[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// CTAs that split one block's positions: as many as fill the SMs, each with a tile of its own at least.
int split(int blocks, int tiles) {
  int n = 1;
  while (n < 8 && 2 * n * blocks <= 148 && 2 * n <= tiles) n *= 2;
  return n;
}

template <int T, int D>
cudaError_t launch(const Rows& a, const void* k, const void* v, int ctx, int tiles, cudaStream_t s) {
  using F = Cfg<T, D>;
  CUtensorMap mk, mv;
  cudaError_t e = map_cache(&mk, k, a.kv_heads, ctx, D);
  if (e == cudaSuccess) e = map_cache(&mv, v, a.kv_heads, ctx, D);
  if (e != cudaSuccess) return e;
  auto* f = k_rows<T, D>;
  static unsigned long long done = 0;
  static std::mutex mu;
  static bool fits = false;
  once_per_device(done, mu, [f] {
    cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
    cudaFuncAttributes at;
    fits = cudaFuncGetAttributes(&at, f) == cudaSuccess && at.numRegs >= REGS;  // else the split would wait for good
  });
  if (!fits) return cudaErrorLaunchOutOfResources;
  const int blocks = (a.rows + ROWS - 1) / ROWS;
  const int nranks = split(blocks * a.kv_heads, tiles);
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(nranks, a.kv_heads, blocks);
  c.blockDim = dim3(THREADS);
  c.dynamicSmemBytes = F::SMEM;
  c.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = nranks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, f, mk, mv, a);
}

cudaError_t by_type(int type, int d, const Rows& a, const void* k, const void* v, int ctx, int tiles, cudaStream_t s) {
  if (type == T_F32)
    return d == 64 ? launch<T_F32, 64>(a, k, v, ctx, tiles, s) : launch<T_F32, 128>(a, k, v, ctx, tiles, s);
  if (type == T_F16)
    return d == 64 ? launch<T_F16, 64>(a, k, v, ctx, tiles, s) : launch<T_F16, 128>(a, k, v, ctx, tiles, s);
  return d == 64 ? launch<T_BF16, 64>(a, k, v, ctx, tiles, s) : launch<T_BF16, 128>(a, k, v, ctx, tiles, s);
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

cudaError_t take_status_tc(unsigned* bits, cudaStream_t s) { return take_status(bits, s); }

}  // namespace cache
}  // namespace lfm
