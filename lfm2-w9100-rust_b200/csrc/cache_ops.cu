// C ABI of the attention over session caches (include/lfm_cuda.h,
// lfm_attention_* and lfm_cache_evict): the checks of every argument that the
// host can see. The kernels check what only the device holds (slots, lengths).
#include <math.h>
#include <stdio.h>

#include <mutex>

#include "../../include/lfm_cuda.h"
#include "cache_attn.h"
#include "kernels.h"

namespace {
using namespace lfm::cache;

constexpr uint32_t MAX_CTX = 1u << 24, MAX_N = 1u << 20, MAX_BATCH = 65535, MAX_KV_HEADS = 1024;

lfm_status bad(const char* who, const char* what) {
  char m[256];
  snprintf(m, sizeof m, "%s: %s", who, what);
  lfm::ops_set_error(m);
  return LFM_ERR_ARG;
}

lfm_status done(const char* who, cudaError_t e) {
  if (e == cudaSuccess) return LFM_OK;
  cudaGetLastError();  // reported here, not by the caller's next check
  char m[256];
  snprintf(m, sizeof m, "%s: CUDA: %s", who, cudaGetErrorString(e));
  lfm::ops_set_error(m);
  return LFM_ERR_CUDA;
}

// Whether the current device's kernels may read p: its own memory, or managed memory.
bool here(const void* p) {
  cudaPointerAttributes at;
  int device = -1;
  if (cudaGetDevice(&device) != cudaSuccess || cudaPointerGetAttributes(&at, p) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == device);
}
const char* const ELSEWHERE = "the arrays must be memory of the current device";

bool aligned(const void* p) { return (uintptr_t)p % 16 == 0; }
// the 4-byte arrays (null where they may be left out)
bool aligned4(const void* p) { return (uintptr_t)p % 4 == 0; }

// null: the shape is good
const char* shape_error(const lfm_attn_shape* s, bool caches_only) {
  if (!s) return "shape is null";
  if (s->dtype > LFM_ATTN_BF16) return "dtype must be LFM_ATTN_F32, LFM_ATTN_F16 or LFM_ATTN_BF16";
  if (s->kv_heads == 0 || s->kv_heads > MAX_KV_HEADS) return "1 <= kv_heads <= 1024";
  if (s->head_dim != 64 && s->head_dim != 128) return "head_dim must be 64 or 128";
  if (s->ctx == 0 || s->ctx > MAX_CTX) return "1 <= ctx <= 2^24";
  if (caches_only) return nullptr;
  if (s->heads == 0 || s->heads % s->kv_heads || s->heads / s->kv_heads > LFM_ATTN_MAX_GROUP)
    return "heads must be kv_heads times 1 to 8";
  // the kernels take powers of two: scale * log2 e is finite too, and keeps fp32's bits
  if (!(s->scale == 0.f || (s->scale >= 0x1p-126f && s->scale <= 0x1p127f)))
    return "scale must be 2^-126 to 2^127 (0: 1/sqrt(head_dim))";
  return nullptr;
}

float scale_of(const lfm_attn_shape* s) { return s->scale > 0.f ? s->scale : 1.0f / sqrtf((float)s->head_dim); }

// null: rows of heads x head_dim values at `stride` are good
const char* rows_error(const lfm_attn_shape* s, const void* p, uint64_t stride) {
  const uint32_t per16 = s->dtype == LFM_ATTN_F32 ? 4 : 8;
  if (!p || !aligned(p)) return "q and out must be 16-byte aligned device pointers";
  if (stride < (uint64_t)s->heads * s->head_dim || stride % per16 || stride > (1ull << 40))
    return "q_stride and out_stride must be >= heads * head_dim and a multiple of 16 bytes";
  return nullptr;
}

const char* slots_error(const lfm_attn_shape* s, uint64_t slot_stride, uint32_t n_slots, const void* slots,
                        const void* lens, uint32_t batch, uint32_t max_len) {
  if (!lens) return "lens is null";
  if (!aligned4(lens) || !aligned4(slots)) return "lens and slots must be 4-byte aligned";
  if (batch == 0 || batch > MAX_BATCH) return "1 <= batch <= 65535";
  if (n_slots == 0 || n_slots > 0x7fffffffu) return "n_slots must be 1 to 2^31 - 1";
  if (!slots && batch > n_slots) return "without slots, batch must be <= n_slots";
  if (slot_stride % 8 || slot_stride > (1ull << 40)) return "slot_stride must be a multiple of 8 elements";
  if (n_slots > 1 && slot_stride < (uint64_t)s->kv_heads * s->ctx * s->head_dim)
    return "slot_stride must be >= kv_heads * ctx * head_dim";
  if (max_len > s->ctx) return "max_len must be <= ctx";
  return nullptr;
}

lfm_status prompt_args(const char* who, const lfm_attn_shape* s, const void* q, uint64_t q_stride, const void* k,
                       uint32_t start, uint32_t n, uint32_t window, uint32_t sinks, Prompt* a) {
  if (const char* e = shape_error(s, false)) return bad(who, e);
  if (const char* e = rows_error(s, q, q_stride)) return bad(who, e);
  if (!k || !aligned(k)) return bad(who, "the caches must be 16-byte aligned device pointers");
  if (n == 0 || n > MAX_N || (uint64_t)start + n > s->ctx) return bad(who, "1 <= n <= 2^20 and start + n <= ctx");
  *a = {};
  a->type = (int)s->dtype, a->heads = (int)s->heads, a->kv_heads = (int)s->kv_heads, a->d = (int)s->head_dim;
  a->ctx = (int)s->ctx, a->scale = scale_of(s);
  a->q = q, a->q_stride = q_stride, a->k = k;
  a->start = (int)start, a->n = (int)n;
  a->window = window >= start + n ? 0 : (int)window;  // one that spans every position hides nothing
  a->sinks = (int)(sinks < s->ctx ? sinks : s->ctx);
  return LFM_OK;
}

lfm_status decode_args(const char* who, const lfm_attn_shape* s, const void* q, uint64_t q_stride, const void* k,
                       const void* v, uint64_t slot_stride, uint32_t n_slots, const int32_t* slots,
                       const int32_t* lens, uint32_t batch, uint32_t max_len, void* out, uint64_t out_stride,
                       Decode* a) {
  if (const char* e = shape_error(s, false)) return bad(who, e);
  if (const char* e = rows_error(s, q, q_stride)) return bad(who, e);
  if (const char* e = rows_error(s, out, out_stride)) return bad(who, e);
  if (!k || !v || !aligned(k) || !aligned(v)) return bad(who, "the caches must be 16-byte aligned device pointers");
  if (const char* e = slots_error(s, slot_stride, n_slots, slots, lens, batch, max_len)) return bad(who, e);
  *a = {};
  a->type = (int)s->dtype, a->heads = (int)s->heads, a->kv_heads = (int)s->kv_heads, a->d = (int)s->head_dim;
  a->ctx = (int)s->ctx, a->scale = scale_of(s);
  a->q = q, a->q_stride = q_stride, a->k = k, a->v = v;
  a->slot_stride = slot_stride, a->n_slots = (int)n_slots, a->slots = slots, a->lens = lens;
  a->batch = (int)batch, a->max_len = (int)max_len;
  a->out = out, a->out_stride = out_stride;
  return LFM_OK;
}

bool decode_here(const Decode& a) {
  return here(a.q) && here(a.k) && here(a.v) && here(a.lens) && here(a.out) && (!a.slots || here(a.slots)) &&
         (!a.acc || here(a.acc));
}

// What has been reported is taken and cleared in one step of each word: kernels of other streams report meanwhile.
__device__ unsigned g_taken;
__global__ void k_take(unsigned* a, unsigned* b, unsigned* c, unsigned* d) {
  g_taken = atomicExch(a, 0u) | atomicExch(b, 0u) | atomicExch(c, 0u) | atomicExch(d, 0u);
}

// `count` blocks of n bytes, `stride` bytes from one to the next; in 128 bits, since n_slots and slot_stride may be
// anything that an array could not have.
using Wide = __int128;
struct Blocks {
  const void* p;
  Wide n, stride, count;
};
Wide floor_div(Wide a, Wide b) { return a / b - (a % b < 0); }
// Blocks of one stride (or one block alone): some i - j = k of theirs meet where -b.n < b.p - a.p - k stride < a.n.
bool overlap(const Blocks& a, const Blocks& b) {
  if (!a.p || !b.p) return false;
  const Wide stride = a.count > 1 ? a.stride : b.count > 1 ? b.stride : 1;
  const Wide d = (Wide)(uintptr_t)b.p - (Wide)(uintptr_t)a.p;
  const Wide lo = floor_div(d - a.n, stride) + 1, hi = -floor_div(-(d + b.n), stride) - 1;
  return (lo > 1 - b.count ? lo : 1 - b.count) <= (hi < a.count - 1 ? hi : a.count - 1);
}
}  // namespace

extern "C" {

lfm_status lfm_attention_window(const lfm_attn_shape* shape, const void* q, uint64_t q_stride, const void* k_cache,
                                const void* v_cache, uint32_t start, uint32_t n, uint32_t window, uint32_t sinks,
                                void* out, uint64_t out_stride, float* lse, void* stream) {
  const char* who = "lfm_attention_window";
  Prompt a;
  if (lfm_status st = prompt_args(who, shape, q, q_stride, k_cache, start, n, window, sinks, &a)) return st;
  if (const char* e = rows_error(shape, out, out_stride)) return bad(who, e);
  if (!v_cache || !aligned(v_cache)) return bad(who, "the caches must be 16-byte aligned device pointers");
  if (!aligned4(lse)) return bad(who, "lse must be 4-byte aligned");
  if (!here(q) || !here(k_cache) || !here(v_cache) || !here(out) || (lse && !here(lse))) return bad(who, ELSEWHERE);
  a.v = v_cache, a.out = out, a.out_stride = out_stride, a.lse = lse;
  return done(who, lfm::cache::window(a, (cudaStream_t)stream));
}

lfm_status lfm_attention_weights(const lfm_attn_shape* shape, const void* q, uint64_t q_stride, const void* k_cache,
                                 uint32_t start, uint32_t n, uint32_t window, uint32_t sinks, const float* lse,
                                 float* acc, void* stream) {
  const char* who = "lfm_attention_weights";
  Prompt a;
  if (lfm_status st = prompt_args(who, shape, q, q_stride, k_cache, start, n, window, sinks, &a)) return st;
  if (!lse || !acc) return bad(who, "lse and acc must be device pointers");
  if (!aligned4(lse) || !aligned4(acc)) return bad(who, "lse and acc must be 4-byte aligned");
  if (!here(q) || !here(k_cache) || !here(lse) || !here(acc)) return bad(who, ELSEWHERE);
  a.lse = const_cast<float*>(lse), a.acc = acc;
  return done(who, lfm::cache::weights(a, (cudaStream_t)stream));
}

lfm_status lfm_attention_decode(const lfm_attn_shape* shape, const void* q, uint64_t q_stride, const void* k_cache,
                                const void* v_cache, uint64_t slot_stride, uint32_t n_slots, const int32_t* slots,
                                const int32_t* lens, uint32_t batch, uint32_t max_len, uint32_t window,
                                uint32_t sinks, float* acc, void* out, uint64_t out_stride, void* stream) {
  const char* who = "lfm_attention_decode";
  Decode a;
  if (lfm_status st = decode_args(who, shape, q, q_stride, k_cache, v_cache, slot_stride, n_slots, slots, lens, batch,
                                  max_len, out, out_stride, &a))
    return st;
  a.window = window >= max_len ? 0 : (int)window;
  a.sinks = (int)(sinks < shape->ctx ? sinks : shape->ctx);
  if (!aligned4(acc)) return bad(who, "acc must be 4-byte aligned");
  a.acc = acc;
  if (!decode_here(a)) return bad(who, ELSEWHERE);
  return done(who, lfm::cache::decode(a, (cudaStream_t)stream));
}

size_t lfm_attention_shared_workspace(const lfm_attn_shape* shape, uint32_t batch, uint32_t prefix_len) {
  if (shape_error(shape, false) || batch == 0 || batch > MAX_BATCH || prefix_len > MAX_CTX) return 0;
  Decode a = {};
  a.heads = (int)shape->heads, a.kv_heads = (int)shape->kv_heads, a.d = (int)shape->head_dim;
  a.batch = (int)batch, a.prefix_len = (int)prefix_len;
  return lfm::cache::shared_workspace(a);
}

lfm_status lfm_attention_shared(const lfm_attn_shape* shape, const void* q, uint64_t q_stride, const void* prefix_k,
                                const void* prefix_v, uint32_t prefix_ctx, uint32_t prefix_len, const void* k_cache,
                                const void* v_cache, uint64_t slot_stride, uint32_t n_slots, const int32_t* slots,
                                const int32_t* lens, uint32_t batch, uint32_t max_len, void* out,
                                uint64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "lfm_attention_shared";
  Decode a;
  if (lfm_status st = decode_args(who, shape, q, q_stride, k_cache, v_cache, slot_stride, n_slots, slots, lens, batch,
                                  max_len, out, out_stride, &a))
    return st;
  if (prefix_len > prefix_ctx || prefix_ctx > MAX_CTX) return bad(who, "prefix_len <= prefix_ctx <= 2^24");
  if (prefix_len && (!prefix_k || !prefix_v || !aligned(prefix_k) || !aligned(prefix_v)))
    return bad(who, "the prefix must be 16-byte aligned device pointers");
  a.pk = prefix_k, a.pv = prefix_v, a.prefix_ctx = (int)prefix_ctx, a.prefix_len = (int)prefix_len;
  if (!workspace || !aligned(workspace) || workspace_bytes < lfm::cache::shared_workspace(a))
    return bad(who, "workspace must be 16-byte aligned, of lfm_attention_shared_workspace bytes");
  if (!decode_here(a) || !here(workspace) || (prefix_len && (!here(prefix_k) || !here(prefix_v))))
    return bad(who, ELSEWHERE);
  a.work = workspace;
  return done(who, lfm::cache::shared(a, (cudaStream_t)stream));
}

lfm_status lfm_cache_evict(const lfm_attn_shape* shape, const void* k_src, const void* v_src, const float* acc_src,
                           const int32_t* pos_src, void* k_dst, void* v_dst, float* acc_dst, int32_t* pos_dst,
                           uint64_t slot_stride, uint32_t n_slots, const int32_t* slots, const int32_t* lens,
                           int32_t* lens_out, uint32_t batch, uint32_t max_len, uint32_t budget, uint32_t keep_first,
                           uint32_t keep_last, void* stream) {
  const char* who = "lfm_cache_evict";
  if (const char* e = shape_error(shape, true)) return bad(who, e);
  if (!k_src || !v_src || !k_dst || !v_dst || !aligned(k_src) || !aligned(v_src) || !aligned(k_dst) || !aligned(v_dst))
    return bad(who, "the caches must be 16-byte aligned device pointers");
  if (!acc_src || !acc_dst || !lens_out) return bad(who, "acc_src, acc_dst and lens_out must be device pointers");
  if (!aligned4(acc_src) || !aligned4(acc_dst) || !aligned4(pos_src) || !aligned4(pos_dst) || !aligned4(lens_out))
    return bad(who, "acc, pos and lens_out must be 4-byte aligned");
  if (!pos_src != !pos_dst) return bad(who, "pos_src and pos_dst are both given or both null");
  if (const char* e = slots_error(shape, slot_stride, n_slots, slots, lens, batch, max_len)) return bad(who, e);
  if (budget == 0 || (uint64_t)keep_first + keep_last > budget)
    return bad(who, "budget >= 1 and keep_first + keep_last <= budget");
  const Wide rows = (Wide)shape->kv_heads * shape->ctx, step = 2 * (Wide)slot_stride;
  auto slots_of = [&](const void* p) { return Blocks{p, 2 * rows * shape->head_dim, step, n_slots}; };
  auto records = [&](const void* p) { return Blocks{p, 4 * rows * n_slots, 0, 1}; };
  auto list = [&](const void* p) { return Blocks{p, 4 * (Wide)batch, 0, 1}; };
  const Blocks src[4] = {slots_of(k_src), slots_of(v_src), records(acc_src), records(pos_src)};
  const Blocks dst[5] = {slots_of(k_dst), slots_of(v_dst), records(acc_dst), records(pos_dst), list(lens_out)};
  const Blocks in[2] = {list(lens), list(slots)};
  const bool in_place = k_src == k_dst;
  for (int i = 0; i < 5; i++) {
    for (int j = 0; j < 4; j++) {
      if (i == j && in_place && src[i].p == dst[i].p) continue;
      if (overlap(dst[i], src[j]))
        return bad(who, "the destinations are the sources, all of them, or overlap no source");
      if (i == j && in_place && src[i].p)
        return bad(who, "the destinations are the sources, all of them, or overlap no source");
    }
    for (int j = 0; j < 2; j++)
      if (overlap(dst[i], in[j])) return bad(who, "the destinations overlap neither lens nor slots");
    for (int j = 0; j < i; j++)
      if (overlap(dst[i], dst[j])) return bad(who, "the destinations overlap one another");
  }
  for (const Blocks& r : src)
    if (r.p && !here(r.p)) return bad(who, ELSEWHERE);
  for (const Blocks& r : dst)
    if (r.p && !here(r.p)) return bad(who, ELSEWHERE);
  for (const Blocks& r : in)
    if (r.p && !here(r.p)) return bad(who, ELSEWHERE);
  Evict a = {};
  a.kv_heads = (int)shape->kv_heads, a.d = (int)shape->head_dim, a.ctx = (int)shape->ctx;
  a.k = k_src, a.v = v_src, a.acc = acc_src, a.pos = pos_src;
  a.k_out = k_dst, a.v_out = v_dst, a.acc_out = acc_dst, a.pos_out = pos_dst;
  a.slot_stride = slot_stride, a.n_slots = (int)n_slots, a.slots = slots, a.lens = lens, a.lens_out = lens_out;
  a.batch = (int)batch, a.max_len = (int)max_len;
  // a session of max_len <= ctx keeps all it has under a larger budget: the numbers below stay ints
  a.budget = (int)(budget < MAX_CTX ? budget : MAX_CTX);
  a.keep_first = (int)(keep_first < MAX_CTX ? keep_first : MAX_CTX);
  a.keep_last = (int)(keep_last < MAX_CTX ? keep_last : MAX_CTX);
  return done(who, lfm::cache::evict(a, (cudaStream_t)stream));
}

lfm_status lfm_attention_status(uint32_t* status, void* stream) {
  const char* who = "lfm_attention_status";
  if (!status) return bad(who, "status is null");
  const cudaStream_t s = (cudaStream_t)stream;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaError_t e = cudaStreamIsCapturing(s, &capture)) return done(who, e);
  if (capture != cudaStreamCaptureStatusNone) return bad(who, "waits for the stream, which is being captured");
  unsigned *words[4] = {}, *taken = nullptr, bits = 0;
  cudaError_t e = lfm::cache::status_word_tc(&words[0]);
  if (e == cudaSuccess) e = lfm::cache::status_word_weights(&words[1]);
  if (e == cudaSuccess) e = lfm::cache::status_word_decode(&words[2]);
  if (e == cudaSuccess) e = lfm::cache::status_word_evict(&words[3]);
  if (e == cudaSuccess) e = cudaGetSymbolAddress((void**)&taken, g_taken);
  if (e != cudaSuccess) return done(who, e);
  // one call at a time, to the end of its wait: g_taken is the device's
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  k_take<<<1, 1, 0, s>>>(words[0], words[1], words[2], words[3]);
  e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyAsync(&bits, taken, sizeof bits, cudaMemcpyDeviceToHost, s);
  const cudaError_t waited = cudaStreamSynchronize(s);
  if (e == cudaSuccess) e = waited;
  if (e == cudaSuccess) *status = bits;
  return done(who, e);
}

}  // extern "C"
