// Attention over session caches (lfm_attention_*, lfm_cache_evict): launch
// arguments shared by the kernels and the C entry points that check them.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace lfm {
namespace cache {

// What a kernel reports in the device's status word (LFM_ATTN_BAD_*).
constexpr unsigned BAD_WAIT = 1u, BAD_SLOT = 2u, BAD_LEN = 4u;

enum Type { T_F32 = 0, T_F16 = 1, T_BF16 = 2 };

// Strides in elements.
struct Prompt {
  int type, heads, kv_heads, d, ctx;
  float scale;
  const void* q;
  size_t q_stride;
  const void *k, *v;  // one slot
  int start, n, window, sinks;
  void* out;
  size_t out_stride;
  float* lse;        // written by the attention, read by the weights
  float* acc;        // weights only
};

struct Decode {
  int type, heads, kv_heads, d, ctx;
  float scale;
  const void* q;
  size_t q_stride;
  const void *k, *v;
  size_t slot_stride;
  int n_slots;
  const int *slots, *lens;
  int batch, max_len, window, sinks;
  float* acc;
  void* out;
  size_t out_stride;
  // shared prefix (prefix_len 0: none)
  const void *pk, *pv;
  int prefix_ctx, prefix_len;
  void* work;
};

struct Evict {
  int kv_heads, d, ctx;
  const void *k, *v;
  const float* acc;
  const int* pos;
  void *k_out, *v_out;
  float* acc_out;
  int* pos_out;
  size_t slot_stride;
  int n_slots;
  const int *slots, *lens;
  int* lens_out;
  int batch, max_len, budget, keep_first, keep_last;
};

cudaError_t window(const Prompt& a, cudaStream_t s);
cudaError_t weights(const Prompt& a, cudaStream_t s);
cudaError_t decode(const Decode& a, cudaStream_t s);
// decode joined with the prefix's part: o [kv head][session * g + head][d] not divided by l, ml (m in log2 units, l)
cudaError_t decode_joined(const Decode& a, const float* o, const float2* ml, cudaStream_t s);
size_t shared_workspace(const Decode& a);
cudaError_t shared(const Decode& a, cudaStream_t s);
cudaError_t evict(const Evict& a, cudaStream_t s);
// Where the kernels of each file report on the current device.
cudaError_t status_word_tc(unsigned** at);
cudaError_t status_word_weights(unsigned** at);
cudaError_t status_word_decode(unsigned** at);
cudaError_t status_word_evict(unsigned** at);

}  // namespace cache
}  // namespace lfm
