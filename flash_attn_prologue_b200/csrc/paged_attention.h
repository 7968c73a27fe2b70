// Arguments of the paged attention kernels (paged_decode.cu, paged_prefill.cu).
#pragma once

#include "paged_host.h"

namespace flash_prologue {

// Probabilities of FP16 caches are 2^7 times as large while they are multiplied
// with V (and summed): those down to 2^-21 of the largest then keep all of their
// bits, where unscaled ones below 2^-14 would lose them. The largest may be 2^8
// (paged_prefill.cu), which is 2^15 so, inside the type. BF16 has FP32's range.
template <typename T>
constexpr float kProbabilityShift = std::is_same<T, __half>::value ? 7.f : 0.f;

struct AttentionArgs {
  const void* q;
  void* out;
  float* lse;                // [T, Hq] natural logarithm, or null
  int64_t q_n, q_h, out_n, out_h;
  const void* k;
  const void* v;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;  // elements
  PagedTarget pages;
  int tokens;
  int heads, kv_heads, group;  // group = heads / kv_heads
  float scale_log2;          // softmax_scale * log2(e)
  int window;                // keys a row sees at most; 0: all
  void* workspace;
  int whole;                 // single-token kernel: items are not split (set at launch)
  int max_keys;              // pages.max_pages * page_size
};

// Lets the next kernel of the stream be placed (see launch_following), and
// waits until the one before has ended and its writes can be read.
__device__ __forceinline__ void start_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// One request as the kernels see it: its new tokens and the keys it may reach.
struct Request {
  int first;   // packed index of its first new token
  int news;    // new tokens
  int total;   // tokens in the cache
};

// Requests that a kernel goes through: split by cu_seqlens, two more than there
// are, for the rows behind the last request and before the first.
__device__ __forceinline__ int requests_of(const PagedTarget& p) { return p.batch + (p.cu_seqlens ? 2 : 0); }

// Sizes are clamped to what the tensors hold, so wrong ones cannot lead outside
// them. r == batch is the padding behind the last request, r == batch + 1 that
// before the first: tokens without keys.
// The host keeps tokens x heads below 2^31 and max_keys below 2^30.
__device__ __forceinline__ Request request_at(const PagedTarget& p, int tokens, int max_keys, int r, bool* too_long) {
  Request q;
  const int total = r < p.batch ? __ldg(p.seq_lens + r) : 0;
  if (p.cu_seqlens) {
    const int a = r <= p.batch ? __ldg(p.cu_seqlens + r) : 0;
    const int b = r < p.batch ? __ldg(p.cu_seqlens + r + 1) : r == p.batch ? tokens : __ldg(p.cu_seqlens);
    q.first = min(max(a, 0), tokens);
    q.news = min(max(b, q.first), tokens) - q.first;
  } else {
    q.first = r;
    q.news = r < p.batch ? 1 : 0;
  }
  *too_long = total > max_keys;
  q.total = min(max(total, 0), max_keys);
  return q;
}

// Workspace bytes that cover every call of the kernel on a device of `sms` SMs.
size_t paged_decode_workspace(int D, int sms);
size_t paged_prefill_workspace(int D, int sms);
struct PrefillPlan {
  int tile_rows;     // 128 or (over a cache of 4 bits, D = 128) 256
  int tile_tokens;   // whole tokens of a tile
  int splits;        // shares of the keys of the items behind whole_items
  int64_t whole_items;
  int64_t tiles;     // tiles there can be, all requests
};
PrefillPlan plan_paged_prefill(int64_t tokens, int64_t batch, bool ragged, int64_t kv_heads, int64_t group, int D,
                               int64_t max_keys, int64_t window, int sms, bool int4);
// Workspace bytes that the plan's shares take: never more than paged_prefill_workspace, which a test and each call check.
size_t paged_prefill_needs(const PrefillPlan& plan, int64_t kv_heads, int D);
// False where the cache's layout has no tensor map (the other kernel reads it). wait_cycles: 0, or
// (self-test, BF16) the limit of the kernel's waits, but for those for copies and products under way.
// scales: null, or the cache is one of 4 bits (a.k, a.v: codes, strides in bytes).
bool launch_paged_prefill(const AttentionArgs& a, const PrefillPlan& plan, const flash_prologue_scales* scales, int dtype,
                          int D, int64_t page_size, long long wait_cycles, cudaStream_t stream, cudaError_t* err);
cudaError_t launch_paged_decode(const AttentionArgs& a, int dtype, int D, cudaStream_t stream);
// The same over a cache of 4 bits (a.k, a.v: codes, strides in bytes).
size_t paged_int4_decode_workspace(int D, int sms);
cudaError_t launch_paged_int4_decode(const AttentionArgs& a, const flash_prologue_scales& s, int dtype, int D,
                                     cudaStream_t stream);

}  // namespace flash_prologue
