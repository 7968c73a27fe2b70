// C ABI of paged attention: argument checks and the choice of kernel.
// Declarations: include/flash_prologue.h.
#include <float.h>
#include <math.h>

#include "paged_attention.h"

// Callers pack the struct field by field: every field is 8 bytes wide.
static_assert(sizeof(flash_prologue_attention_args) == 272, "argument struct layout");

using namespace flash_prologue;

namespace {

int device_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return sms;
}

// The factor of the scores' base-2 exponentials.
double scale_log2_of(const flash_prologue_attention_args* a) { return a->softmax_scale * 1.4426950408889634; }

int size_checks(const flash_prologue_attention_args* a, bool int4) {
  if (!a || a->tokens < 0 || a->window < 0 || !(fabs(scale_log2_of(a)) <= FLT_MAX) || a->Hq < 0 || a->Hk <= 0 ||
      a->Hq % a->Hk)
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if ((a->dtype != FLASH_PROLOGUE_BF16 && a->dtype != FLASH_PROLOGUE_FP16) || a->Hq > kMaxGqaHeads ||
      (a->D != 64 && a->D != 128) || a->tokens >= (int64_t(1) << 31) / kMaxGqaHeads)
    return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  return check_cache(a->cache, a->tokens, int4 ? 1 : 2);
}

// Tiles of 128 rows on the tensor cores where the requests have more rows a key
// head than the other kernel's 16-row tile on average. The tiled kernel takes
// the maximum of the unscaled scores and multiplies masked ones (-infinity) by the
// scale, so the FP32 scale has to be positive (and normal), and a tile holds at
// least one whole token.
//
// Over a cache of 4 bits the other kernel takes tiles of 8 and 16 rows, and the rule stays. 12 rows a key head
// (20 rows, tiled), 8 key heads x 128: 64 requests of 8,192 keys 250 (465) us, 64 of 2,048 keys 88 (128), 16 of
// 4,096 50 (64), 32 of 1,024 34 (38); where there is little to read tiles would win a little, 4 of 4,096 32 (27).
bool use_prefill(const flash_prologue_attention_args* a, float scale_log2) {
  const int64_t group = a->Hq / a->Hk;
  return a->tokens * group > 16 * a->cache.batch && group <= 128 && scale_log2 >= FLT_MIN;
}

size_t int4_workspace_of(int64_t D, int sms) {
  const size_t decode = paged_int4_decode_workspace((int)D, sms), prefill = paged_prefill_workspace((int)D, sms);
  return prefill > decode ? prefill : decode;
}

size_t workspace_of(int64_t D, int sms) {
  const size_t decode = paged_decode_workspace((int)D, sms), prefill = paged_prefill_workspace((int)D, sms);
  return prefill > decode ? prefill : decode;
}

// wait_cycles: 0, or the limit of the tiled kernel's waits (self-test), and no other kernel is taken.
// scales: null, or the cache is one of 4 bits.
int attention(const flash_prologue_attention_args* a, const flash_prologue_scales* scales, int64_t wait_cycles,
              void* stream) {
  int st = size_checks(a, scales != nullptr);
  if (st != FLASH_PROLOGUE_OK || a->tokens == 0 || a->Hq == 0) return st;
  if (scales) {
    if ((st = check_scales(*scales, a->cache, a->D)) != FLASH_PROLOGUE_OK) return st;
    // The kernels multiply pages and slots by strides of 31 bits. (A single page has none.)
    const bool pages = a->cache.num_pages > 1;
    for (int64_t s : {a->cache.k_slot, a->cache.v_slot, 2 * scales->k_slot, 2 * scales->v_slot,
                      pages ? a->cache.k_page : 0, pages ? a->cache.v_page : 0, pages ? 2 * scales->k_page : 0,
                      pages ? 2 * scales->v_page : 0})
      if (s > INT32_MAX || s < INT32_MIN) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  }
  const flash_prologue_cache& c = a->cache;
  if (!a->q.data || !a->out.data) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(a->q.data) | reinterpret_cast<uintptr_t>(a->out.data)) & 15 ||
      ((a->q.n | a->q.h | a->out.n | a->out.h) & 7))
    return FLASH_PROLOGUE_ERR_ALIGNMENT;
  if ((a->tokens > 1 && a->out.n == 0) || (a->Hq > 1 && a->out.h == 0)) return FLASH_PROLOGUE_ERR_EXPANDED;
  const int sms = device_sms();
  if (sms <= 0) return FLASH_PROLOGUE_ERR_CUDA;
  if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 15) ||
      a->workspace_bytes < (int64_t)(scales ? int4_workspace_of(a->D, sms) : workspace_of(a->D, sms)))
    return FLASH_PROLOGUE_ERR_WORKSPACE;
  AttentionArgs g{};
  g.q = a->q.data;
  g.q_n = a->q.n;
  g.q_h = a->q.h;
  g.out = a->out.data;
  g.out_n = a->out.n;
  g.out_h = a->out.h;
  g.lse = a->lse;
  g.k = c.k;
  g.v = c.v;
  g.k_page = c.k_page;
  g.k_slot = c.k_slot;
  g.k_head = c.k_head;
  g.v_page = c.v_page;
  g.v_slot = c.v_slot;
  g.v_head = c.v_head;
  g.pages = paged_target(c);
  g.tokens = (int)a->tokens;
  g.heads = (int)a->Hq;
  g.kv_heads = (int)a->Hk;
  g.group = g.heads / g.kv_heads;
  g.scale_log2 = (float)scale_log2_of(a);
  g.workspace = a->workspace;
  g.max_keys = (int)(c.max_pages * c.page_size);
  g.window = a->window < g.max_keys ? (int)a->window : 0;  // as long as any request: all keys
  if (use_prefill(a, g.scale_log2)) {
    const PrefillPlan plan = plan_paged_prefill(a->tokens, c.batch, c.cu_seqlens != nullptr, a->Hk, g.group, (int)a->D,
                                                g.max_keys, g.window, sms, scales != nullptr);
    if (paged_prefill_needs(plan, a->Hk, (int)a->D) > paged_prefill_workspace((int)a->D, sms))
      return FLASH_PROLOGUE_ERR_WORKSPACE;
    cudaError_t err = cudaSuccess;
    if (launch_paged_prefill(g, plan, scales, (int)a->dtype, (int)a->D, c.page_size,
                             wait_cycles, static_cast<cudaStream_t>(stream), &err))
      return err == cudaSuccess ? FLASH_PROLOGUE_OK : FLASH_PROLOGUE_ERR_CUDA;
  }
  if (wait_cycles) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  if (scales)
    return launch_paged_int4_decode(g, *scales, (int)a->dtype, (int)a->D, static_cast<cudaStream_t>(stream)) == cudaSuccess
               ? FLASH_PROLOGUE_OK
               : FLASH_PROLOGUE_ERR_CUDA;
  return launch_paged_decode(g, (int)a->dtype, (int)a->D, static_cast<cudaStream_t>(stream)) == cudaSuccess
             ? FLASH_PROLOGUE_OK
             : FLASH_PROLOGUE_ERR_CUDA;
}

}  // namespace

extern "C" {

int flash_prologue_paged_attention_workspace_size(int64_t D, size_t* bytes) {
  if (!bytes) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  if (D != 64 && D != 128) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  const int sms = device_sms();
  if (sms <= 0) return FLASH_PROLOGUE_ERR_CUDA;
  *bytes = workspace_of(D, sms);
  return FLASH_PROLOGUE_OK;
}

int flash_prologue_paged_attention(const flash_prologue_attention_args* a, void* stream) {
  return attention(a, nullptr, 0, stream);
}

int flash_prologue_paged_attention_int4_workspace_size(int64_t D, size_t* bytes) {
  if (!bytes) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  if (D != 64 && D != 128) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  const int sms = device_sms();
  if (sms <= 0) return FLASH_PROLOGUE_ERR_CUDA;
  *bytes = int4_workspace_of(D, sms);
  return FLASH_PROLOGUE_OK;
}

int flash_prologue_paged_attention_int4(const flash_prologue_attention_args* a, const flash_prologue_scales* scales,
                                        void* stream) {
  return scales ? attention(a, scales, 0, stream) : FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
}

int flash_prologue_selftest_attention_plan(const flash_prologue_attention_args* a, int int4, int64_t sms, size_t* needed,
                                           size_t* available) {
  if (!a || !needed || !available || sms < 1 || sms > 4096) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  *needed = *available = 0;
  if (a->tokens < 1 || a->Hk < 1 || a->Hq < a->Hk || a->Hq % a->Hk || a->cache.batch < 1 || a->window < 0 ||
      (a->D != 64 && a->D != 128))
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  const int64_t max_keys = a->cache.max_pages * a->cache.page_size;
  *available = paged_prefill_workspace((int)a->D, (int)sms);
  if (use_prefill(a, (float)scale_log2_of(a)))
    *needed = paged_prefill_needs(
        plan_paged_prefill(a->tokens, a->cache.batch, a->cache.cu_seqlens != nullptr, a->Hk, a->Hq / a->Hk, (int)a->D,
                           max_keys, a->window < max_keys ? a->window : 0, (int)sms, int4 != 0),
        a->Hk, (int)a->D);
  return FLASH_PROLOGUE_OK;
}

static int attention_waits(const flash_prologue_attention_args* a, const flash_prologue_scales* scales, int64_t wait_cycles,
                           void* stream) {
  if (!a || wait_cycles < 1 || wait_cycles > (int64_t(1) << 33)) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (a->dtype != FLASH_PROLOGUE_BF16) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  return attention(a, scales, wait_cycles, stream);
}
int flash_prologue_selftest_attention_waits(const flash_prologue_attention_args* a, int64_t wait_cycles, void* stream) {
  return attention_waits(a, nullptr, wait_cycles, stream);
}
int flash_prologue_selftest_attention_int4_waits(const flash_prologue_attention_args* a, const flash_prologue_scales* scales,
                                                 int64_t wait_cycles, void* stream) {
  return scales ? attention_waits(a, scales, wait_cycles, stream) : FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
}

}  // extern "C"
