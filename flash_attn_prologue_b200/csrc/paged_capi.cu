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

int size_checks(const flash_prologue_attention_args* a) {
  if (!a || a->tokens < 0 || a->window < 0 || !(fabs(scale_log2_of(a)) <= FLT_MAX) || a->Hq < 0 || a->Hk <= 0 ||
      a->Hq % a->Hk)
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if ((a->dtype != FLASH_PROLOGUE_BF16 && a->dtype != FLASH_PROLOGUE_FP16) || a->Hq > kMaxGqaHeads ||
      (a->D != 64 && a->D != 128) || a->tokens >= (int64_t(1) << 31) / kMaxGqaHeads)
    return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  return check_cache(a->cache, a->tokens, a->dtype);
}

// Tiles of 128 rows on the tensor cores where the requests have more rows a key
// head than the other kernel's 16-row tile on average. The tiled kernel takes
// the maximum of the unscaled scores and multiplies masked ones (-infinity) by the
// scale, so the FP32 scale has to be positive (and normal), and a tile holds at
// least one whole token.
bool use_prefill(const flash_prologue_attention_args* a, float scale_log2) {
  const int64_t group = a->Hq / a->Hk;
  return a->tokens * group > 16 * a->cache.batch && group <= 128 && scale_log2 >= FLT_MIN;
}

size_t workspace_of(int64_t D, int sms) {
  const size_t decode = paged_decode_workspace((int)D, sms), prefill = paged_prefill_workspace((int)D, sms);
  return prefill > decode ? prefill : decode;
}

// wait_cycles: 0, or the limit of the tiled kernel's waits (self-test), and no other kernel is taken.
int attention(const flash_prologue_attention_args* a, int64_t wait_cycles, void* stream) {
  const int st = size_checks(a);
  if (st != FLASH_PROLOGUE_OK || a->tokens == 0 || a->Hq == 0) return st;
  const flash_prologue_cache& c = a->cache;
  if (!a->q.data || !a->out.data) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(a->q.data) | reinterpret_cast<uintptr_t>(a->out.data)) & 15 ||
      ((a->q.n | a->q.h | a->out.n | a->out.h) & 7))
    return FLASH_PROLOGUE_ERR_ALIGNMENT;
  if ((a->tokens > 1 && a->out.n == 0) || (a->Hq > 1 && a->out.h == 0)) return FLASH_PROLOGUE_ERR_EXPANDED;
  const int sms = device_sms();
  if (sms <= 0) return FLASH_PROLOGUE_ERR_CUDA;
  if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 15) ||
      a->workspace_bytes < (int64_t)workspace_of(a->D, sms))
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
                                                g.max_keys, g.window, sms);
    cudaError_t err = cudaSuccess;
    if (launch_paged_prefill(g, plan, (int)a->dtype, (int)a->D, c.page_size,
                             wait_cycles, static_cast<cudaStream_t>(stream), &err))
      return err == cudaSuccess ? FLASH_PROLOGUE_OK : FLASH_PROLOGUE_ERR_CUDA;
  }
  if (wait_cycles) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
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
  return attention(a, 0, stream);
}

int flash_prologue_selftest_attention_waits(const flash_prologue_attention_args* a, int64_t wait_cycles, void* stream) {
  if (!a || wait_cycles < 1 || wait_cycles > (int64_t(1) << 33)) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (a->dtype != FLASH_PROLOGUE_BF16) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  return attention(a, wait_cycles, stream);
}

}  // extern "C"
