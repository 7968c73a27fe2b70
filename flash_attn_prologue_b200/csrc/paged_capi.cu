// C ABI of paged attention: argument checks and the choice of kernel.
// Declarations: include/flash_prologue.h.
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

int head_checks(int64_t Hq, int64_t Hk, int64_t D) {
  if (Hq < 0 || Hk <= 0 || Hq % Hk != 0) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  return Hq > kMaxGqaHeads || (D != 64 && D != 128) ? FLASH_PROLOGUE_ERR_UNSUPPORTED : FLASH_PROLOGUE_OK;
}

}  // namespace

extern "C" {

int flash_prologue_paged_attention_workspace_size(int64_t Hq, int64_t Hk, int64_t D, size_t* bytes) {
  if (!bytes) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  const int st = head_checks(Hq, Hk, D);
  if (st != FLASH_PROLOGUE_OK) return st;
  const int sms = device_sms();
  if (sms <= 0) return FLASH_PROLOGUE_ERR_CUDA;
  *bytes = paged_decode_workspace((int)D, sms);
  return FLASH_PROLOGUE_OK;
}

int flash_prologue_paged_attention(const flash_prologue_attention_args* a, void* stream) {
  if (!a || a->tokens < 0 || a->window < 0 || !isfinite(a->softmax_scale)) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (a->dtype != FLASH_PROLOGUE_BF16 && a->dtype != FLASH_PROLOGUE_FP16) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  int st = head_checks(a->Hq, a->Hk, a->D);
  if (st != FLASH_PROLOGUE_OK) return st;
  if (a->tokens >= (int64_t(1) << 31) / 512) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  const flash_prologue_cache& c = a->cache;
  st = check_cache(c, a->tokens, a->dtype);
  if (st != FLASH_PROLOGUE_OK || a->tokens == 0 || a->Hq == 0) return st;
  if (!a->q.data || !a->out.data) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(a->q.data) | reinterpret_cast<uintptr_t>(a->out.data)) & 15 ||
      ((a->q.n | a->q.h | a->out.n | a->out.h) & 7))
    return FLASH_PROLOGUE_ERR_ALIGNMENT;
  if ((a->tokens > 1 && a->out.n == 0) || (a->Hq > 1 && a->out.h == 0)) return FLASH_PROLOGUE_ERR_EXPANDED;
  const int sms = device_sms();
  if (sms <= 0) return FLASH_PROLOGUE_ERR_CUDA;
  if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 15) ||
      a->workspace_bytes < (int64_t)paged_decode_workspace((int)a->D, sms))
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
  g.tokens = a->tokens;
  g.heads = (int)a->Hq;
  g.kv_heads = (int)a->Hk;
  g.group = g.heads / g.kv_heads;
  g.scale_log2 = (float)(a->softmax_scale * 1.4426950408889634);
  g.window = a->window;
  g.workspace = a->workspace;
  g.max_keys = c.max_pages * c.page_size;
  return launch_paged_decode(g, (int)a->dtype, (int)a->D, static_cast<cudaStream_t>(stream)) == cudaSuccess
             ? FLASH_PROLOGUE_OK
             : FLASH_PROLOGUE_ERR_CUDA;
}

}  // extern "C"
