// C ABI of the grouped-query prologue and of the paged cache append: argument
// checks and launch planning. Declarations: include/flash_prologue.h.
#include <math.h>

#include "../../include/flash_prologue.h"
#include "gqa_rows.cuh"
#include "paged_host.h"

// Callers pack these structs field by field: every field is 8 bytes wide.
static_assert(sizeof(flash_prologue_rows) == 32 && sizeof(flash_prologue_rotation) == 56 &&
                  sizeof(flash_prologue_cache) == 128 && sizeof(flash_prologue_gqa_args) == 464 &&
                  sizeof(flash_prologue_append_args) == 376 && sizeof(flash_prologue_axes) == 80 &&
                  sizeof(flash_prologue_scales) == 64,
              "argument struct layout");

namespace flash_prologue {
namespace {

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

size_t elem_size(int64_t dtype) { return dtype == FLASH_PROLOGUE_FP32 ? 4 : 2; }

bool supported(int64_t D, int64_t dtype) {
  return (D == 32 || D == 64 || D == 128 || D == 256) && dtype >= 0 && dtype <= 2;
}

// Every 16-byte chunk of every row is aligned.
bool rows_vec(const flash_prologue_rows& r, size_t es) {
  return aligned(r.data, 16) && ((r.b | r.h | r.n) * (int64_t)es & 15) == 0;
}

bool rotation_vec(const flash_prologue_rotation& r) {
  return aligned(r.sin, 16) && aligned(r.cos, 16) && r.sin_j == 1 && r.cos_j == 1 &&
         ((r.sin_n | r.cos_n) & 3) == 0;
}

bool expanded(const flash_prologue_rows& r, int64_t B, int64_t H, int64_t N) {
  return (B > 1 && r.b == 0) || (H > 1 && r.h == 0) || (N > 1 && r.n == 0);
}

RowStrides strides(const flash_prologue_rows& r) { return RowStrides{r.b, r.h, r.n}; }

int sms_of_device() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return sms;
}

GqaTables tables_of(const flash_prologue_rotation& r) {
  GqaTables t{};
  t.sin = r.sin;
  t.cos = r.cos;
  t.sin_n = r.sin_n;
  t.sin_j = r.sin_j;
  t.cos_n = r.cos_n;
  t.cos_j = r.cos_j;
  t.rows = r.rows;
  return t;
}

// Heads of one token (or tokens of one head) next to each other in memory.
bool heads_inner(const flash_prologue_rows& q, int64_t H, int64_t N) {
  if (N == 1) return true;
  return H > 1 && llabs(q.h) <= llabs(q.n);
}

// Positions of several axes: count, bits, and no pair of an axis that there is none of.
int axes_checks(const flash_prologue_axes* x, const flash_prologue_rotation& r, int64_t D) {
  if (!x->positions || x->count < 1 || x->count > 4 || (x->position_bits != 32 && x->position_bits != 64))
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  for (int64_t j = 0; j < D / 2; ++j)
    if ((int64_t)(x->pairs[j >> 5] >> (2 * (j & 31)) & 3) >= x->count) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  return r.rows < (int64_t(1) << 31) ? FLASH_PROLOGUE_OK : FLASH_PROLOGUE_ERR_UNSUPPORTED;
}

int gqa_checks(const flash_prologue_gqa_args* a, const flash_prologue_axes* axes) {
  if (!a || a->B < 0 || a->N < 0 || a->Hq < 0 || a->Hk < 0) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (!(a->eps > 0) || !isfinite(a->eps)) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (!supported(a->D, a->dtype) || a->Hq > kMaxGqaHeads || a->B >= (int64_t(1) << 31) || a->N >= (int64_t(1) << 31) ||
      a->B * a->N >= (int64_t(1) << 31) - (1 << 20))
    return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  if (a->Hk > 0 ? a->Hq % a->Hk != 0 : a->Hq != 0) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (a->B * a->N * a->Hq == 0) return FLASH_PROLOGUE_OK;
  if (!a->q.data || !a->k.data || !a->rmsnorm_weight || !a->scales || !a->rotation.sin || !a->rotation.cos)
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (axes) {
    const int st = axes_checks(axes, a->rotation, a->D);
    if (st != FLASH_PROLOGUE_OK) return st;
  } else if (a->positions ? (a->position_bits != 32 && a->position_bits != 64) : a->rotation.rows < a->N)
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (!aligned(a->rmsnorm_weight, 16)) return FLASH_PROLOGUE_ERR_ALIGNMENT;
  if (expanded(a->q, a->B, a->Hq, a->N) || expanded(a->k, a->B, a->Hk, a->N)) return FLASH_PROLOGUE_ERR_EXPANDED;
  return FLASH_PROLOGUE_OK;
}

void set_axes(GqaTables* t, const flash_prologue_axes* x) {
  t->positions = x->positions;
  t->pos_b = x->position_b;
  t->pos_n = x->position_n;
  t->pos_is64 = x->position_bits == 64;
  t->axes = (int)x->count;
  t->pos_axis = x->position_axis;
  for (int i = 0; i < 4; ++i) t->pair_axes[i] = x->pairs[i];
}

GqaTables tables_of(const flash_prologue_gqa_args* a, const flash_prologue_axes* axes) {
  GqaTables t = tables_of(a->rotation);
  if (axes) {
    set_axes(&t, axes);
    return t;
  }
  t.positions = a->positions;
  t.pos_b = a->position_b;
  t.pos_n = a->position_n;
  t.pos_is64 = a->position_bits == 64;
  return t;
}

}  // namespace

int check_cache(const flash_prologue_cache& c, int64_t tokens, size_t es) {
  if (c.batch < 0 || c.num_pages < 0 || c.max_pages < 0 || c.page_size < 8 || (c.page_size & (c.page_size - 1)))
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (c.batch >= (1 << 24) || c.page_size > (1 << 20) || c.num_pages >= (int64_t(1) << 31) ||
      c.max_pages >= (int64_t(1) << 30) / c.page_size)
    return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  if (!c.cu_seqlens && tokens != c.batch) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return FLASH_PROLOGUE_OK;
  if (c.batch == 0) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (!c.seq_lens || (c.max_pages > 0 && !c.page_table) || (c.num_pages > 0 && (!c.k || !c.v)))
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  for (int64_t s : {c.k_page, c.k_slot, c.k_head, c.v_page, c.v_slot, c.v_head})
    if ((s * (int64_t)es) & 15) return FLASH_PROLOGUE_ERR_ALIGNMENT;
  if (!aligned(c.k, 16) || !aligned(c.v, 16)) return FLASH_PROLOGUE_ERR_ALIGNMENT;
  return FLASH_PROLOGUE_OK;
}

int check_scales(const flash_prologue_scales& s, const flash_prologue_cache& c, int64_t D) {
  if (c.num_pages > 0 && (!s.k || !s.v)) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  for (int64_t x : {s.k_page, s.k_slot, s.k_head, s.v_page, s.v_slot, s.v_head})
    if (x & (D / 32 - 1)) return FLASH_PROLOGUE_ERR_ALIGNMENT;
  return aligned(s.k, D / 16) && aligned(s.v, D / 16) ? FLASH_PROLOGUE_OK : FLASH_PROLOGUE_ERR_ALIGNMENT;
}

}  // namespace flash_prologue

using namespace flash_prologue;

extern "C" {

static int gqa_fwd(const flash_prologue_gqa_args* a, const flash_prologue_axes* axes, void* stream) {
  const int st = gqa_checks(a, axes);
  if (st != FLASH_PROLOGUE_OK || a->B * a->N * a->Hq == 0) return st;
  if (!a->q_out.data || !a->k_out.data) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (expanded(a->q_out, a->B, a->Hq, a->N) || expanded(a->k_out, a->B, a->Hk, a->N))
    return FLASH_PROLOGUE_ERR_EXPANDED;
  const size_t es = elem_size(a->dtype);
  const bool vec = rows_vec(a->q, es) && rows_vec(a->k, es) && rows_vec(a->q_out, es) && rows_vec(a->k_out, es) &&
                   rotation_vec(a->rotation);
  const int sms = sms_of_device();
  if (sms <= 0) return FLASH_PROLOGUE_ERR_CUDA;
  GqaFwdArgs g{};
  const flash_prologue_rows* in[2] = {&a->q, &a->k};
  const flash_prologue_rows* out[2] = {&a->q_out, &a->k_out};
  for (int t = 0; t < 2; ++t) {
    g.x[t] = in[t]->data;
    g.sx[t] = strides(*in[t]);
    g.y[t] = out[t]->data;
    g.sy[t] = strides(*out[t]);
  }
  g.w = a->rmsnorm_weight;
  g.scales = a->scales;
  g.tab = tables_of(a, axes);
  g.B = a->B;
  g.N = a->N;
  g.H[0] = (int)a->Hq;
  g.H[1] = (int)a->Hk;
  g.eps = (float)a->eps;
  g.p = plan_rows(a->B * a->N, g.H[0], g.H[1], 0, (int)a->D, heads_inner(a->q, a->Hq, a->N), 16LL * sms);
  return launch_gqa_fwd(g, (int)a->dtype, (int)a->D, vec, static_cast<cudaStream_t>(stream)) == cudaSuccess
             ? FLASH_PROLOGUE_OK
             : FLASH_PROLOGUE_ERR_CUDA;
}

int flash_prologue_gqa_bwd_workspace_size(int64_t Hq, int64_t D, size_t* bytes) {
  if (!bytes) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  *bytes = 0;
  if (Hq < 0) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (!supported(D, 0) || Hq > kMaxGqaHeads) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  const int sms = sms_of_device();
  if (sms <= 0) return FLASH_PROLOGUE_ERR_CUDA;
  *bytes = (size_t)kGqaBwdMaxCtasPerSm * sms * (size_t)(2 * D + Hq) * sizeof(float);
  return FLASH_PROLOGUE_OK;
}

static int gqa_bwd(const flash_prologue_gqa_args* a, const flash_prologue_axes* axes, void* stream) {
  int st = gqa_checks(a, axes);
  if (st != FLASH_PROLOGUE_OK) return st;
  if (!a->grad_rmsnorm_weight || !a->grad_scales) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->B * a->N * a->Hq == 0) {
    if (a->peers) return FLASH_PROLOGUE_ERR_UNSUPPORTED;  // every rank must add rows
    if (cudaMemsetAsync(a->grad_rmsnorm_weight, 0, sizeof(float) * 2 * a->D, s) != cudaSuccess ||
        (a->Hq > 0 && cudaMemsetAsync(a->grad_scales, 0, sizeof(float) * a->Hq, s) != cudaSuccess))
      return FLASH_PROLOGUE_ERR_CUDA;
    return FLASH_PROLOGUE_OK;
  }
  if (!a->grad_q_out.data || !a->grad_k_out.data || !a->grad_q.data || !a->grad_k.data)
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (expanded(a->grad_q, a->B, a->Hq, a->N) || expanded(a->grad_k, a->B, a->Hk, a->N))
    return FLASH_PROLOGUE_ERR_EXPANDED;
  BwdReduce red;
  if (a->peers) {
    if (!valid_peers(a->peers, a->epoch, 2 * a->D + a->Hq)) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
    red.peers = a->peers;
    red.epoch = (uint32_t)a->epoch;
  }
  size_t need = 0;
  st = flash_prologue_gqa_bwd_workspace_size(a->Hq, a->D, &need);
  if (st != FLASH_PROLOGUE_OK) return st;
  if (!a->workspace || a->workspace_bytes < (int64_t)need || !aligned(a->workspace, 16))
    return FLASH_PROLOGUE_ERR_WORKSPACE;
  const size_t es = elem_size(a->dtype);
  const bool vec = rows_vec(a->q, es) && rows_vec(a->k, es) && rows_vec(a->grad_q_out, es) &&
                   rows_vec(a->grad_k_out, es) && rows_vec(a->grad_q, es) && rows_vec(a->grad_k, es) &&
                   rotation_vec(a->rotation);
  const int sms = sms_of_device();
  GqaBwdArgs g{};
  const flash_prologue_rows* in[2] = {&a->q, &a->k};
  const flash_prologue_rows* up[2] = {&a->grad_q_out, &a->grad_k_out};
  const flash_prologue_rows* out[2] = {&a->grad_q, &a->grad_k};
  for (int t = 0; t < 2; ++t) {
    g.x[t] = in[t]->data;
    g.sx[t] = strides(*in[t]);
    g.gy[t] = up[t]->data;
    g.sgy[t] = strides(*up[t]);
    g.dx[t] = out[t]->data;
    g.sdx[t] = strides(*out[t]);
  }
  g.w = a->rmsnorm_weight;
  g.scales = a->scales;
  g.tab = tables_of(a, axes);
  g.partials = static_cast<float*>(a->workspace);
  g.B = a->B;
  g.N = a->N;
  g.H[0] = (int)a->Hq;
  g.H[1] = (int)a->Hk;
  g.eps = (float)a->eps;
  g.p = plan_rows(a->B * a->N, g.H[0], g.H[1], 0, (int)a->D, heads_inner(a->q, a->Hq, a->N), 16LL * sms);
  return launch_gqa_bwd(g, a->grad_rmsnorm_weight, a->grad_scales, (int)a->dtype, (int)a->D, vec, red, s) ==
                 cudaSuccess
             ? FLASH_PROLOGUE_OK
             : FLASH_PROLOGUE_ERR_CUDA;
}

int flash_prologue_gqa_fwd(const flash_prologue_gqa_args* a, void* stream) { return gqa_fwd(a, nullptr, stream); }
int flash_prologue_gqa_bwd(const flash_prologue_gqa_args* a, void* stream) { return gqa_bwd(a, nullptr, stream); }
int flash_prologue_gqa_fwd_axes(const flash_prologue_gqa_args* a, const flash_prologue_axes* axes, void* stream) {
  return axes ? gqa_fwd(a, axes, stream) : FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
}
int flash_prologue_gqa_bwd_axes(const flash_prologue_gqa_args* a, const flash_prologue_axes* axes, void* stream) {
  return axes ? gqa_bwd(a, axes, stream) : FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
}

// scales: null, or K and V go to a cache of 4 bits.
static int append_paged(const flash_prologue_append_args* a, const flash_prologue_scales* scales,
                        const flash_prologue_axes* axes, void* stream) {
  if (!a || a->tokens < 0 || a->Hq < 0 || a->Hk < 0) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (!(a->eps > 0) || !isfinite(a->eps)) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (!supported(a->D, a->dtype) || a->Hq > kMaxGqaHeads || a->tokens >= (int64_t(1) << 31) - (1 << 20))
    return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  if (scales && ((a->D != 64 && a->D != 128) || a->dtype == FLASH_PROLOGUE_FP32)) return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  if (a->Hk > 0 ? a->Hq % a->Hk != 0 : a->Hq != 0) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  const flash_prologue_cache& c = a->cache;
  int st = scales ? check_cache(c, a->tokens, 1) : check_cache(c, a->tokens, elem_size(a->dtype));
  if (st != FLASH_PROLOGUE_OK || a->tokens == 0 || a->Hq == 0) return st;
  if (scales && (st = check_scales(*scales, c, a->D)) != FLASH_PROLOGUE_OK) return st;
  if (axes && (st = axes_checks(axes, a->rotation, a->D)) != FLASH_PROLOGUE_OK) return st;
  if (!a->q.data || !a->k.data || !a->v.data || !a->q_out.data || !a->rotation.sin || !a->rotation.cos)
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (!aligned(a->rmsnorm_weight, 16)) return FLASH_PROLOGUE_ERR_ALIGNMENT;
  if (expanded(a->q_out, 1, a->Hq, a->tokens)) return FLASH_PROLOGUE_ERR_EXPANDED;
  if (c.k_slot == 0 || c.v_slot == 0 || (c.num_pages > 1 && (c.k_page == 0 || c.v_page == 0)) ||
      (a->Hk > 1 && (c.k_head == 0 || c.v_head == 0)))
    return FLASH_PROLOGUE_ERR_EXPANDED;  // slots that are written must be apart
  if (scales && (scales->k_slot == 0 || scales->v_slot == 0 ||
                 (c.num_pages > 1 && (scales->k_page == 0 || scales->v_page == 0)) ||
                 (a->Hk > 1 && (scales->k_head == 0 || scales->v_head == 0))))
    return FLASH_PROLOGUE_ERR_EXPANDED;
  const size_t es = elem_size(a->dtype);
  const bool vec = rows_vec(a->q, es) && rows_vec(a->k, es) && rows_vec(a->v, es) && rows_vec(a->q_out, es) &&
                   rotation_vec(a->rotation);
  const int sms = sms_of_device();
  if (sms <= 0) return FLASH_PROLOGUE_ERR_CUDA;
  GqaFwdArgs g{};
  const flash_prologue_rows* in[3] = {&a->q, &a->k, &a->v};
  for (int t = 0; t < 3; ++t) {
    g.x[t] = in[t]->data;
    g.sx[t] = strides(*in[t]);
  }
  g.y[0] = a->q_out.data;
  g.sy[0] = strides(a->q_out);
  g.y[1] = c.k;
  g.sy[1] = RowStrides{c.k_page, c.k_head, c.k_slot};
  g.y[2] = c.v;
  g.sy[2] = RowStrides{c.v_page, c.v_head, c.v_slot};
  g.w = a->rmsnorm_weight;
  g.scales = a->scales;
  g.tab = tables_of(a->rotation);
  if (axes) set_axes(&g.tab, axes);
  if (scales) {
    g.scale[0] = static_cast<uint16_t*>(scales->k);
    g.scale[1] = static_cast<uint16_t*>(scales->v);
    g.ss[0] = RowStrides{scales->k_page, scales->k_head, scales->k_slot};
    g.ss[1] = RowStrides{scales->v_page, scales->v_head, scales->v_slot};
  }
  g.append = true;
  g.paged = paged_target(c);
  g.B = 1;
  g.N = a->tokens;
  g.H[0] = (int)a->Hq;
  g.H[1] = g.H[2] = (int)a->Hk;
  g.eps = (float)a->eps;
  g.p = plan_rows(a->tokens, g.H[0], g.H[1], g.H[2], (int)a->D, heads_inner(a->q, a->Hq, a->tokens), 16LL * sms);
  return launch_gqa_fwd(g, (int)a->dtype, (int)a->D, vec, static_cast<cudaStream_t>(stream)) == cudaSuccess
             ? FLASH_PROLOGUE_OK
             : FLASH_PROLOGUE_ERR_CUDA;
}

int flash_prologue_append_paged(const flash_prologue_append_args* a, void* stream) {
  return append_paged(a, nullptr, nullptr, stream);
}
int flash_prologue_append_paged_axes(const flash_prologue_append_args* a, const flash_prologue_axes* axes, void* stream) {
  return axes ? append_paged(a, nullptr, axes, stream) : FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
}
int flash_prologue_append_paged_int4(const flash_prologue_append_args* a, const flash_prologue_scales* scales,
                                     const flash_prologue_axes* axes, void* stream) {
  return scales ? append_paged(a, scales, axes, stream) : FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
}

}  // extern "C"
