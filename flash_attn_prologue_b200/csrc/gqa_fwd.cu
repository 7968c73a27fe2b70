// Grouped-query prologue, forward: rows of Q (Hq heads) and K (Hk heads) with
// per-head RMSNorm, the split-half rotation of the token's position and the Q
// scale, written to dense outputs, or with K and V going to the pages of a
// cache (append). Per row
//   y = x / sqrt(mean(x^2) + eps) * w;  o = R(pos) y;  Q: o *= exp(scale[h])
// with the arithmetic (and rounding order) of the equal-heads forward.
//
// Bound by HBM: every row is read and written once, the tables once a token.
// A lane owns one chunk pair of a row (rotation partners in one lane) and a
// warp owns a token group: HS heads x TP tokens at a time, the token's sin/cos
// kept in registers while it walks the heads of Q, K and V. kAhead row blocks
// are loaded before the first is used, so a warp has that many KB in flight.
#include "gqa_rows.cuh"

namespace flash_prologue {
namespace {

constexpr int kAhead = 2;

// Request of packed token `u`: the last b with cu[b] <= u (requests without
// new tokens share a start with the next one).
__device__ __forceinline__ int request_of(const int32_t* cu, int batch, int64_t u) {
  int lo = 0, hi = batch;  // cu[lo] <= u < cu[hi] unless u is outside every request
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= u) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kThreads) gqa_fwd_kernel(const GqaFwdArgs a) {
  constexpr int L = D / 16;
  constexpr int HALF = D / 2;
  const int lane = threadIdx.x & 31;
  const int slot = lane / L;
  const int j0 = (lane % L) * kChunk;
  const int HS = 1 << a.p.log2_hs;
  const int TP = (32 / L) >> a.p.log2_hs;
  const int hslot = slot & (HS - 1), tslot = slot >> a.p.log2_hs;
  const int64_t items = a.p.groups * a.p.slices;
  const int64_t warps = (int64_t)gridDim.x * kWarps;
  const int all_iters = a.p.iters[0] + a.p.iters[1] + a.p.iters[2];

  for (int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); item < items; item += warps) {
    const int64_t group = a.p.slices == 1 ? item : item / a.p.slices;
    const int i0 = (int)(item - group * a.p.slices) * a.p.per_slice;
    const int i1 = min(i0 + a.p.per_slice, all_iters);
    const int64_t token = group * TP + tslot;
    // Where this lane's token lies, and the row of the tables that turns it.
    bool there = token < a.B * a.N;
    int64_t b = 0, n = token, pos = -1, page = 0, in_page = 0;
    if (there) {
      if (a.paged.page_table) {
        const PagedTarget& pg = a.paged;
        int64_t first = token, count = 1;
        int64_t r = token;
        if (pg.cu_seqlens) {
          r = request_of(pg.cu_seqlens, pg.batch, token);
          first = __ldg(pg.cu_seqlens + r);
          count = (int64_t)__ldg(pg.cu_seqlens + r + 1) - first;
        }
        // Tokens past the last request (padding) belong to none: their Q rows come out as zeros.
        if (token >= first && token < first + count) {
          const int64_t at = (int64_t)__ldg(pg.seq_lens + r) - count + (token - first);
          bool ok = at >= 0 && at < a.tab.rows && (at >> pg.page_log2) < pg.max_pages;
          if (ok) {
            page = __ldg(pg.page_table + r * pg.table_stride + (at >> pg.page_log2));
            ok = page >= 0 && page < pg.num_pages;
          }
          if (ok) {
            pos = at;
            in_page = at & ((1 << pg.page_log2) - 1);
          } else {
            atomicOr(&g_device_error, kDeviceErrorIndex);
          }
        }
      } else {
        if (a.B > 1) {
          b = token / a.N;
          n = token - b * a.N;
        }
        pos = rotation_row(a.tab, b, n);
      }
    }
    float sn[kChunk], cs[kChunk];
    if (pos >= 0) {
      load_table<VEC>(sn, a.tab.sin + pos * a.tab.sin_n + j0 * a.tab.sin_j, a.tab.sin_j);
      load_table<VEC>(cs, a.tab.cos + pos * a.tab.cos_n + j0 * a.tab.cos_j, a.tab.cos_j);
    } else {
      // A position out of range rotates by NaN (dense rows); a token without a place gives zeros.
      const float v = a.paged.page_table ? 0.f : __int_as_float(0x7fc00000);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) { sn[j] = v; cs[j] = v; }
    }

    float wa[kChunk], wb[kChunk];
    int w_of = -1;
    for (int i = i0; i < i1; i += kAhead) {
      Chunk<T> x1[kAhead], x2[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        int t = 0, it = i + k;
        if (it >= a.p.iters[0]) { it -= a.p.iters[0]; t = 1; }
        if (t == 1 && it >= a.p.iters[1]) { it -= a.p.iters[1]; t = 2; }
        const int h = it * HS + hslot;
        if (there && i + k < i1 && h < a.H[t]) {
          const T* p = static_cast<const T*>(a.x[t]) + b * a.sx[t].b + h * a.sx[t].h + n * a.sx[t].n + j0;
          load_stream<T, VEC>(x1[k], p);
          load_stream<T, VEC>(x2[k], p + HALF);
        } else {
          chunk_zero(x1[k]);
          chunk_zero(x2[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (i + k >= i1) break;
        int t = 0, it = i + k;
        if (it >= a.p.iters[0]) { it -= a.p.iters[0]; t = 1; }
        if (t == 1 && it >= a.p.iters[1]) { it -= a.p.iters[1]; t = 2; }
        const int h = it * HS + hslot;
        const bool ok = there && h < a.H[t];
        const bool to_cache = t != 0 && a.paged.page_table;
        T* out = static_cast<T*>(a.y[t]) + h * a.sy[t].h + j0 +
                 (to_cache ? page * a.sy[t].b + in_page * a.sy[t].n : b * a.sy[t].b + n * a.sy[t].n);
        const bool store = ok && !(to_cache && pos < 0);
        if (t == 2) {
          if (store) {
            store_stream<T, VEC>(out, x1[k]);
            store_stream<T, VEC>(out + HALF, x2[k]);
          }
          continue;
        }
        if (w_of != t) {
          w_of = t;
#pragma unroll
          for (int j = 0; j < kChunk; ++j) {
            wa[j] = a.w ? __ldg(a.w + t * D + j0 + j) : 1.f;
            wb[j] = a.w ? __ldg(a.w + t * D + HALF + j0 + j) : 1.f;
          }
        }
        float r = 1.f;
        if (a.w) r = inv_rms<D>(row_sum<L>(lane_sumsq(x1[k], x2[k])), a.eps);
        if (!store) continue;  // after the shuffles: every lane took part in them
        const bool scale = t == 0 && a.scales;
        Chunk<T> o1, o2;
        fwd_lane(x1[k], x2[k], r, wa, wb, sn, cs, scale, scale ? expf(__ldg(a.scales + h)) : 1.f, o1, o2);
        if (pos < 0 && a.paged.page_table) {  // also where the row holds infinities
          chunk_zero(o1);
          chunk_zero(o2);
        }
        store_stream<T, VEC>(out, o1);
        store_stream<T, VEC>(out + HALF, o2);
      }
    }
  }
}

const void* fwd_kernel_for(int dtype, int D, bool vec) { FLASH_PROLOGUE_GQA_KERNEL(gqa_fwd_kernel) }

}  // namespace

// HS is the largest power of two that divides both head counts (no idle slot)
// and fits the warp's 32 / L slots; where positions lie next to each other in
// memory (dense [B, H, N, D] views) a warp takes consecutive tokens of one head.
RowsPlan plan_rows(int64_t tokens, int Hq, int Hk, int Hv, int D, bool heads_inner, int64_t want_warps) {
  RowsPlan p{};
  const int slots = 32 / (D / 16);
  int hs = 1;
  while (heads_inner && hs * 2 <= slots && Hq % (hs * 2) == 0 && Hk % (hs * 2) == 0) {
    hs *= 2;
    ++p.log2_hs;
  }
  const int tp = slots / hs;
  p.iters[0] = (Hq + hs - 1) / hs;
  p.iters[1] = (Hk + hs - 1) / hs;
  p.iters[2] = (Hv + hs - 1) / hs;
  p.groups = (tokens + tp - 1) / tp;
  const int all = p.iters[0] + p.iters[1] + p.iters[2];
  int64_t slices = p.groups > 0 ? (want_warps + p.groups - 1) / p.groups : 1;
  if (slices > all) slices = all;
  if (slices < 1) slices = 1;
  p.per_slice = (int)((all + slices - 1) / slices);
  p.slices = (all + p.per_slice - 1) / p.per_slice;
  return p;
}

cudaError_t launch_gqa_fwd(const GqaFwdArgs& a, int dtype, int D, bool vec, cudaStream_t stream) {
  const void* fn = fwd_kernel_for(dtype, D, vec);
  if (!fn) return cudaErrorInvalidValue;
  const int64_t grid = persistent_grid(fn, 0, (a.p.groups * a.p.slices + kWarps - 1) / kWarps);
  if (grid <= 0) return cudaErrorInvalidConfiguration;
  GqaFwdArgs args = a;
  void* params[] = {&args};
  return cudaLaunchKernel(fn, dim3((unsigned)grid), dim3(kThreads), params, 0, stream);
}

cudaError_t read_gqa_fwd_device_error(int* value, bool reset) {
  cudaError_t err = cudaMemcpyFromSymbol(value, g_device_error, sizeof(int));
  if (err != cudaSuccess || !reset) return err;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
}

}  // namespace flash_prologue
