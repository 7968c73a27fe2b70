// Grouped-query prologue, forward: rows of Q (Hq heads) and K (Hk heads) with
// per-head RMSNorm, the split-half rotation of the token's position and the Q
// scale, written to dense outputs, or with K and V going to the pages of a
// cache (append). Per row
//   y = x / sqrt(mean(x^2) + eps) * w;  o = R(pos) y;  Q: o *= exp(scale[h])
// with the arithmetic (and rounding order) of the equal-heads forward. Into a
// cache of 4 bits K and V go as codes and scales (int4_rows.cuh), from FP32.
//
// Bound by HBM: every row is read and written once, the tables once a token.
// A lane owns one chunk pair of a row (rotation partners in one lane) and a
// warp owns a token group: HS heads x TP tokens at a time, the token's sin/cos
// kept in registers while it walks the heads of Q, K and V. Its loads go through
// a ring in shared memory: each lane copies its own chunks with cp.async,
// kStages - 1 row blocks ahead, and reads back only what it copied.
#include "gqa_rows.cuh"
#include "int4_rows.cuh"

namespace flash_prologue {
namespace {

// Slots of the ring. 65,536 tokens x 40 heads x 128 BF16, forward and backward:
// 553 us with the ring, 569 with four row blocks loaded into registers at a time.
constexpr int kStages = 4;

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

// 1 / sqrt(mean + eps) from a sum in 64 bits, rounded once: where a row is rounded to codes, those do
// not depend on the order of its sum. The hardware's approximation (relative error below 2^-22) and one
// step of Newton's iteration in 64 bits, which leaves 2^-43.
template <typename T, int D, int L>
__device__ __forceinline__ float inv_rms_exact(const Chunk<T>& x1, const Chunk<T>& x2, float eps) {
  double sum = 0;
#pragma unroll
  for (int p = 0; p < kPairs; ++p) {
    const float2 a = chunk_get2(x1, p), b = chunk_get2(x2, p);
    sum = fma((double)a.x, (double)a.x, fma((double)a.y, (double)a.y, sum));
    sum = fma((double)b.x, (double)b.x, fma((double)b.y, (double)b.y, sum));
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const double m = sum * (1.0 / D) + (double)eps;
  const float y = rsqrtf((float)m);
  if (y == 0.f) return y;  // as where the sum of squares leaves FP32
  return (float)fma((double)y, fma(-0.5 * m, (double)y * (double)y, 0.5), (double)y);
}

template <typename T, int D, bool VEC, bool AXES, bool INT4 = false>
__global__ void __launch_bounds__(kThreads, 3) gqa_fwd_kernel(const GqaFwdArgs a) {
  constexpr int L = D / 16;
  constexpr int HALF = D / 2;
  using C = Columns<T, D>;
  constexpr int kStageBytes = VEC ? 2 * C::kPieces * 512 : 0;  // x1, x2 of 32 lanes
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int lane = threadIdx.x & 31;
  unsigned char* ring = smem_raw + (threadIdx.x >> 5) * kStages * kStageBytes + lane * 16;
  const uint32_t ring_u = smem_u32(ring);
  const int slot = lane / L;
  const int j0 = Columns<T, D>::first(lane % L);
  const int HS = 1 << a.p.log2_hs;
  const int TP = (32 / L) >> a.p.log2_hs;
  const int hslot = slot & (HS - 1), tslot = slot >> a.p.log2_hs;
  // Items, tokens and rows are counted in 32 bits (the host checks): fewer registers and no 64-bit division.
  const int items = (int)(a.p.groups * a.p.slices), warps = gridDim.x * kWarps, tokens = (int)(a.B * a.N), N = (int)a.N;
  const bool paged = a.append;  // the table may be null: one without columns has no address
  const int q_iters = a.p.iters[0], qk_iters = q_iters + a.p.iters[1], all_iters = qk_iters + a.p.iters[2];

  // The loads' walk over the warp's row blocks: for each of its token groups the
  // slice's head blocks of Q, K and V. `pre_in` points at this lane's first columns.
  int pre_item = blockIdx.x * kWarps + (threadIdx.x >> 5), pre_i = 0, pre_i1 = 0, pre_b = 0, pre_n = 0;
  bool pre_there = false;
  const T* pre_in = nullptr;
  const auto pre_at = [&](int t, int it) {
    pre_in = static_cast<const T*>(a.x[t]) + pre_b * a.sx[t].b + (it * HS + hslot) * a.sx[t].h + pre_n * a.sx[t].n + j0;
  };
  const auto pre_enter = [&]() {
    if (pre_item >= items) return;
    const int group = a.p.slices == 1 ? pre_item : pre_item / a.p.slices;
    pre_i = (pre_item - group * a.p.slices) * a.p.per_slice;
    pre_i1 = min(pre_i + a.p.per_slice, all_iters);
    const int token = group * TP + tslot;
    pre_there = token < tokens;  // the pointer stays at a token that exists
    pre_b = 0;
    pre_n = pre_there ? token : 0;
    if (a.B > 1) {
      pre_b = pre_n / N;
      pre_n -= pre_b * N;
    }
    if (pre_i < q_iters) pre_at(0, pre_i);
    else if (pre_i < qk_iters) pre_at(1, pre_i - q_iters);
    else pre_at(2, pre_i - qk_iters);
  };
  const auto prefetch = [&](int stage) {
    if constexpr (VEC) {
      if (pre_item < items) {
        const uint32_t dst = ring_u + stage * kStageBytes;
#pragma unroll
        for (int q = 0; q < C::kPieces; ++q) {
          cp_async16(dst + q * 512, pre_in + q * C::kApart, pre_there);
          cp_async16(dst + (C::kPieces + q) * 512, pre_in + HALF + q * C::kApart, pre_there);
        }
        ++pre_i;
        if (pre_i == pre_i1) {
          pre_item += warps;
          pre_enter();
        } else if (pre_i == q_iters) {
          pre_at(1, 0);
        } else if (pre_i == qk_iters) {
          pre_at(2, 0);
        } else {
          pre_in += HS * (pre_i < q_iters ? a.sx[0].h : pre_i < qk_iters ? a.sx[1].h : a.sx[2].h);
        }
      }
      cp_async_commit();  // an empty group past the end keeps the count
    }
  };
  if constexpr (VEC) {
    pre_enter();
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) prefetch(s);
  }
  int stage = 0;

  for (int item = blockIdx.x * kWarps + (threadIdx.x >> 5); item < items; item += warps) {
    const int group = a.p.slices == 1 ? item : item / a.p.slices;
    const int i0 = (item - group * a.p.slices) * a.p.per_slice, i1 = i0 + a.p.per_slice;
    const int token = group * TP + tslot;
    // Where this lane's token lies, and the row of the tables that turns it.
    const bool there = token < tokens;
    int b = 0, n = there ? token : 0, page = 0, in_page = 0;
    int64_t pos = -1;
    [[maybe_unused]] int rows[4];  // AXES: pos only says whether the token is turned and placed
    if (there) {
      if (paged) {
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
          bool ok = at >= 0 && (AXES || at < a.tab.rows) && (at >> pg.page_log2) < pg.max_pages;
          if (ok) {
            page = __ldg(pg.page_table + r * pg.table_stride + (at >> pg.page_log2));
            ok = page >= 0 && page < pg.num_pages;
          }
          if constexpr (AXES) {
            if (ok) ok = rotation_rows(a.tab, 0, token, rows);
          }
          if (ok) {
            pos = at;
            in_page = (int)at & ((1 << pg.page_log2) - 1);
          } else {
            atomicOr(&g_device_error, kDeviceErrorIndex);
          }
        }
      } else {
        if (a.B > 1) {
          b = token / N;
          n = token - b * N;
        }
        if constexpr (AXES) pos = rotation_rows(a.tab, b, n, rows) ? 0 : -1;
        else pos = rotation_row(a.tab, b, n);
      }
    }
    const bool placed = pos >= 0;
    float sn[kChunk], cs[kChunk];
    if constexpr (AXES)
      load_turned<T, D, VEC>(sn, cs, a.tab, rows, placed, j0, a.p.log2_hs, hslot, (tslot << a.p.log2_hs) * L + lane % L);
    if (placed) {
      if constexpr (!AXES) {
        load_columns<T, D, VEC>(sn, a.tab.sin + pos * a.tab.sin_n + j0 * a.tab.sin_j, a.tab.sin_j);
        load_columns<T, D, VEC>(cs, a.tab.cos + pos * a.tab.cos_n + j0 * a.tab.cos_j, a.tab.cos_j);
      }
    } else {
      // A position out of range rotates by NaN (dense rows); a token without a place gives zeros.
      const float v = paged ? 0.f : __int_as_float(0x7fc00000);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) { sn[j] = v; cs[j] = v; }
    }

    // The slice's row blocks of Q, then K, then V; HS divides their heads.
    int begin = 0;
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      const int it0 = max(i0 - begin, 0), it1 = min(i1 - begin, a.p.iters[t]);
      begin += a.p.iters[t];
      if (it0 >= it1) continue;
      const int h0 = it0 * HS + hslot;
      const bool to_cache = t != 0 && paged;
      const T* in = static_cast<const T*>(a.x[t]) + b * a.sx[t].b + h0 * a.sx[t].h + n * a.sx[t].n + j0;
      T* out = static_cast<T*>(a.y[t]) + h0 * a.sy[t].h + j0 +
               (to_cache ? page * a.sy[t].b + in_page * a.sy[t].n : b * a.sy[t].b + n * a.sy[t].n);
      const bool store = there && (placed || !to_cache);
      // A cache of 4 bits: this lane's word of a row's first half, its scale (one of two lanes writes it).
      unsigned char* codes = nullptr;
      uint16_t* scale = nullptr;
      if constexpr (INT4) {
        if (t != 0) {
          codes = static_cast<unsigned char*>(a.y[t]) + h0 * a.sy[t].h + page * a.sy[t].b + in_page * a.sy[t].n +
                  lane % L * 4;
          scale = a.scale[t - 1] + h0 * a.ss[t - 1].h + page * a.ss[t - 1].b + in_page * a.ss[t - 1].n + lane % L;
        }
      }
      float wa[kChunk], wb[kChunk];
      const float* scales = t == 0 ? a.scales : nullptr;
      if (t != 2) {
        if (a.w) {
          load_columns<T, D, true>(wa, a.w + t * D + j0, 1);
          load_columns<T, D, true>(wb, a.w + t * D + HALF + j0, 1);
        } else {
#pragma unroll
          for (int j = 0; j < kChunk; ++j) wa[j] = wb[j] = 1.f;
        }
      }
      for (int it = it0; it < it1; ++it) {
        Chunk<T> x1, x2;
        if constexpr (VEC) {
          prefetch(stage == 0 ? kStages - 1 : stage - 1);
          cp_async_wait<kStages - 1>();
          const uint4* src = reinterpret_cast<const uint4*>(ring + stage * kStageBytes);
#pragma unroll
          for (int q = 0; q < C::kPieces; ++q) {
            const uint4 v0 = src[q * 32], v1 = src[(C::kPieces + q) * 32];
            x1.w[4 * q] = v0.x; x1.w[4 * q + 1] = v0.y; x1.w[4 * q + 2] = v0.z; x1.w[4 * q + 3] = v0.w;
            x2.w[4 * q] = v1.x; x2.w[4 * q + 1] = v1.y; x2.w[4 * q + 2] = v1.z; x2.w[4 * q + 3] = v1.w;
          }
          if (++stage == kStages) stage = 0;
        } else if (there) {
          load_chunk<T, D, false>(x1, in);
          load_chunk<T, D, false>(x2, in + HALF);
          in += HS * a.sx[t].h;
        } else {
          chunk_zero(x1);
          chunk_zero(x2);
        }
        if constexpr (INT4) {
          if (t != 0) {
            float2 o1[kPairs], o2[kPairs];
            if (t == 1) {
              const float r = a.w ? inv_rms_exact<T, D, L>(x1, x2, a.eps) : 1.f;
              fwd_lane_values(x1, x2, r, wa, wb, sn, cs, false, 1.f, o1, o2);
            } else {
#pragma unroll
              for (int p = 0; p < kPairs; ++p) {
                o1[p] = chunk_get2(x1, p);
                o2[p] = chunk_get2(x2, p);
              }
            }
            uint32_t w1, w2;
            uint16_t s;
            int4_encode<T, L>(o1, o2, w1, w2, s);
            if (store) {
              *reinterpret_cast<uint32_t*>(codes) = w1;
              *reinterpret_cast<uint32_t*>(codes + D / 4) = w2;
              if (lane % L < L / 2) *scale = s;
            }
            codes += HS * a.sy[t].h;
            scale += HS * a.ss[t - 1].h;
            continue;
          }
        }
        if (t != 2) {
          const float r = a.w ? inv_rms<D>(row_sum<L>(lane_sumsq(x1, x2)), a.eps) : 1.f;
          const float e = scales ? expf(__ldg(scales + it * HS + hslot)) : 1.f;
          fwd_lane(x1, x2, r, wa, wb, sn, cs, scales != nullptr, e, x1, x2);
          if (!placed && paged) {  // also where the row holds infinities
            chunk_zero(x1);
            chunk_zero(x2);
          }
        }
        if (store) {
          store_chunk<T, D, VEC>(out, x1);
          store_chunk<T, D, VEC>(out + HALF, x2);
        }
        out += HS * a.sy[t].h;
      }
    }
  }
  if constexpr (VEC) cp_async_wait<0>();
}

const void* fwd_kernel_for(int dtype, int D, bool vec, bool axes) { FLASH_PROLOGUE_GQA_KERNEL(gqa_fwd_kernel) }

template <typename T, bool AXES>
const void* int4_kernel_of(int D, bool vec) {
  if (D == 64)
    return vec ? reinterpret_cast<const void*>(&gqa_fwd_kernel<T, 64, true, AXES, true>)
               : reinterpret_cast<const void*>(&gqa_fwd_kernel<T, 64, false, AXES, true>);
  return vec ? reinterpret_cast<const void*>(&gqa_fwd_kernel<T, 128, true, AXES, true>)
             : reinterpret_cast<const void*>(&gqa_fwd_kernel<T, 128, false, AXES, true>);
}
const void* int4_kernel_for(int dtype, int D, bool vec, bool axes) {
  if (axes) return dtype == 0 ? int4_kernel_of<__nv_bfloat16, true>(D, vec) : int4_kernel_of<__half, true>(D, vec);
  return dtype == 0 ? int4_kernel_of<__nv_bfloat16, false>(D, vec) : int4_kernel_of<__half, false>(D, vec);
}

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
  p.iters[0] = Hq / hs;
  p.iters[1] = Hk / hs;
  p.iters[2] = Hv / hs;
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
  const bool axes = a.tab.axes != 0;
  const void* fn = a.scale[0] ? int4_kernel_for(dtype, D, vec, axes) : fwd_kernel_for(dtype, D, vec, axes);
  if (!fn) return cudaErrorInvalidValue;
  const size_t smem = vec ? (size_t)kWarps * kStages * (dtype == 2 ? 2048 : 1024) : 0;
  if (smem > 48 * 1024) {
    const cudaError_t err = allow_shared_memory(fn, smem);
    if (err != cudaSuccess) return err;
  }
  const int64_t grid = persistent_grid(fn, smem, (a.p.groups * a.p.slices + kWarps - 1) / kWarps);
  if (grid <= 0) return cudaErrorInvalidConfiguration;
  GqaFwdArgs args = a;
  void* params[] = {&args};
  return cudaLaunchKernel(fn, dim3((unsigned)grid), dim3(kThreads), params, smem, stream);
}

cudaError_t read_gqa_fwd_device_error(int* value, bool reset) {
  cudaError_t err = cudaMemcpyFromSymbol(value, g_device_error, sizeof(int));
  if (err != cudaSuccess || !reset) return err;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
}

}  // namespace flash_prologue
