// Grouped-query prologue, backward: dq, dk and the sums over tokens and heads
// of d rmsnorm_weight [2, D] and d scales [Hq]. Per row (d0 = R^T g, re = r e,
// n' = x re, u = d0 w, s = <u, n'>; e = exp(scale[h]) for Q, 1 for K)
//   dx = re u - n' (r / e) s / D;   d w += d0 n';   d scale[h] += s
// (bwd_lane_reduce / lane_dx), with r recomputed from x.
//
// Bound by HBM: x and g are read once, dx is written once; the sums stay in
// registers (d w: each lane's 16 columns, for Q and for K) and shared memory
// (d scale: one row of Hq sums a warp) until the end of the persistent CTA,
// which writes one partial row; the rows are added in a fixed order, so equal
// inputs give equal bits. The accumulators leave a thread too few registers to
// keep enough row loads in flight, so the loads go through a ring in shared
// memory: each lane copies its own chunks with cp.async, kStages row blocks
// ahead, and reads back only what it copied (no barrier between lanes).
#include "gqa_rows.cuh"

namespace flash_prologue {
namespace {

constexpr int kStages = 3;
constexpr float kSmallScale = 0x1p-115f;

// A warp's walk over its row blocks: for each of its token groups the slice's
// head blocks of Q, then of K. `in` and `g` point at this lane's first columns.
template <typename T>
struct Walk {
  int item;
  int i, i1;          // head block of Q and K together, end of the slice
  const T* in[2];
  bool there;         // this lane's token exists (the pointers stay put where not)
};

template <typename T, int D, bool VEC, bool AXES>
__global__ void __launch_bounds__(kThreads, 2) gqa_bwd_kernel(const GqaBwdArgs a) {
  constexpr int L = D / 16;
  constexpr int HALF = D / 2;
  using C = Columns<T, D>;
  constexpr int kStageBytes = VEC ? 4 * C::kPieces * 512 : 0;  // x1, x2, g1, g2 of 32 lanes
  extern __shared__ __align__(16) unsigned char smem_raw[];
  float* w_s = reinterpret_cast<float*>(smem_raw);  // [q, k][half][lane of a row][8]: as the lanes own them
  float2* e_s = reinterpret_cast<float2*>(w_s + 2 * D);  // [Hq] e = exp(scale), 1 / e
  float* ds_s = reinterpret_cast<float*>(e_s + a.H[0]);  // [kWarps][Hq]
  float* dw_s = ds_s + kWarps * a.H[0];                  // [kWarps][2 * D]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t floats = (uint32_t)(2 * D + a.H[0] * (kWarps + 2) + kWarps * 2 * D);
  unsigned char* ring = smem_raw + ((floats * 4 + 15) & ~15u) + warp * kStages * kStageBytes + lane * 16;
  const uint32_t ring_u = smem_u32(ring);
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    const int c = i / kChunk % L, j = i % kChunk;
    w_s[i] = a.w[i / HALF * HALF + C::of(c, j)];
  }
  for (int i = threadIdx.x; i < a.H[0]; i += kThreads) {
    const float v = a.scales[i];
    const float e = expf(v);
    // Where 1 / e may be infinite it is kept as 2^-32 / e (0 where e has vanished), and s is 2^32 times as large beside it.
    e_s[i] = make_float2(e, e >= kSmallScale ? expf(-v) : e > 0.f ? 0x1p-32f / e : 0.f);
  }
  for (int i = threadIdx.x; i < kWarps * a.H[0]; i += kThreads) ds_s[i] = 0.f;
  __syncthreads();

  const int slot = lane / L, c_lane = lane % L;
  const int j0 = C::first(c_lane);
  const int HS = 1 << a.p.log2_hs;
  const int TP = (32 / L) >> a.p.log2_hs;
  const int hslot = slot & (HS - 1), tslot = slot >> a.p.log2_hs;
  // Items, tokens and rows are counted in 32 bits (the host checks): fewer registers and no 64-bit division.
  const int items = (int)(a.p.groups * a.p.slices), warps = gridDim.x * kWarps, tokens = (int)(a.B * a.N), N = (int)a.N;
  const int q_iters = a.p.iters[0], all_iters = q_iters + a.p.iters[1];

  float2 acc[2][2][kPairs];  // d w of this lane's columns: [q, k][first, second half]
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int p = 0; p < kPairs; ++p) acc[t][0][p] = acc[t][1][p] = make_float2(0.f, 0.f);

  // This lane's token of an item, and its first row of tensor t under head block it.
  const auto token_of = [&](int item, int& b, int& n, int& i) {
    const int group = a.p.slices == 1 ? item : item / a.p.slices;
    i = (item - group * a.p.slices) * a.p.per_slice;
    const int token = group * TP + tslot;
    const bool there = token < tokens;
    b = 0;
    n = there ? token : 0;
    if (a.B > 1) {
      b = n / N;
      n -= b * N;
    }
    return there;
  };
  Walk<T> pre;
  int pre_b = 0, pre_n = 0;
  const auto pre_at = [&](int t, int it) {
    const int h = it * HS + hslot;
    pre.in[0] = static_cast<const T*>(a.x[t]) + pre_b * a.sx[t].b + h * a.sx[t].h + pre_n * a.sx[t].n + j0;
    pre.in[1] = static_cast<const T*>(a.gy[t]) + pre_b * a.sgy[t].b + h * a.sgy[t].h + pre_n * a.sgy[t].n + j0;
  };
  const auto pre_enter = [&]() {
    if (pre.item >= items) return;
    pre.there = token_of(pre.item, pre_b, pre_n, pre.i);
    pre.i1 = min(pre.i + a.p.per_slice, all_iters);
    if (pre.i < q_iters) pre_at(0, pre.i);
    else pre_at(1, pre.i - q_iters);
  };
  pre.item = blockIdx.x * kWarps + warp;
  pre_enter();

  const auto prefetch = [&](int stage) {
    if constexpr (VEC) {
      if (pre.item < items) {
        const uint32_t dst = ring_u + stage * kStageBytes;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int q = 0; q < C::kPieces; ++q) {
            cp_async16(dst + ((2 * s) * C::kPieces + q) * 512, pre.in[s] + q * C::kApart, pre.there);
            cp_async16(dst + ((2 * s + 1) * C::kPieces + q) * 512, pre.in[s] + HALF + q * C::kApart, pre.there);
          }
        ++pre.i;
        if (pre.i == pre.i1) {
          pre.item += warps;
          pre_enter();
        } else if (pre.i == q_iters) {
          pre_at(1, 0);
        } else {
          pre.in[0] += HS * (pre.i < q_iters ? a.sx[0].h : a.sx[1].h);
          pre.in[1] += HS * (pre.i < q_iters ? a.sgy[0].h : a.sgy[1].h);
        }
      }
      cp_async_commit();  // an empty group past the end keeps the count
    }
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) prefetch(s);

  int stage = 0;
  for (int item = blockIdx.x * kWarps + warp; item < items; item += warps) {
    int b, n, i0;
    const bool there = token_of(item, b, n, i0);
    const int i1 = i0 + a.p.per_slice;
    float sn[kChunk], cs[kChunk];
    int64_t pos;
    [[maybe_unused]] int rows[4];
    if constexpr (AXES) pos = there && rotation_rows(a.tab, b, n, rows) ? 0 : -1;
    else pos = there ? rotation_row(a.tab, b, n) : -1;
    if constexpr (AXES)
      load_turned<T, D, VEC>(sn, cs, a.tab, rows, pos >= 0, j0, a.p.log2_hs, hslot, (tslot << a.p.log2_hs) * L + c_lane);
    if (pos >= 0) {
      if constexpr (!AXES) {
        load_columns<T, D, VEC>(sn, a.tab.sin + pos * a.tab.sin_n + j0 * a.tab.sin_j, a.tab.sin_j);
        load_columns<T, D, VEC>(cs, a.tab.cos + pos * a.tab.cos_n + j0 * a.tab.cos_j, a.tab.cos_j);
      }
    } else {
      const float v = there ? __int_as_float(0x7fc00000) : 0.f;  // as in the forward
#pragma unroll
      for (int j = 0; j < kChunk; ++j) { sn[j] = v; cs[j] = v; }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int begin = t ? q_iters : 0;
      const int it0 = max(i0 - begin, 0), it1 = min(i1 - begin, a.p.iters[t]);
      if (it0 >= it1) continue;
      const int h0 = it0 * HS + hslot;
      T* out = static_cast<T*>(a.dx[t]) + b * a.sdx[t].b + h0 * a.sdx[t].h + n * a.sdx[t].n + j0;
      const float* wa = w_s + t * D + c_lane * kChunk;
      const float* wb = wa + HALF;
      for (int it = it0; it < it1; ++it) {
        const int h = it * HS + hslot;
        Chunk<T> x1, x2, g1, g2;
        if constexpr (VEC) {
          int ahead = stage + kStages - 1;
          if (ahead >= kStages) ahead -= kStages;
          prefetch(ahead);
          cp_async_wait<kStages - 1>();
          const uint4* src = reinterpret_cast<const uint4*>(ring + stage * kStageBytes);
#pragma unroll
          for (int q = 0; q < C::kPieces; ++q) {
            const uint4 v0 = src[(0 * C::kPieces + q) * 32], v1 = src[(1 * C::kPieces + q) * 32];
            const uint4 v2 = src[(2 * C::kPieces + q) * 32], v3 = src[(3 * C::kPieces + q) * 32];
            x1.w[4 * q] = v0.x; x1.w[4 * q + 1] = v0.y; x1.w[4 * q + 2] = v0.z; x1.w[4 * q + 3] = v0.w;
            x2.w[4 * q] = v1.x; x2.w[4 * q + 1] = v1.y; x2.w[4 * q + 2] = v1.z; x2.w[4 * q + 3] = v1.w;
            g1.w[4 * q] = v2.x; g1.w[4 * q + 1] = v2.y; g1.w[4 * q + 2] = v2.z; g1.w[4 * q + 3] = v2.w;
            g2.w[4 * q] = v3.x; g2.w[4 * q + 1] = v3.y; g2.w[4 * q + 2] = v3.z; g2.w[4 * q + 3] = v3.w;
          }
          if (++stage == kStages) stage = 0;
        } else if (there) {
          const T* x = static_cast<const T*>(a.x[t]) + b * a.sx[t].b + h * a.sx[t].h + n * a.sx[t].n + j0;
          const T* g = static_cast<const T*>(a.gy[t]) + b * a.sgy[t].b + h * a.sgy[t].h + n * a.sgy[t].n + j0;
          load_chunk<T, D, false>(x1, x);
          load_chunk<T, D, false>(x2, x + HALF);
          load_chunk<T, D, false>(g1, g);
          load_chunk<T, D, false>(g2, g + HALF);
        } else {
          chunk_zero(x1);
          chunk_zero(x2);
          chunk_zero(g1);
          chunk_zero(g2);
        }
        const float r = inv_rms_bwd<D>(row_sum<L>(lane_sumsq2(x1, x2)), a.eps);
        const float2 e = t == 0 ? e_s[h] : make_float2(1.f, 1.f);
        const float re = r * e.x;
        float2 u1[kPairs], u2[kPairs], n1[kPairs], n2[kPairs];
        const float s = row_sum<L>(
            bwd_lane_reduce(x1, x2, g1, g2, re, wa, wb, sn, cs, acc[t][0], acc[t][1], u1, u2, n1, n2));
        if (t == 0) {
          float sum = s;  // over the warp's tokens of this head
          for (int o = L * HS; o < 32; o <<= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
          if (c_lane == 0 && tslot == 0) ds_s[warp * a.H[0] + h] += sum;
        }
        if (there) {
          const float lift = e.x >= kSmallScale ? 1.f : 0x1p32f;
          lane_dx(n1, n2, u1, u2, re, r * (s * lift * (1.f / D)) * e.y, x1, x2);
          store_chunk<T, D, VEC>(out, x1);
          store_chunk<T, D, VEC>(out + HALF, x2);
        }
        out += HS * a.sdx[t].h;
      }
    }
  }
  if constexpr (VEC) cp_async_wait<0>();

  // d w: over the warp's row slots, then over the CTA's warps.
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float v[kChunk];
      unpair(acc[t][half], v);
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
#pragma unroll
        for (int o = L; o < 32; o <<= 1) v[j] = __fadd_rn(v[j], __shfl_xor_sync(0xffffffffu, v[j], o));
        if (slot == 0) dw_s[warp * 2 * D + t * D + half * HALF + C::of(c_lane, j)] = v[j];
      }
    }
  }
  __syncthreads();
  const int C2 = 2 * D + a.H[0];
  float* out = a.partials + (int64_t)blockIdx.x * C2;
  for (int col = threadIdx.x; col < C2; col += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      v = __fadd_rn(v, col < 2 * D ? dw_s[w * 2 * D + col] : ds_s[w * a.H[0] + col - 2 * D]);
    out[col] = v;
  }
}

const void* bwd_kernel_for(int dtype, int D, bool vec, bool axes) { FLASH_PROLOGUE_GQA_KERNEL(gqa_bwd_kernel) }

size_t smem_bytes(int Hq, int D, int dtype, bool vec) {
  const size_t floats = (size_t)2 * D + (size_t)Hq * (kWarps + 2) + (size_t)kWarps * 2 * D;
  const size_t stage = vec ? (dtype == 2 ? 4096 : 2048) : 0;
  return ((floats * 4 + 15) & ~(size_t)15) + kWarps * kStages * stage;
}

// The kernel with its shared memory allowed (above 48 KB it has to be asked for).
const void* ready_kernel(int Hq, int D, int dtype, bool vec, bool axes, size_t* smem) {
  const void* fn = bwd_kernel_for(dtype, D, vec, axes);
  if (!fn) return nullptr;
  *smem = smem_bytes(Hq, D, dtype, vec);
  if (*smem > 48 * 1024 && allow_shared_memory(fn, *smem) != cudaSuccess) return nullptr;
  return fn;
}

}  // namespace

int64_t gqa_bwd_grid(const RowsPlan& p, int Hq, int D, int dtype, bool vec, bool axes) {
  size_t smem = 0;
  const void* fn = ready_kernel(Hq, D, dtype, vec, axes, &smem);
  if (!fn) return -1;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return -1;
  const int64_t want = (p.groups * p.slices + kWarps - 1) / kWarps, most = (int64_t)kGqaBwdMaxCtasPerSm * sms;
  return persistent_grid(fn, smem, want < most ? want : most);
}

cudaError_t launch_gqa_bwd(const GqaBwdArgs& a, float* dw, float* ds, int dtype, int D, bool vec,
                           const BwdReduce& red, cudaStream_t stream) {
  size_t smem = 0;
  const void* fn = ready_kernel(a.H[0], D, dtype, vec, a.tab.axes != 0, &smem);
  const int64_t grid = gqa_bwd_grid(a.p, a.H[0], D, dtype, vec, a.tab.axes != 0);
  if (!fn || grid <= 0) return cudaErrorInvalidConfiguration;
  GqaBwdArgs args = a;
  void* params[] = {&args};
  const cudaError_t err = cudaLaunchKernel(fn, dim3((unsigned)grid), dim3(kThreads), params, smem, stream);
  if (err != cudaSuccess) return err;
  return launch_bwd_reduce(a.partials, grid, 2 * D + a.H[0], 2 * D, dw, ds, red, stream);
}

cudaError_t read_gqa_bwd_device_error(int* value, bool reset) {
  cudaError_t err = cudaMemcpyFromSymbol(value, g_device_error, sizeof(int));
  if (err != cudaSuccess || !reset) return err;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
}

}  // namespace flash_prologue
