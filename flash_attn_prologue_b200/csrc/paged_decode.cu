// Attention of a few new tokens a request over a paged cache (single tokens,
// drafted tokens): o_i = sum_j p_ij v_j with p the softmax of the scaled scores
// over the keys that row i sees (causal, optional window).
//
// Bound by HBM: the K and V of every request have to be read once and each key
// meets few rows. The rows of one key head -- its query heads times the new
// tokens -- are packed into tiles of 16, so one read of a key serves them all,
// and both products run on 16 x 8 x 16 matrix instructions, far from their
// limit. Work is counted in blocks of 64 keys over all requests, row tiles and
// key heads, and every CTA of a full GPU takes an equal run of them, whatever
// the requests' lengths (with few items, a piece of one: cut_of). Where a run
// ends inside an item its part goes to the workspace (row maximum, sum and
// unscaled output, FP32) and a second kernel joins the parts in order. A warp
// takes 16 of a block's keys and loads them with cp.async into a ring of its
// own, two blocks ahead, so no barrier stands between a load and its use; the
// four warps join at an item's end.
//
// Scores, softmax statistics and outputs are FP32; the probabilities are
// rounded to the cache's type for the second product (their sum is taken
// before the rounding), an error of the size of the output's own rounding.
#include "paged_runs.cuh"

namespace flash_prologue {
namespace {

constexpr int kRows = 16;       // rows of a tile
constexpr int kBlockKeys = kWarpKeys * kDecodeWarps;
using Tiles = Tiling<kRows, kBlockKeys, 1>;
constexpr int kRing = 3;        // steps of a warp's ring

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  const int bytes = ok ? 16 : 0;  // 0: zeros, src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Infinity or NaN in either half of a pair of 16-bit values.
template <typename T>
__device__ __forceinline__ bool non_finite(uint32_t pair) {
  constexpr uint32_t m = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (pair & m) == m || (pair >> 16 & m) == m;
}
template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T, int D>
__global__ void __launch_bounds__(kDecodeThreads) paged_decode_kernel(const AttentionArgs a) {
  constexpr int kRowBytes = D * 2;
  constexpr int kStepBytes = 2 * kWarpKeys * kRowBytes;  // K then V
  constexpr int kPerLane = kWarpKeys * (D / 8) / 32;     // 16-byte pieces of K (and of V) a lane loads
  constexpr int kTiles = D / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ RunScratch shared;
  __shared__ float stat[kDecodeWarps][kRows][2];
  __shared__ int bad_page;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem) + warp * kRing * kStepBytes;

  if (!a.whole) start_next_kernel();
  const int64_t slots = 2 * (int64_t)gridDim.x, cta = blockIdx.x;
  float* part_out = static_cast<float*>(a.workspace);                    // [slots][kRows][D]
  float* part_stat = part_out + slots * kRows * D;                       // [slots][kRows][2]
  Part* parts = reinterpret_cast<Part*>(part_stat + slots * kRows * 2);  // [grid]
  Run run;
  if (!find_run<Tiles>(a, shared, parts, run)) return;

  for (int64_t unit = run.begin; unit < run.end;) {
    Item it;
    find_item<Tiles>(a, run, unit, it);
    const Request& q = it.q;
    const int b0 = it.b0, b1 = it.b1, blocks = it.blocks, head = it.head, row0 = it.row0, rows = it.rows, base = it.base,
              key0 = it.key0, hi = it.hi, lo = it.lo;

    // The tile's Q as operand fragments: rows lane / 4 and lane / 4 + 8.
    uint32_t qf[D / 16][4];
    int row_pos[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int row = lane / 4 + s * 8;
      const int at = row0 + row, i = at / a.group;
      row_pos[s] = row < rows ? base + i : -1;
      const T* p = static_cast<const T*>(a.q) + (q.first + i) * a.q_n +
                   (head * a.group + (at - i * a.group)) * a.q_h + (lane % 4) * 2;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        qf[c][s] = row < rows ? __ldg(reinterpret_cast<const uint32_t*>(p + c * 16)) : 0;
        qf[c][s + 2] = row < rows ? __ldg(reinterpret_cast<const uint32_t*>(p + c * 16 + 8)) : 0;
      }
    }
    float acc[kTiles][4], top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    if (threadIdx.x == 0) bad_page = it.too_long;
    __syncthreads();

    // Positions relative to this warp's first key, in 32 bits (a request has fewer than 2^30 keys).
    const int steps = b1 - b0;
    const int warp_key = key0 + b0 * kBlockKeys + warp * kWarpKeys;
    const int key_lo = lo - warp_key, key_hi = hi - warp_key;
    const int all_lo = a.window ? base + (row0 + rows - 1) / a.group - a.window + 1 - warp_key : kNone;
    const int all_hi = base + row0 / a.group - warp_key;  // every row sees keys all_lo .. all_hi
    int see_lo[2], see_hi[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      see_hi[e] = row_pos[e] < 0 ? kNone : row_pos[e] - warp_key;
      see_lo[e] = a.window ? row_pos[e] - a.window + 1 - warp_key : kNone;
    }
    const int32_t* table = a.pages.page_table + (int64_t)it.r * a.pages.table_stride;
    const int in_page = (1 << a.pages.page_log2) - 1;
    // A lane's pieces of a step: rows lane / kPieces + i * kRowStep, 16 bytes at column lane % kPieces.
    constexpr int kPieces = D / 8, kRowStep = 32 / kPieces;
    const int64_t k_lane = head * a.k_head + lane / kPieces * a.k_slot + lane % kPieces * 8;
    const int64_t v_lane = head * a.v_head + lane / kPieces * a.v_slot + lane % kPieces * 8;
    int page_of[2] = {0, 0};  // pages of the 16 keys of step page_step + lane (two where pages hold 8)
    int page_step = -32;
    auto load = [&](int step) {
      if (step < steps) {
        if (step - page_step >= 32) {
          page_step = step;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int k = (step + lane) * kBlockKeys + s * 8;
            page_of[s] = 0;
            if (step + lane < steps && k < key_hi && k + 8 > key_lo) {
              page_of[s] = __ldg(table + ((warp_key + k) >> a.pages.page_log2));
              if (page_of[s] < 0 || page_of[s] >= a.pages.num_pages) {
                page_of[s] = -1;
                bad_page = 1;
              }
            }
          }
        }
        const int page[2] = {__shfl_sync(0xffffffffu, page_of[0], step - page_step),
                             __shfl_sync(0xffffffffu, page_of[1], step - page_step)};
        const int key = step * kBlockKeys;
        const uint32_t dst = ring + (step % kRing) * kStepBytes;
        const bool full = key >= key_lo && key + kWarpKeys <= key_hi && page[0] >= 0 && page[1] >= 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int slot = (warp_key + key + s * 8) & in_page;
          const T* kp = static_cast<const T*>(a.k);
          const T* vp = static_cast<const T*>(a.v);
          if (page[s] >= 0) {
            kp += page[s] * a.k_page + slot * a.k_slot + k_lane;
            vp += page[s] * a.v_page + slot * a.v_slot + v_lane;
          }
#pragma unroll
          for (int i = 0; i < kPerLane / 2; ++i) {
            const int row = s * 8 + i * kRowStep + lane / kPieces;
            const uint32_t at = dst + row * kRowBytes + ((lane % kPieces) ^ (row & 7)) * 16;
            const bool ok = full || (key + row >= key_lo && key + row < key_hi && page[s] >= 0);
            cp_async16(at, kp, ok);
            cp_async16(at + kWarpKeys * kRowBytes, vp, ok);
            if (page[s] >= 0) {
              kp += kRowStep * a.k_slot;
              vp += kRowStep * a.v_slot;
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s < kRing - 1; ++s) load(s);

    for (int step = 0; step < steps; ++step) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
      __syncwarp();
      load(step + kRing - 1);
      const int key = step * kBlockKeys;
      if (key >= key_hi || key + kWarpKeys <= key_lo) continue;
      const uint32_t ks = ring + (step % kRing) * kStepBytes, vs = ks + kWarpKeys * kRowBytes;
      float s[2][4] = {};
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        // matrices: keys 0-7 / d 0-7, keys 0-7 / d 8-15, keys 8-15 / d 0-7, keys 8-15 / d 8-15
        const int row = (lane & 7) + (lane >> 4) * 8, piece = c * 2 + ((lane >> 3) & 1);
        uint32_t b[4];
        ldmatrix4(b, ks + row * kRowBytes + ((piece ^ (row & 7)) * 16));
        mma16816<T>(s[0], qf[c], b[0], b[1]);
        mma16816<T>(s[1], qf[c], b[2], b[3]);
      }
      // Row e of this lane: scores s[n][2 e + x] of keys n * 8 + (lane % 4) * 2 + x.
      const bool edge = key < all_lo || key + kWarpKeys - 1 > all_hi;  // some row does not see some key
      float p[2][4];
      float scale[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float most = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) p[n][2 * e + x] = s[n][2 * e + x] * a.scale_log2;
        if (edge) {
          const int lo_e = see_lo[e] - key - (lane % 4) * 2, hi_e = see_hi[e] - key - (lane % 4) * 2;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              if (n * 8 + x > hi_e || n * 8 + x < lo_e) p[n][2 * e + x] = -INFINITY;
        }
        most = fmaxf(fmaxf(p[0][2 * e], p[0][2 * e + 1]), fmaxf(p[1][2 * e], p[1][2 * e + 1]));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const float now = fmaxf(top[e], most);
        const float from = now == -INFINITY ? 0.f : now;
        scale[e] = exp2_approx(top[e] - from);
        top[e] = now;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            p[n][2 * e + x] = exp2_approx(p[n][2 * e + x] - (from - kProbabilityShift<T>));
        sum[e] = sum[e] * scale[e] + ((p[0][2 * e] + p[0][2 * e + 1]) + (p[1][2 * e] + p[1][2 * e + 1]));
      }
      if (__any_sync(0xffffffffu, scale[0] != 1.f || scale[1] != 1.f)) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          acc[t][0] *= scale[0];
          acc[t][1] *= scale[0];
          acc[t][2] *= scale[1];
          acc[t][3] *= scale[1];
        }
      }
      // Where a row of the tile does not see a key that others may, an infinity or NaN in
      // that key's V must not reach it through 0 * V: such values are taken out of the
      // product and added to the rows that see them.
      if (edge) {
        uint32_t* v32 = reinterpret_cast<uint32_t*>(smem + (vs - smem_u32(smem)));
        bool wild = false;
        for (int i = lane; i < kWarpKeys * D / 2; i += 32) wild |= non_finite<T>(v32[i]);
        if (__any_sync(0xffffffffu, wild)) {
          for (int j = 0; j < kWarpKeys; ++j) {
            const T* vrow = reinterpret_cast<const T*>(smem + (vs - smem_u32(smem)) + j * kRowBytes);
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const float val = to_float(vrow[((t ^ (j & 7)) * 8) + (lane % 4) * 2 + x]);
                if (isfinite(val)) continue;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (key + j <= see_hi[e] && key + j >= see_lo[e]) acc[t][2 * e + x] += val;
              }
          }
          __syncwarp();
          for (int i = lane; i < kWarpKeys * D / 2; i += 32) {
            constexpr uint32_t m = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
            uint32_t w = v32[i];
            if ((w & m) == m) w &= 0xffff0000u;
            if ((w >> 16 & m) == m) w &= 0x0000ffffu;
            v32[i] = w;
          }
          __syncwarp();
        }
      }
      const uint32_t pf[4] = {pack2<T>(p[0][0], p[0][1]), pack2<T>(p[0][2], p[0][3]), pack2<T>(p[1][0], p[1][1]),
                              pack2<T>(p[1][2], p[1][3])};
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        // matrices (transposed): keys 0-7 / d 0-7, keys 8-15 / d 0-7, keys 0-7 / d 8-15, keys 8-15 / d 8-15
        const int row = lane & 15, piece = c * 2 + (lane >> 4);
        uint32_t b[4];
        ldmatrix4_t(b, vs + row * kRowBytes + ((piece ^ (row & 7)) * 16));
        mma16816<T>(acc[2 * c], pf, b[0], b[1]);
        mma16816<T>(acc[2 * c + 1], pf, b[2], b[3]);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // The four warps' sums over their keys, joined.
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
      sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
      if (lane % 4 == 0) {
        stat[warp][lane / 4 + e * 8][0] = top[e];
        stat[warp][lane / 4 + e * 8][1] = sum[e];
      }
    }
    float* joined = reinterpret_cast<float*>(smem) + warp * kRows * D;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float2* dst = reinterpret_cast<float2*>(joined + (lane / 4 + e * 8) * D + t * 8 + (lane % 4) * 2);
        *dst = make_float2(acc[t][2 * e], acc[t][2 * e + 1]);
      }
    __syncthreads();
    const bool whole = b0 == 0 && b1 == blocks;
    const int64_t slot = 2 * cta + (b0 == 0 ? 1 : 0);
    if (threadIdx.x == 0 && bad_page) atomicOr(&g_device_error, kDeviceErrorIndex);
    for (int i = threadIdx.x; i < rows * D; i += kDecodeThreads) {
      const int row = i / D, col = i % D;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kDecodeWarps; ++w) m = fmaxf(m, stat[w][row][0]);
      const float from = m == -INFINITY ? 0.f : m;
      float o = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kDecodeWarps; ++w) {
        const float f = exp2_approx(stat[w][row][0] - from);
        o += f * reinterpret_cast<float*>(smem)[(w * kRows + row) * D + col];
        l += f * stat[w][row][1];
      }
      if (bad_page) l = o = __int_as_float(0x7fc00000);
      if (whole) {
        const int at = row0 + row, token = at / a.group;
        const int h = head * a.group + (at - token * a.group);
        static_cast<T*>(a.out)[(q.first + token) * a.out_n + h * a.out_h + col] =
            from_float<T>(l == 0.f ? 0.f : o / l);
        if (a.lse && col == 0)
          a.lse[(int64_t)(q.first + token) * a.heads + h] = (m + log2f(l) - kProbabilityShift<T>) * 0.6931471805599453f;
      } else {
        part_out[(slot * kRows + row) * D + col] = o;
        if (col == 0) {
          part_stat[(slot * kRows + row) * 2] = m;
          part_stat[(slot * kRows + row) * 2 + 1] = l;
        }
      }
    }
    if (threadIdx.x == 0 && b0 == 0 && b1 < blocks) parts[cta] = part_of(run, it);
    unit = it.item_start + it.u1;
    __syncthreads();
  }
}

int64_t most_ctas(int D, int sms) { return (int64_t)sms * (D == 64 ? 4 : 2); }

template <typename T, int D>
cudaError_t launch(AttentionArgs a, cudaStream_t stream) {
  // Short caches: a CTA does whole items, which takes it a few steps more and saves the
  // second kernel. 32/8 heads x 128, 64 requests of 128 and 256 keys: 14.5 and 19.0 us,
  // split 20.2 and 24.2. The rule knows the table's width, not the lengths: one request of
  // 256 keys loses by it (9.4 us, split 8.2), and so do many short ones under a wide table.
  a.whole = a.max_keys <= kWholeKeys;
  constexpr size_t smem = (size_t)kDecodeWarps * kRing * 2 * kWarpKeys * D * 2;
  const void* fn = reinterpret_cast<const void*>(&paged_decode_kernel<T, D>);
  cudaError_t err = allow_shared_memory(fn, smem);
  if (err != cudaSuccess) return err;
  // Never more CTAs than there can be units.
  const int64_t tiles = (int64_t)a.tokens * a.group / kRows + (a.tokens < a.pages.batch + 2 ? a.tokens : a.pages.batch + 2);
  const int64_t blocks = a.whole ? 1 : a.max_keys / kBlockKeys + 1;
  int dev = 0, sms = 0;
  if ((err = cudaGetDevice(&dev)) != cudaSuccess ||
      (err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
    return err;
  const int64_t want = tiles * a.kv_heads * blocks, most = most_ctas(D, sms);
  const int64_t grid = persistent_grid(fn, smem, want < most ? want : most, kDecodeThreads);
  if (grid <= 0) return cudaErrorInvalidConfiguration;
  err = launch_kernel(paged_decode_kernel<T, D>, dim3((unsigned)grid), dim3(kDecodeThreads), smem, stream, a);
  if (err != cudaSuccess || a.whole) return err;
  const unsigned rows = a.pages.cu_seqlens || a.group > kRows ? kRows : a.group;  // rows a tile can have
  return launch_following(paged_join_kernel<T, D, kRows, kProbabilityShift<T> != 0>, dim3((unsigned)grid, rows), dim3(kJoinWarps * 32), stream, a, grid);
}

}  // namespace

// Room for the largest grid a device runs at once.
size_t paged_decode_workspace(int D, int sms) {
  return (size_t)most_ctas(D, sms) * (2 * kRows * (size_t)(D + 2) * sizeof(float) + sizeof(Part));
}

cudaError_t launch_paged_decode(const AttentionArgs& a, int dtype, int D, cudaStream_t stream) {
  if (D == 64) return dtype == 0 ? launch<__nv_bfloat16, 64>(a, stream) : launch<__half, 64>(a, stream);
  return dtype == 0 ? launch<__nv_bfloat16, 128>(a, stream) : launch<__half, 128>(a, stream);
}

cudaError_t read_paged_decode_device_error(int* value, bool reset) {
  cudaError_t err = cudaMemcpyFromSymbol(value, g_device_error, sizeof(int));
  if (err != cudaSuccess || !reset) return err;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
}

}  // namespace flash_prologue
