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
#include "paged_attention.h"

namespace flash_prologue {
namespace {

constexpr int kRows = 16;       // rows of a tile
constexpr int kWarpKeys = 16;   // keys of a warp's step
constexpr int kDecodeWarps = 4;
constexpr int kDecodeThreads = kDecodeWarps * 32;
constexpr int kBlockKeys = kWarpKeys * kDecodeWarps;
constexpr int kNone = -(1 << 30);  // below every relative position
constexpr int kWholeKeys = 256; // longest caches whose items are never split
constexpr int kRing = 3;        // steps of a warp's ring

struct Part {  // an item that a CTA began and others go on with
  int token0;  // packed index of its first row's request
  int row0, rows;  // rows of the tile that exist
  int kv_head;
  int last;        // CTA that ends it; -1: nothing to join
};

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
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// Blocks of keys from the first that the request's first new token sees to its last key.
__device__ __forceinline__ int first_key(const Request& q, int window) {
  return window ? max(q.total - q.news - window + 1, 0) : 0;
}
__device__ __forceinline__ int blocks_of(const Request& q, int window) {
  const int lo = first_key(q, window) / kBlockKeys, hi = (q.total + kBlockKeys - 1) / kBlockKeys;
  return max(hi - lo, 1);  // one at least: it writes the zeros of rows without keys
}
// Row tiles times key heads, each an item of blocks_of() blocks.
__device__ __forceinline__ int64_t items_of(const Request& q, const AttentionArgs& a) {
  return (int64_t)((q.news * a.group + kRows - 1) / kRows) * a.kv_heads;
}
// Units of an item: `cut` blocks at most in each.
__device__ __forceinline__ int units_of_item(int blocks, int cut) {
  return cut == 1 ? blocks : (blocks + cut - 1) / cut;
}

// Sums of two values over the CTA (every thread gets them).
__device__ __forceinline__ void cta_sum(int64_t (&v)[2], int64_t (*scratch)[2]) {
  if (__all_sync(0xffffffffu, (v[0] | v[1]) >> 24 == 0)) {
    v[0] = __reduce_add_sync(0xffffffffu, (unsigned)v[0]);
    v[1] = __reduce_add_sync(0xffffffffu, (unsigned)v[1]);
  } else {
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
      for (int i = 0; i < 2; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if ((threadIdx.x & 31) == 0) {
    scratch[threadIdx.x >> 5][0] = v[0];
    scratch[threadIdx.x >> 5][1] = v[1];
  }
  __syncthreads();
  v[0] = v[1] = 0;
#pragma unroll
  for (int w = 0; w < kDecodeWarps; ++w) {
    v[0] += scratch[w][0];
    v[1] += scratch[w][1];
  }
}

// Blocks of a unit. 1: every CTA takes an equal run of units, which may begin
// and end inside items. Where a run crosses an item's border its CTA fills and
// empties its pipeline twice; with fewer items than CTAs, items can be cut into
// pieces of a CTA each instead, longer than the runs. Worth it up to about a
// quarter more and 3 blocks: pieces (runs) of 6 requests x 8,192 keys, 32/8 x
// 128: 39.7 (43.1) us; 16 x up to 6 tokens, 4,096 keys, 16/4 x 64: 17.6 (19.6);
// not taken, pieces half as long again: 32 x 4,096 keys, 16/4 x 64: 27.4 (26.0).
// (kAll: an item is a unit.)
constexpr int kAll = 1 << 30;
__device__ __forceinline__ int cut_of(const AttentionArgs& a, int64_t blocks, int64_t items) {
  const int64_t grid = gridDim.x;
  if (a.whole) return kAll;
  if (blocks <= grid || items >= grid || blocks >= int64_t(1) << 30) return 1;
  // The sum of ceil(b / cut) over the items is below blocks / cut + items <= grid.
  const int cut = (int)(blocks + grid - items - 1) / (int)(grid - items), run = (int)blocks / (int)grid;
  return cut <= run + run / 4 + 3 ? cut : 1;
}

template <typename T, int D>
__global__ void __launch_bounds__(kDecodeThreads) paged_decode_kernel(const AttentionArgs a) {
  constexpr int kRowBytes = D * 2;
  constexpr int kStepBytes = 2 * kWarpKeys * kRowBytes;  // K then V
  constexpr int kPerLane = kWarpKeys * (D / 8) / 32;     // 16-byte pieces of K (and of V) a lane loads
  constexpr int kTiles = D / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int64_t scratch[kDecodeWarps], sums[kDecodeWarps][2];
  __shared__ int64_t found[2];  // request of the CTA's next unit, units before it
  __shared__ float stat[kDecodeWarps][kRows][2];
  __shared__ int bad_page;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int batch = requests_of(a.pages);
  const uint32_t ring = smem_u32(smem) + warp * kRing * kStepBytes;

  if (!a.whole) start_next_kernel();
  // This CTA's run of units.
  int64_t total[2] = {0, 0}, my_items = 0;  // blocks and items of all requests; items of this thread's last one
  int my_blocks = 0;
  bool bad = false;
  for (int r = threadIdx.x; r < batch; r += kDecodeThreads) {
    bool b;
    const Request q = request_at(a.pages, a.tokens, a.max_keys, r, &b);
    bad |= b;
    my_items = items_of(q, a);
    my_blocks = blocks_of(q, a.window);
    total[0] += my_items * my_blocks;
    total[1] += my_items;
  }
  if (bad) atomicOr(&g_device_error, kDeviceErrorIndex);
  if (threadIdx.x == 0) found[0] = -1;
  cta_sum(total, sums);
  const int cut = cut_of(a, total[0], total[1]);
  const bool pieces = cut > 1 && !a.whole;  // a CTA has one unit
  const int64_t units = a.whole ? total[1] : total[0];  // where CTAs have runs of them
  const int64_t slots = 2 * (int64_t)gridDim.x, cta = blockIdx.x;
  float* part_out = static_cast<float*>(a.workspace);                    // [slots][kRows][D]
  float* part_stat = part_out + slots * kRows * D;                       // [slots][kRows][2]
  Part* parts = reinterpret_cast<Part*>(part_stat + slots * kRows * 2);  // [grid]
  if (threadIdx.x == 0 && !a.whole) parts[cta].last = -1;
  const int64_t ctas = min((int64_t)gridDim.x, units);  // every one of these has a unit at least
  if (cta >= ctas) return;
  const bool small = units < (int64_t(1) << 31) / 1024;  // the products below fit 32 bits
  const int64_t begin = pieces ? cta : small ? (int)cta * (int)units / (int)ctas : cta * units / ctas;
  const int64_t end = pieces ? cta + 1 : small ? ((int)cta + 1) * (int)units / (int)ctas : (cta + 1) * units / ctas;

  // The request that `begin` falls into: one scan over the requests, a CTA's width at a time.
  int64_t before = 0;
  for (int r0 = 0; r0 < batch; r0 += kDecodeThreads) {
    const int r = r0 + threadIdx.x;
    int64_t n = my_items * units_of_item(my_blocks, cut);  // one request a thread: read already
    if (batch > kDecodeThreads) {
      n = 0;
      if (r < batch) {
        bool b;
        const Request q = request_at(a.pages, a.tokens, a.max_keys, r, &b);
        n = items_of(q, a) * units_of_item(blocks_of(q, a.window), cut);
      }
    }
    int64_t upto = n;  // inclusive sum within the warp
    if (small) {
      int low = (int)n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, low, o);
        if (lane >= o) low += v;
      }
      upto = low;
    } else {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = upto;
    __syncthreads();
    int64_t start = before + upto - n, all = 0;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      if (w < warp) start += scratch[w];
      all += scratch[w];
    }
    if (begin >= start && begin < start + n) {
      found[0] = r;
      found[1] = start;
    }
    before += all;
    if (before > begin) break;  // the same for every thread
  }
  __syncthreads();
  if (found[0] < 0) return;  // fewer pieces than CTAs
  int r = (int)found[0];
  int64_t start = found[1];

  for (int64_t unit = begin; unit < end;) {
    bool too_long;  // more tokens than the page table has room for
    Request q = request_at(a.pages, a.tokens, a.max_keys, r, &too_long);
    int64_t in_request = items_of(q, a) * units_of_item(blocks_of(q, a.window), cut);
    while (unit >= start + in_request) {
      start += in_request;
      ++r;
      q = request_at(a.pages, a.tokens, a.max_keys, r, &too_long);
      in_request = items_of(q, a) * units_of_item(blocks_of(q, a.window), cut);
    }
    const int blocks = blocks_of(q, a.window), per_item = units_of_item(blocks, cut);
    const int size = cut == 1 ? 1 : (blocks + per_item - 1) / per_item;  // blocks of a unit, evenly
    const int64_t in = unit - start;
    const int item = in >> 31 ? (int)(in / per_item) : (int)in / per_item;  // tiles x heads stay below 2^31
    const int64_t item_start = start + (int64_t)item * per_item;
    const int u0 = (int)(unit - item_start), u1 = (int)min((int64_t)per_item, end - item_start);
    const int b0 = u0 * size, b1 = min(u1 * size, blocks);
    const int head = item % a.kv_heads;
    const int row0 = item / a.kv_heads * kRows;       // of the request's news * group rows
    const int rows = min(kRows, q.news * a.group - row0);
    const int base = q.total - q.news;                // position of new token 0
    const int key0 = first_key(q, a.window) / kBlockKeys * kBlockKeys;
    // Keys that a row of this tile sees.
    const int hi = base + (row0 + rows - 1) / a.group + 1;
    const int lo = a.window ? max(base + row0 / a.group - a.window + 1, 0) : 0;

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
    if (threadIdx.x == 0) bad_page = too_long;
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
    const int32_t* table = a.pages.page_table + (int64_t)r * a.pages.table_stride;
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
    if (threadIdx.x == 0 && b0 == 0 && b1 < blocks) {
      Part p;
      p.token0 = q.first;
      p.row0 = row0;
      p.rows = rows;
      p.kv_head = head;
      p.last = (int)(pieces ? item_start + per_item - 1 : ((item_start + per_item) * ctas - 1) / units);
      parts[cta] = p;
    }
    unit = item_start + u1;
    __syncthreads();
  }
}

// Joins the parts of one row of the item that CTA blockIdx.x of the first kernel
// began: every warp takes each eighth part, its columns over the lanes.
constexpr int kJoinWarps = 8;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const AttentionArgs a, int64_t ctas) {
  constexpr int kCols = D / 32;  // columns of a lane
  __shared__ float joined[kJoinWarps][D], sums[kJoinWarps], tops[kJoinWarps];
  const float* part_out = static_cast<const float*>(a.workspace);
  const float* part_stat = part_out + 2 * ctas * kRows * D;
  wait_for_previous_kernel();
  const Part p = reinterpret_cast<const Part*>(part_stat + 2 * ctas * kRows * 2)[blockIdx.x];
  const int row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (p.last < 0 || row >= p.rows) return;
  const int first = blockIdx.x, parts = p.last - first + 1;
  float top = -INFINITY, sum = 0.f, o[kCols] = {};
  constexpr int kFlight = 4;
  for (int i0 = warp; i0 < parts; i0 += kJoinWarps * kFlight) {
    float2 st[kFlight];
    float x[kFlight][kCols];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int i = i0 + f * kJoinWarps;
      st[f] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int c = 0; c < kCols; ++c) x[f][c] = 0.f;
      if (i < parts) {
        // Part i is in the second slot of the CTA that began the item, in the first slot of the others.
        const int64_t at = (2 * (int64_t)(first + i) + (i == 0)) * kRows + row;
        st[f] = __ldcg(reinterpret_cast<const float2*>(part_stat + at * 2));
        const float* src = part_out + at * D + lane * kCols;
        if constexpr (kCols == 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
          x[f][0] = v.x; x[f][1] = v.y; x[f][2] = v.z; x[f][3] = v.w;
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          x[f][0] = v.x; x[f][1] = v.y;
        }
      }
    }
    float now = top;
#pragma unroll
    for (int f = 0; f < kFlight; ++f) now = fmaxf(now, st[f].x);
    const float from = now == -INFINITY ? 0.f : now, moved = exp2_approx(top - from);
    top = now;
    sum *= moved;
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c] *= moved;
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const float e = exp2_approx(st[f].x - from);
      sum += e * st[f].y;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[c] += e * x[f][c];
    }
  }
#pragma unroll
  for (int c = 0; c < kCols; ++c) joined[warp][lane * kCols + c] = o[c];
  if (lane == 0) {
    sums[warp] = sum;
    tops[warp] = top;
  }
  __syncthreads();
  const int col = threadIdx.x;
  if (col >= D) return;
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) m = fmaxf(m, tops[w]);
  const float from = m == -INFINITY ? 0.f : m;
  float v = 0.f, l = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    const float e = exp2_approx(tops[w] - from);
    v += e * joined[w][col];
    l += e * sums[w];
  }
  const int at = p.row0 + row, token = at / a.group;
  const int h = p.kv_head * a.group + (at - token * a.group);
  static_cast<T*>(a.out)[(p.token0 + token) * a.out_n + h * a.out_h + col] = from_float<T>(l == 0.f ? 0.f : v / l);
  if (a.lse && col == 0) a.lse[(int64_t)(p.token0 + token) * a.heads + h] = (m + log2f(l) - kProbabilityShift<T>) * 0.6931471805599453f;
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
  return launch_following(paged_join_kernel<T, D>, dim3((unsigned)grid, rows), dim3(kJoinWarps * 32), stream, a, grid);
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
