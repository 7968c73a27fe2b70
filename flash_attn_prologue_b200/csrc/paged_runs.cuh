// How the kernels for few new tokens a request (paged_decode.cu, paged_int4_decode.cu)
// share out their work: items (a tile of ROWS rows of a key head's query heads x new
// tokens, over the request's keys, for HEADS key heads next to each other) of blocks
// of KEYS keys, counted over all requests. Every CTA of a full GPU takes an equal run of blocks, or with few items a piece of
// one; items that several CTAs have are joined by a second kernel, in order.
#pragma once

#include "paged_attention.h"

namespace flash_prologue {
namespace {

constexpr int kDecodeWarps = 4;
constexpr int kDecodeThreads = kDecodeWarps * 32;
constexpr int kWarpKeys = 16;   // keys of a warp's step
template <int ROWS_, int KEYS_, int HEADS_>
struct Tiling {
  static constexpr int ROWS = ROWS_, KEYS = KEYS_, HEADS = HEADS_;
  // Head groups (the last may have fewer heads).
  static __device__ __forceinline__ int groups(const AttentionArgs& a) { return HEADS == 1 ? a.kv_heads : (a.kv_heads + HEADS - 1) / HEADS; }
};
constexpr int kNone = -(1 << 30);  // below every relative position
constexpr int kWholeKeys = 256; // longest caches whose items are never split

struct Part {  // an item that a CTA began and others go on with
  int token0;  // packed index of its first row's request
  int row0, rows;  // rows of the tile that exist
  int kv_head;
  int last;        // CTA that ends it; -1: nothing to join
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
template <class B>
__device__ __forceinline__ int blocks_of(const Request& q, int window) {
  const int lo = first_key(q, window) / B::KEYS, hi = (q.total + B::KEYS - 1) / B::KEYS;
  return max(hi - lo, 1);  // one at least: it writes the zeros of rows without keys
}
// Row tiles times head groups, each an item of blocks_of() blocks.
template <class B>
__device__ __forceinline__ int64_t items_of(const Request& q, const AttentionArgs& a) {
  return (int64_t)((q.news * a.group + B::ROWS - 1) / B::ROWS) * B::groups(a);
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

struct RunScratch {
  int64_t scratch[kDecodeWarps], sums[kDecodeWarps][2];
  int64_t found[2];  // request of the CTA's next unit, units before it
};

// A CTA's run of units.
struct Run {
  int64_t begin, end;
  int64_t units, ctas;  // of all requests; CTAs that have any
  int64_t start;        // units before request r
  int r, cut;
  bool pieces;          // a CTA has one unit
};

// This CTA's run; false where it has none. parts[cta] is marked as nothing to join.
template <class B>
__device__ __forceinline__ bool find_run(const AttentionArgs& a, RunScratch& shared, Part* parts, Run& run) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int batch = requests_of(a.pages);
  const int64_t cta = blockIdx.x;
  // This CTA's run of units.
  int64_t total[2] = {0, 0}, my_items = 0;  // blocks and items of all requests; items of this thread's last one
  int my_blocks = 0;
  bool bad = false;
  for (int r = threadIdx.x; r < batch; r += kDecodeThreads) {
    bool b;
    const Request q = request_at(a.pages, a.tokens, a.max_keys, r, &b);
    bad |= b;
    my_items = items_of<B>(q, a);
    my_blocks = blocks_of<B>(q, a.window);
    total[0] += my_items * my_blocks;
    total[1] += my_items;
  }
  if (bad) atomicOr(&g_device_error, kDeviceErrorIndex);
  if (threadIdx.x == 0) shared.found[0] = -1;
  cta_sum(total, shared.sums);
  const int cut = cut_of(a, total[0], total[1]);
  const bool pieces = cut > 1 && !a.whole;  // a CTA has one unit
  const int64_t units = a.whole ? total[1] : total[0];  // where CTAs have runs of them
  if (threadIdx.x == 0 && !a.whole) parts[cta].last = -1;
  const int64_t ctas = min((int64_t)gridDim.x, units);  // every one of these has a unit at least
  if (cta >= ctas) return false;
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
        n = items_of<B>(q, a) * units_of_item(blocks_of<B>(q, a.window), cut);
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
    if (lane == 31) shared.scratch[warp] = upto;
    __syncthreads();
    int64_t start = before + upto - n, all = 0;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
      if (w < warp) start += shared.scratch[w];
      all += shared.scratch[w];
    }
    if (begin >= start && begin < start + n) {
      shared.found[0] = r;
      shared.found[1] = start;
    }
    before += all;
    if (before > begin) break;  // the same for every thread
  }
  __syncthreads();
  if (shared.found[0] < 0) return false;  // fewer pieces than CTAs
  run.begin = begin;
  run.end = end;
  run.units = units;
  run.ctas = ctas;
  run.start = shared.found[1];
  run.r = (int)shared.found[0];
  run.cut = cut;
  run.pieces = pieces;
  return true;
}

// What a unit belongs to, and the CTA's blocks of it.
struct Item {
  Request q;
  int r;
  bool too_long;        // more tokens than the page table has room for
  int per_item, u1;     // units of the item, the end of this CTA's
  int64_t item_start;   // units before the item
  int blocks, b0, b1;   // blocks of the item, this CTA's
  int head;             // first key head
  int row0, rows;       // of the request's news * group rows
  int base;             // position of new token 0
  int key0, lo, hi;     // first key of block 0; keys that a row of this tile sees
};

template <class B>
__device__ __forceinline__ void find_item(const AttentionArgs& a, Run& run, int64_t unit, Item& it) {
  bool too_long;
  int r = run.r;
  int64_t start = run.start;
  const int cut = run.cut;
  const int64_t end = run.end;
  Request q = request_at(a.pages, a.tokens, a.max_keys, r, &too_long);
  int64_t in_request = items_of<B>(q, a) * units_of_item(blocks_of<B>(q, a.window), cut);
  while (unit >= start + in_request) {
    start += in_request;
    ++r;
    q = request_at(a.pages, a.tokens, a.max_keys, r, &too_long);
    in_request = items_of<B>(q, a) * units_of_item(blocks_of<B>(q, a.window), cut);
  }
  const int blocks = blocks_of<B>(q, a.window), per_item = units_of_item(blocks, cut);
  const int size = cut == 1 ? 1 : (blocks + per_item - 1) / per_item;  // blocks of a unit, evenly
  const int64_t in = unit - start;
  const int item = in >> 31 ? (int)(in / per_item) : (int)in / per_item;  // tiles x heads stay below 2^31
  const int64_t item_start = start + (int64_t)item * per_item;
  const int u0 = (int)(unit - item_start), u1 = (int)min((int64_t)per_item, end - item_start);
  const int b0 = u0 * size, b1 = min(u1 * size, blocks);
  const int groups = B::groups(a), head = item % groups * B::HEADS;
  const int row0 = item / groups * B::ROWS;         // of the request's news * group rows
  const int rows = min(B::ROWS, q.news * a.group - row0);
  const int base = q.total - q.news;                // position of new token 0
  const int key0 = first_key(q, a.window) / B::KEYS * B::KEYS;
  // Keys that a row of this tile sees.
  const int hi = base + (row0 + rows - 1) / a.group + 1;
  const int lo = a.window ? max(base + row0 / a.group - a.window + 1, 0) : 0;
  run.r = r;
  run.start = start;
  it.q = q;
  it.r = r;
  it.too_long = too_long;
  it.per_item = per_item;
  it.u1 = u1;
  it.item_start = item_start;
  it.blocks = blocks;
  it.b0 = b0;
  it.b1 = b1;
  it.head = head;
  it.row0 = row0;
  it.rows = rows;
  it.base = base;
  it.key0 = key0;
  it.lo = lo;
  it.hi = hi;
}

// What the join needs of an item that the calling CTA has begun and others go on with.
__device__ __forceinline__ Part part_of(const Run& run, const Item& it) {
  Part p;
  p.token0 = it.q.first;
  p.row0 = it.row0;
  p.rows = it.rows;
  p.kv_head = it.head;
  p.last = (int)(run.pieces ? it.item_start + it.per_item - 1 : ((it.item_start + it.per_item) * run.ctas - 1) / run.units);
  return p;
}

// Joins the parts of one row (and head) of an item that CTAs of the first kernel share: each of TEAM warps
// takes every TEAM-th part, its columns over the lanes; a CTA has WARPS / TEAM rows. Which item: the one that CTA blockIdx.x
// of the first kernel began, or (PICK) the blockIdx.x-th of those that any CTA began, with a grid as large as the
// items there can be.
constexpr int kJoinWarps = 8;
template <typename T, int D, int ROWS, bool SHIFTED, int HEADS = 1, int WARPS = kJoinWarps, int FLIGHT = 4, bool PICK = false,
          int TEAM = WARPS>
__global__ void __launch_bounds__(WARPS * 32) paged_join_kernel(const AttentionArgs a, int64_t ctas) {
  constexpr int kCols = D / 32;  // columns of a lane
  const float* part_out = static_cast<const float*>(a.workspace);
  const float* part_stat = part_out + 2 * ctas * HEADS * ROWS * D;
  wait_for_previous_kernel();
  const Part* all_parts = reinterpret_cast<const Part*>(part_stat + 2 * ctas * HEADS * ROWS * 2);
  static_assert(TEAM == WARPS || TEAM == 1, "rows of a CTA");
  const int head = HEADS == 1 ? 0 : blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = TEAM == 1 ? blockIdx.y * WARPS + warp : blockIdx.y, mate = TEAM == 1 ? 0 : warp;
  int first = blockIdx.x;
  if constexpr (PICK) {
    constexpr int kRounds = 16 / WARPS;  // loads in flight
    __shared__ int counts[kRounds * WARPS], found;
    int before = 0;
    for (int c0 = 0; c0 < ctas; c0 += kRounds * WARPS * 32) {
      int last[kRounds];
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const int c = c0 + (r * WARPS + warp) * 32 + lane;
        last[r] = c < ctas ? all_parts[c].last : -1;
      }
      unsigned begun[kRounds];
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        begun[r] = __ballot_sync(0xffffffffu, last[r] >= 0);
        if (lane == 0) counts[r * WARPS + warp] = __popc(begun[r]);
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        int at = before + __popc(begun[r] & ((1u << lane) - 1u));
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          if (w < warp) at += counts[r * WARPS + w];
          before += counts[r * WARPS + w];
        }
        if (begun[r] >> lane & 1 && at == (int)blockIdx.x) found = c0 + (r * WARPS + warp) * 32 + lane;
      }
      __syncthreads();
    }
    if (before <= (int)blockIdx.x) return;
    first = found;
  }
  const Part p = all_parts[first];
  if (p.last < 0 || row >= p.rows || (HEADS > 1 && p.kv_head + head >= a.kv_heads)) return;
  const int parts = p.last - first + 1;
  float top = -INFINITY, sum = 0.f, o[kCols] = {};
  for (int i0 = mate; i0 < parts; i0 += TEAM * FLIGHT) {
    float2 st[FLIGHT];
    float x[FLIGHT][kCols];
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      const int i = i0 + f * TEAM;
      st[f] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int c = 0; c < kCols; ++c) x[f][c] = 0.f;
      if (i < parts) {
        // Part i is in the second slot of the CTA that began the item, in the first slot of the others.
        const int64_t at = ((2 * (int64_t)(first + i) + (i == 0)) * HEADS + head) * ROWS + row;
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
    for (int f = 0; f < FLIGHT; ++f) now = fmaxf(now, st[f].x);
    const float from = now == -INFINITY ? 0.f : now, moved = exp2_approx(top - from);
    top = now;
    sum *= moved;
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c] *= moved;
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      const float e = exp2_approx(st[f].x - from);
      sum += e * st[f].y;
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[c] += e * x[f][c];
    }
  }
  const int at = p.row0 + row, token = at / a.group;
  const int h = (p.kv_head + head) * a.group + (at - token * a.group);
  T* out = static_cast<T*>(a.out) + (p.token0 + token) * a.out_n + h * a.out_h;
  const auto put_lse = [&](float m, float l) {
    if (a.lse) a.lse[(int64_t)(p.token0 + token) * a.heads + h] = (m + log2f(l) - (SHIFTED ? kProbabilityShift<T> : 0.f)) * 0.6931471805599453f;
  };
  if constexpr (TEAM == 1) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) out[lane * kCols + c] = from_float<T>(sum == 0.f ? 0.f : o[c] / sum);
    if (lane == 0) put_lse(top, sum);
  } else {
    __shared__ float joined[WARPS][D], sums[WARPS], tops[WARPS];
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
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, tops[w]);
    const float from = m == -INFINITY ? 0.f : m;
    float v = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float e = exp2_approx(tops[w] - from);
      v += e * joined[w][col];
      l += e * sums[w];
    }
    out[col] = from_float<T>(l == 0.f ? 0.f : v / l);
    if (col == 0) put_lse(m, l);
  }
}

}  // namespace
}  // namespace flash_prologue
