// Attention of chunks of new tokens over a paged cache on the tensor cores
// (tcgen05): o_i = sum_j p_ij v_j with p the softmax of the scaled scores over
// the keys that row i sees (causal, optional window).
//
// Bound by the tensor cores and, as much, by the exponentials: 128 rows x 128
// keys cost 4 * 128 * 128 * D operations (1,024 cycles of an SM's tensor core
// at D = 128) and 128 * 128 exponentials (1,024 cycles of its 16 a cycle). So
// neither may wait for the other. Keys come in blocks of 64: a block's scores
// (64 columns of tensor memory) are free as soon as the rows have them in
// registers, so the next block's scores are computed beside this one's softmax,
// and the probabilities have two buffers, so the product with V runs beside the
// next softmax. With the output that is 256 columns of the 512, so two CTAs share
// an SM and two warps a scheduler do softmax. Ragged chunks of up to 2,000 tokens
// with a window of 1,024 keys, 16/4 heads x 64 FP16: 81 us; probabilities over
// the scores they came from, with two buffers for both: 83 us; one such buffer
// of 128 keys: 101 us.
//
// A CTA takes one tile: the rows (query heads x whole tokens) of one key head
// that fit into 128, and its blocks of keys (or a share of them where there
// are fewer tiles than the GPU holds; a second kernel adds the shares up).
//   warps 0-3  one row a thread: scores from tensor memory, running maximum
//              and sum, probabilities to tensor memory, output to global memory;
//   warp 4     issues S = Q K^T (both from shared memory);
//   warp 6     issues O += P V (P from tensor memory, V read transposed from
//              shared memory);
//   warp 5     TMA loads of K and V, one box of a page a lane;
//   warp 7     cleans V in blocks that some row of the tile does not see whole:
//              zeros for slots outside the tile's keys, and for infinities and
//              NaNs, which 0 * V would carry into rows that do not see them
//              (the epilogue adds them to the rows that do).
// The running maximum that scales O is only moved when a row's maximum has
// grown by more than 2^8: until then the probabilities are at most 2^8 instead
// of 1, which neither type nor sum minds, and O stays where it is.
//
// Scores, statistics, sums and O are FP32; the probabilities are rounded to the
// cache's type for the second product (their sum is taken before the rounding),
// an error of the size of the output's own rounding. Waits are bounded; tensor
// memory is released on every path.
#include "paged_attention.h"
#include "tensor_map.h"
#include "umma_util.cuh"

namespace flash_prologue {
namespace {

constexpr int kTile = 128;             // rows of a tile
constexpr int kKeys = 64;              // keys of a block
constexpr int kPrefillThreads = 256;
constexpr int kRowThreads = 128;
constexpr int kTmemCols = 256;

template <int D>
struct Layout {
  static constexpr int kHalves = D / 64;           // 64-column (128-byte) halves of a row
  static constexpr int kStages = D == 64 ? 4 : 2;  // K and V blocks in flight
  static constexpr int kQ = kTile * D * 2, kQHalf = kTile * 128;      // bytes of the Q tile, of its halves
  static constexpr int kBlock = kKeys * D * 2, kHalf = kKeys * 128;   // of a K or V block
  // Tensor-memory columns: blocks of scores (two where there is room), two of probabilities, the output.
  static constexpr int kScores = D == 64 ? 2 : 1;
  static constexpr int kSCol = 0, kPCol = kScores * kKeys, kOCol = kPCol + kKeys;
  static_assert(kOCol + D <= kTmemCols, "tensor memory");
  static constexpr size_t kSmem = 1024 + (size_t)kQ + (size_t)kBlock * 2 * kStages;
};

constexpr int kMaxStages = 4;
struct Barriers {
  uint64_t k_full[kMaxStages], k_empty[kMaxStages], v_full[kMaxStages], v_empty[kMaxStages];
  uint64_t s_full[2], s_read[2], p_full[2], o_done[2], clean_ask, v_clean, drain[2];
  uint32_t tmem;
  int bad, wild;
  int sums[kPrefillThreads / 32];
  int found, found_tile;  // request of the CTA's tile (-1: none), its tile of it
  Request request;
};

struct Tile {  // what the join needs to know of a tile
  int token0, rows, kv_head, parts;
};

struct PrefillArgs {
  AttentionArgs a;
  int tile_tokens;       // whole tokens of a tile: 128 / group
  int splits;            // shares that the blocks of the last items may be cut into
  int whole_items;       // items (tile, key head) before those
  int box_rows;          // keys of a TMA box: page_size, at most 64
  int tiles;             // tiles the grid has room for, all requests
  float* part_out;       // [cut items * splits][128][D]
  float* part_stat;      // [...][128][2]
  Tile* joins;           // [cut items]
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
// mbar_wait without the suspend hint, whose try takes twice as long where the
// phase is complete (102 cycles instead of 51) and wakes later where it is not
// (a round trip of two warps: 434 cycles instead of 289); bounded by the clock.
__device__ __forceinline__ bool phase_done(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
__device__ __forceinline__ bool phase_wait(uint64_t* bar, uint32_t parity) {
  constexpr long long kMostCycles = 8000000000ll;  // about 4 s
  const uint32_t a = smem_u32(bar);
  if (phase_done(a, parity)) return true;
  const long long start = clock64();
  do {
    if (phase_done(a, parity)) return true;
  } while (clock64() - start < kMostCycles);
  atomicOr(&g_device_error, kDeviceErrorTimeout);
  return false;
}
// One lane of the (whole) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// D[tmem] (+)= A[tmem] * B[smem], issued by one thread.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
        "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
        "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Names registers behind a tcgen05.wait::ld, so that no use of them moves above it.
template <int N>
__device__ __forceinline__ void pin(uint32_t (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("" : "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]),
                      "+r"(v[i + 6]), "+r"(v[i + 7]));
}
// kind::f16 with A and B of one 16-bit type (format 1: BF16, 0: FP16), FP32 accumulator.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_of(int N, bool b_mn) {
  constexpr uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(kTile >> 4) << 24);
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
template <typename T>
constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;

// The keys of a tile and the split's share of its blocks.
struct Work {
  Request q;
  int r;
  int head;
  int token0;       // first token of the tile, of the request's new ones
  int rows;         // valid rows
  int pos0, pos1;   // positions of the first and last token
  int lo, hi;       // keys that some row sees
  int first, last;  // this split's blocks (of 64 keys)
  int parts;        // splits that have blocks
};

__device__ __forceinline__ bool partial_block(const Work& w, int window, int block) {
  const int kb = block * kKeys;
  return kb + kKeys - 1 > w.pos0 || (window && kb < w.pos1 - window + 1);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPrefillThreads, 2)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                         const __grid_constant__ PrefillArgs p) {
  using L = Layout<D>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Barriers bar;
  const AttentionArgs& a = p.a;
  unsigned char* q_s = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* k_s = q_s + L::kQ;
  unsigned char* v_s = k_s + L::kStages * L::kBlock;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (p.splits > 1) start_next_kernel();
  // ---- this CTA's tile: last tiles first (they have the most keys), splits innermost
  const int cut = (int)blockIdx.x - p.whole_items;  // CTAs of the items that are cut
  const int splits = cut < 0 ? 1 : p.splits;
  const int item = cut < 0 ? (int)blockIdx.x : p.whole_items + cut / p.splits;
  const int split = cut < 0 ? 0 : cut % p.splits;
  const int tile_of_all = p.tiles - 1 - item / a.kv_heads;
  const int requests = a.pages.batch + (a.pages.cu_seqlens ? 1 : 0);
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&bar.k_full[s], 1);
      mbar_init(&bar.k_empty[s], 1);
      mbar_init(&bar.v_full[s], 1);
      mbar_init(&bar.v_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bar.s_full[b], 1);
      mbar_init(&bar.s_read[b], kRowThreads / 32);
      mbar_init(&bar.p_full[b], kRowThreads / 32);
      mbar_init(&bar.o_done[b], 1);
    }
    mbar_init(&bar.clean_ask, 1);
    mbar_init(&bar.v_clean, 1);
    mbar_init(&bar.drain[0], 1);
    mbar_init(&bar.drain[1], 1);
    bar.found = -1;
    bar.bad = 0;
    bar.wild = 0;
    fence_mbar_init();
  }
  int before = 0;
  for (int r0 = 0; r0 < requests; r0 += kPrefillThreads) {
    const int r = r0 + threadIdx.x;
    Request q{0, 0, 0};
    bool too_long = false;
    if (r < requests) q = request_at(a.pages, a.tokens, a.max_keys, r, &too_long);
    const int n = (q.news + p.tile_tokens - 1) / p.tile_tokens;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) bar.sums[warp] = upto;
    __syncthreads();
    int start = before + upto - n, all = 0;
#pragma unroll
    for (int w = 0; w < kPrefillThreads / 32; ++w) {
      if (w < warp) start += bar.sums[w];
      all += bar.sums[w];
    }
    if (tile_of_all >= start && tile_of_all < start + n) {
      bar.found = r;
      bar.found_tile = tile_of_all - start;
      bar.request = q;
      bar.bad = too_long;
    }
    before += all;
    __syncthreads();
    if (before > tile_of_all) break;
  }
  Tile* join = splits > 1 ? p.joins + (item - p.whole_items) : nullptr;
  if (bar.found < 0) {  // the grid has room for more tiles than there are
    if (join && split == 0 && threadIdx.x == 0) join->parts = 0;
    return;
  }
  Work w;
  w.r = bar.found;
  w.head = item % a.kv_heads;
  w.q = bar.request;
  w.token0 = bar.found_tile * p.tile_tokens;
  const int tokens = min(p.tile_tokens, w.q.news - w.token0);
  w.rows = tokens * a.group;
  w.pos0 = w.q.total - w.q.news + w.token0;
  w.pos1 = w.pos0 + tokens - 1;
  w.hi = max(w.pos1 + 1, 0);
  w.lo = a.window ? max(w.pos0 - a.window + 1, 0) : 0;
  {
    const int first = w.lo / kKeys, blocks = max((w.hi + kKeys - 1) / kKeys - first, 0);
    // Shares of at least four blocks: a share's fixed cost is about theirs.
    int share = blocks;
    if (splits > 1) share = max((blocks + splits - 1) / splits, 4);
    w.parts = blocks && splits > 1 ? (blocks + share - 1) / share : 1;
    w.first = first + split * share;
    w.last = min(first + blocks, w.first + share);
  }
  if (join && split == 0 && threadIdx.x == 0) {
    join->token0 = w.q.first + w.token0;
    join->rows = w.rows;
    join->kv_head = w.head;
    join->parts = w.parts;
  }
  if (split >= w.parts) return;
  const int blocks = max(w.last - w.first, 0);

  // ---- tensor memory, Q
  if (warp == 4) {
    tmem_alloc(&bar.tmem, kTmemCols);
    tmem_relinquish();
  }
  // The loads begin before the other warps have Q in shared memory.
  const int boxes = kKeys / p.box_rows, in_page = (1 << a.pages.page_log2) - 1;
  const uint32_t box_bytes = (uint32_t)p.box_rows * 128;
  // The page of this lane's box of a block, -1 where there is nothing to load.
  const auto page_of = [&](int j) {
    int page = -1;
    if (lane < boxes && j < blocks) {
      const int key = (w.first + j) * kKeys + lane * p.box_rows;
      if (key < w.hi && key + p.box_rows > w.lo) {
        page = __ldg(a.pages.page_table + w.r * a.pages.table_stride + (key >> a.pages.page_log2));
        if (page < 0 || page >= a.pages.num_pages) {
          page = -1;
          bar.bad = 1;
        }
      }
    }
    return page;
  };
  const auto load = [&](int j, int page, const CUtensorMap* map, unsigned char* ring, uint64_t* full) {
    const int s = j % L::kStages;
    const uint32_t count = __popc(__ballot_sync(0xffffffffu, page >= 0));
    if (lane == 0) mbar_arrive_expect_tx(&full[s], count * box_bytes * L::kHalves);
    __syncwarp();
    if (page >= 0) {
      const int key = (w.first + j) * kKeys + lane * p.box_rows;
      const uint32_t dst = smem_u32(ring) + s * L::kBlock + lane * box_bytes;
#pragma unroll
      for (int h = 0; h < L::kHalves; ++h)
        tma_load_4d(dst + h * L::kHalf, map, h * 64, key & in_page, w.head, page, &full[s]);
    }
    __syncwarp();
  };
  int next_page = -1;  // of the first block that the loop below loads
  if (warp == 5) {
    int page[L::kStages];
#pragma unroll
    for (int j = 0; j < L::kStages; ++j) page[j] = page_of(j);
    next_page = page_of(L::kStages);
#pragma unroll
    for (int j = 0; j < L::kStages; ++j)
      if (j < blocks) {
        load(j, page[j], &k_map, k_s, bar.k_full);
        load(j, page[j], &v_map, v_s, bar.v_full);
      }
  }
  for (int i = threadIdx.x; i < kTile * (D / 8); i += kPrefillThreads) {
    const int row = i / (D / 8), c = i % (D / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < w.rows) {
      const int t = row / a.group, g = row - t * a.group;
      v = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (w.q.first + w.token0 + t) * a.q_n +
                                               (w.head * a.group + g) * a.q_h + c * 8));
    }
    *reinterpret_cast<uint4*>(q_s + (c >> 3) * L::kQHalf + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v;
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem;

  // Row state (warps 0-3); the row's keys are [see_lo, see_hi].
  const int row = threadIdx.x;
  int see_hi = -1, see_lo = 0;
  float top = -INFINITY, sum = 0.f;

  if (warp >= 4) {
    // The issuing warps walk the blocks whole, with values the compiler knows to be the same
    // in all lanes, and one lane issues. Each has one product: a warp that issued both, with
    // its waits, took longer for a block than its softmax does.
    const int n = __shfl_sync(0xffffffffu, blocks, 0);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    if (warp == 4) {
      // ---------------- scores ----------------
      constexpr uint32_t idesc = idesc_of<T>(kKeys, false);
      const uint64_t q_desc = smem_desc_k_sw128(smem_u32(q_s));
      bool failed = false;
      for (int j = 0; j < n; ++j) {
        const int s = j % L::kStages, b = j % L::kScores, before = j - L::kScores;
        // The last scores of this buffer are in the rows' registers, K is here.
        if (!__all_sync(0xffffffffu, (before < 0 || phase_wait(&bar.s_read[b], (before / L::kScores) & 1)) &&
                                         phase_wait(&bar.k_full[s], (j / L::kStages) & 1))) {
          failed = true;
          break;
        }
        tc_fence_after();
        const uint64_t k_desc = smem_desc_k_sw128(smem_u32(k_s) + s * L::kBlock);
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < L::kHalves; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c)  // 16 columns (32 bytes) a step
              umma_bf16(tm + L::kSCol + b * kKeys, q_desc + h * (L::kQHalf / 16) + 2 * c,
                        k_desc + h * (L::kHalf / 16) + 2 * c, idesc, (h | c) != 0);
          umma_commit(&bar.k_empty[s]);
          umma_commit(&bar.s_full[b]);
        }
        __syncwarp();
      }
      if (failed) {  // tensor memory is not released under products still running
        if (elect_one()) umma_commit(&bar.drain[0]);
        phase_wait(&bar.drain[0], 0);
      }
    } else if (warp == 6) {
      // ---------------- output ----------------
      constexpr uint32_t idesc = idesc_of<T>(D, true);
      bool failed = false;
      uint32_t cleaned = 0;
      for (int j = 0; j < n; ++j) {
        const int s = j % L::kStages;
        bool ok = phase_wait(&bar.v_full[s], (j / L::kStages) & 1);
        const bool partial = partial_block(w, a.window, w.first + j);
        if (partial && lane == 0) mbar_arrive(&bar.clean_ask);  // cleaned beside the block's softmax
        ok = ok && (!partial || phase_wait(&bar.v_clean, cleaned & 1)) && phase_wait(&bar.p_full[j & 1], (j >> 1) & 1);
        cleaned += partial;
        if (!__all_sync(0xffffffffu, ok)) {
          failed = true;
          break;
        }
        tc_fence_after();
        const uint64_t v_desc = smem_desc_mn_sw128(smem_u32(v_s) + s * L::kBlock, L::kHalf);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < kKeys / 16; ++c)  // 16 keys a step: 8 columns of P, two 8-row groups of V (2,048 bytes)
            umma_ts(tm + L::kOCol, tm + L::kPCol + (j & 1) * (kKeys / 2) + 8 * c, v_desc + 128 * c, idesc, (j | c) != 0);
          umma_commit(&bar.v_empty[s]);
          umma_commit(&bar.o_done[j & 1]);
        }
        __syncwarp();
      }
      if (failed) {
        if (elect_one()) umma_commit(&bar.drain[1]);
        phase_wait(&bar.drain[1], 0);
      }
    } else if (warp == 5) {
      // ---------------- loads ----------------
      bool ok = true;
      int j = L::kStages;
      for (int page = next_page; j < blocks; ++j) {
        const int s = j % L::kStages, next = page_of(j + 1);
        const uint32_t parity = ((j / L::kStages) & 1) ^ 1;
        if (!(ok = __all_sync(0xffffffffu, phase_wait(&bar.k_empty[s], parity)))) break;
        load(j, page, &k_map, k_s, bar.k_full);
        if (!(ok = __all_sync(0xffffffffu, phase_wait(&bar.v_empty[s], parity)))) break;
        load(j, page, &v_map, v_s, bar.v_full);
        page = next;
      }
      // No product's arrival on an empty barrier lands after the CTA has gone.
      for (int e = blocks; e < blocks + L::kStages && blocks && ok; ++e) {
        const int s = e % L::kStages;
        ok = phase_wait(&bar.k_empty[s], ((e / L::kStages) & 1) ^ 1) && phase_wait(&bar.v_empty[s], ((e / L::kStages) & 1) ^ 1);
      }
      if (j < blocks) {  // a wait ran out: wait (bounded) for the loads still in flight
        for (int s = 0; s < L::kStages; ++s) {
          for (int e = j; e >= 0 && e > j - L::kStages - 1; --e)
            if (e % L::kStages == s) {
              phase_wait(&bar.k_full[s], (e / L::kStages) & 1);
              phase_wait(&bar.v_full[s], (e / L::kStages) & 1);
              break;
            }
        }
      }
    } else {
      // ---------------- cleaning ----------------
      uint32_t asked = 0;
      for (int j = 0; j < blocks; ++j) {
        if (!partial_block(w, a.window, w.first + j)) continue;
        const int s = j % L::kStages;
        // Asked by the warp that has seen the block arrive.
        if (!__all_sync(0xffffffffu, phase_wait(&bar.clean_ask, asked++ & 1) &&
                                         phase_wait(&bar.v_full[s], (j / L::kStages) & 1)))
          break;
        const int kb = (w.first + j) * kKeys;
        uint4* v = reinterpret_cast<uint4*>(v_s + s * L::kBlock);
        bool wild = false;
#pragma unroll 4
        for (int i = lane; i < kKeys * D / 8; i += 32) {
          const int key = kb + ((i >> 3) & (kKeys - 1));
          uint4 x = v[i];
          if (key < w.lo || key >= w.hi) {
            v[i] = make_uint4(0, 0, 0, 0);
            continue;
          }
          uint32_t* word = reinterpret_cast<uint32_t*>(&x);
          bool changed = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            constexpr uint32_t m = kExponent<T>;
            if ((word[e] & m) == m) { word[e] &= 0xffff0000u; changed = true; }
            if ((word[e] >> 16 & m) == m) { word[e] &= 0x0000ffffu; changed = true; }
          }
          if (changed) {
            v[i] = x;
            wild = true;
          }
        }
        if (wild) bar.wild = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.v_clean);
      }
    }
  } else {
    // ---------------- softmax ----------------
    if (row < w.rows) {
      see_hi = w.pos0 + row / a.group;
      if (a.window && see_hi - a.window + 1 > 0) see_lo = see_hi - a.window + 1;
    }
    const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
    const float scale = a.scale_log2;
    bool ok = true;
    for (int j = 0; j < blocks; ++j) {
      if (!(ok = __all_sync(0xffffffffu, phase_wait(&bar.s_full[j % L::kScores], (j / L::kScores) & 1)))) break;
      tc_fence_after();
      uint32_t s[2][32];
      tmem_ld32(mine + L::kSCol + j % L::kScores * kKeys, s[0]);
      tmem_ld32(mine + L::kSCol + j % L::kScores * kKeys + 32, s[1]);
      tmem_wait_ld();
      pin(s[0]);
      pin(s[1]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.s_read[j % L::kScores]);
      const int block = w.first + j;
      if (partial_block(w, a.window, block)) {
        const int hi = see_hi - block * kKeys, lo = see_lo - block * kKeys;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (32 * c + i > hi || 32 * c + i < lo) s[c][i] = 0xff800000u;  // -infinity
      }
      float most[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) most[i] = __uint_as_float(s[0][i]);
#pragma unroll
      for (int i = 8; i < kKeys; i += 8)
#pragma unroll
        for (int e = 0; e < 8; ++e) most[e] = fmaxf(most[e], __uint_as_float(s[(i + e) >> 5][(i + e) & 31]));
      const float block_top = fmaxf(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])),
                                    fmaxf(fmaxf(most[4], most[5]), fmaxf(most[6], most[7])));
      const float now = fmaxf(top, block_top);
      const bool fresh = top == -INFINITY;  // nothing summed yet, O is zero
      if (fresh) top = now;
      const bool move = !fresh && (now - top) * scale > 8.f;
      if (__any_sync(0xffffffffu, move)) {
        // O has to be at rest: the last product with V done; the next one waits for this block's P.
        if (!(ok = __all_sync(0xffffffffu, phase_wait(&bar.o_done[(j - 1) & 1], ((j - 1) >> 1) & 1)))) break;
        tc_fence_after();
        const float f = move ? exp2_approx((top - now) * scale) : 1.f;
        sum *= f;
        if (move) top = now;
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld16(mine + L::kOCol + 16 * c, o);
          tmem_wait_ld();
          pin(o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
          tmem_st16(mine + L::kOCol + 16 * c, o);
        }
      }
      const float from = (top == -INFINITY ? 0.f : top * scale) - kProbabilityShift<T>;
      const float2 scale2 = make_float2(scale, scale), from2 = make_float2(-from, -from);
      float2 add[4] = {};
      uint32_t out[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int c = i >> 4, e = (i & 15) * 2;
        float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])), scale2, from2);
        x.x = exp2_approx(x.x);
        x.y = exp2_approx(x.y);
        add[i & 3] = __fadd2_rn(add[i & 3], x);
        out[i] = pack2<T>(x.x, x.y);
      }
      // The buffer's last P has to be used up.
      if (j >= 2 && !(ok = __all_sync(0xffffffffu, phase_wait(&bar.o_done[j & 1], ((j - 2) >> 1) & 1)))) break;
      tc_fence_after();
      tmem_st32(mine + L::kPCol + (j & 1) * (kKeys / 2), out);
      const float2 both = __fadd2_rn(__fadd2_rn(add[0], add[1]), __fadd2_rn(add[2], add[3]));
      sum += both.x + both.y;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.p_full[j & 1]);
    }
    if (blocks && ok) ok = phase_wait(&bar.o_done[(blocks - 1) & 1], ((blocks - 1) >> 1) & 1);
    if (!ok) sum = __int_as_float(0x7fc00000);  // a wait ran out: no output that could pass for one
  }
  __syncthreads();  // `bad` and `wild` are final

  // ---- output
  if (warp < 4) {
    tc_fence_after();
    const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
    const bool bad = bar.bad, wild = bar.wild, whole = w.parts == 1;
    const float nan = __int_as_float(0x7fc00000);
    if (bad) sum = nan;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int t = row / a.group, g = row - t * a.group;
    const int token = w.q.first + w.token0 + t;
    const int h = w.head * a.group + g;
    const bool valid = row < w.rows;
    const int64_t slot = cut;  // of the cut items' shares
    const float top2 = top == -INFINITY ? top : top * a.scale_log2;
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32];
      __syncwarp();
      if (blocks) {
        tmem_ld32(mine + L::kOCol + 32 * c, o);
        tmem_wait_ld();
        pin(o);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0;
      }
      if (wild && valid) {
        // The infinities and NaNs taken out of V, added to a row that sees them.
        for (int j = 0; j < blocks; ++j) {
          if (!partial_block(w, a.window, w.first + j)) continue;
          const int kb = (w.first + j) * kKeys;
          for (int k = max(kb, see_lo); k <= min(kb + kKeys - 1, see_hi); ++k) {
            const int32_t* entry = a.pages.page_table + (int64_t)w.r * a.pages.table_stride + (k >> a.pages.page_log2);
            const int64_t page = __ldg(entry);
            if (page < 0 || page >= a.pages.num_pages) continue;
            const T* v = static_cast<const T*>(a.v) + page * a.v_page +
                         (k & ((1 << a.pages.page_log2) - 1)) * a.v_slot + w.head * a.v_head + 32 * c;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float x = (float)v[i];
              if (!isfinite(x)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
            }
          }
        }
      }
      if (!valid) continue;
      if (whole) {
        uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(a.out) + token * a.out_n + (int64_t)h * a.out_h + 32 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] = pack2<T>(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
          out[i] = make_uint4(x[0], x[1], x[2], x[3]);
        }
      } else {
        float4* out = reinterpret_cast<float4*>(p.part_out + (slot * kTile + row) * D + 32 * c);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          out[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                               __uint_as_float(o[4 * i + 3]));
      }
    }
    if (valid) {
      if (!whole) {
        p.part_stat[(slot * kTile + row) * 2] = top2;
        p.part_stat[(slot * kTile + row) * 2 + 1] = sum;
      } else if (a.lse) {
        a.lse[(int64_t)token * a.heads + h] = (top2 + log2f(sum) - kProbabilityShift<T>) * 0.6931471805599453f;
      }
    }
  }
  if (threadIdx.x == 0 && bar.bad) atomicOr(&g_device_error, kDeviceErrorIndex);
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Adds up the shares of a tile, a row a warp: 16 rows a CTA.
template <typename T, int D>
__global__ void __launch_bounds__(512) prefill_join_kernel(const PrefillArgs p) {
  const AttentionArgs& a = p.a;
  const int64_t item = blockIdx.x / (kTile / 16);  // of those that were cut
  wait_for_previous_kernel();
  const Tile t = p.joins[item];
  const int row = (int)(blockIdx.x % (kTile / 16)) * 16 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t.parts <= 1 || row >= t.rows) return;
  const int64_t slot0 = item * p.splits;
  float m = -INFINITY;
  for (int s = 0; s < t.parts; ++s) m = fmaxf(m, p.part_stat[((slot0 + s) * kTile + row) * 2]);
  const float from = m == -INFINITY ? 0.f : m;
  float o[D / 32] = {}, l = 0.f;
#pragma unroll 4
  for (int s = 0; s < t.parts; ++s) {
    const int64_t at = (slot0 + s) * kTile + row;
    const float f = exp2_approx(p.part_stat[at * 2] - from);
    l += f * p.part_stat[at * 2 + 1];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] += f * p.part_out[at * D + 32 * c + lane];
  }
  const int token = row / a.group, h = t.kv_head * a.group + row - token * a.group;
  T* out = static_cast<T*>(a.out) + (t.token0 + token) * a.out_n + (int64_t)h * a.out_h;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    const float x = l == 0.f ? 0.f : o[c] / l;
    if constexpr (std::is_same<T, __half>::value) out[32 * c + lane] = __float2half_rn(x);
    else out[32 * c + lane] = __float2bfloat16_rn(x);
  }
  if (a.lse && lane == 0) a.lse[(int64_t)(t.token0 + token) * a.heads + h] = (m + log2f(l) - kProbabilityShift<T>) * 0.6931471805599453f;
}

// A cache as {D, slots, heads, pages}, a box of 64 columns x box_rows slots.
bool encode_cache(CUtensorMap* map, const void* base, int dtype, int D, int64_t page_size, int64_t heads, int64_t pages,
                  int64_t s_slot, int64_t s_head, int64_t s_page, int box_rows) {
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)page_size, (uint64_t)heads, (uint64_t)pages};
  // A dimension of one entry gets a stride that no address depends on.
  const uint64_t strides[3] = {(uint64_t)(2 * s_slot), heads > 1 ? (uint64_t)(2 * s_head) : 128,
                               pages > 1 ? (uint64_t)(2 * s_page) : 128};
  for (uint64_t s : strides)
    if (s == 0 || (int64_t)s < 0) return false;
  const uint32_t box[4] = {64, (uint32_t)box_rows, 1, 1};
  return encode_tensor_map(map, dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base,
                           dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, int D>
cudaError_t launch(const CUtensorMap& k_map, const CUtensorMap& v_map, const PrefillArgs& p, int64_t items,
                   cudaStream_t stream) {
  const void* fn = reinterpret_cast<const void*>(&paged_prefill_kernel<T, D>);
  cudaError_t err = allow_shared_memory(fn, Layout<D>::kSmem);
  if (err != cudaSuccess) return err;
  const int64_t cut = items - p.whole_items;
  err = launch_kernel(paged_prefill_kernel<T, D>, dim3((unsigned)(p.whole_items + cut * p.splits)), dim3(kPrefillThreads),
                      Layout<D>::kSmem, stream, k_map, v_map, p);
  if (err != cudaSuccess || p.splits == 1) return err;
  return launch_following(prefill_join_kernel<T, D>, dim3((unsigned)(cut * (kTile / 16))), dim3(512), stream, p);
}

}  // namespace

// Tiles, and the shares that blocks are cut into. The GPU holds 2 CTAs an SM;
// the items that would leave its last round partly empty (all of them, where
// there are few) are cut so that they fill it. Lengths are only known on the
// device: the bound on the shares is the page table's width. 4,096 tokens over
// 16,384 keys, 32/8 heads x 128 (1,024 items, 3.46 rounds): 1,075 us with whole items, 1,046 us so.
PrefillPlan plan_paged_prefill(int64_t tokens, int64_t batch, bool ragged, int64_t kv_heads, int64_t group, int D,
                               int64_t max_keys, int64_t window, int sms) {
  PrefillPlan p{};
  p.tile_tokens = (int)(kTile / group);
  p.tiles = tokens;
  if (ragged) {
    // Every request (and the padding) may leave its last tile partly empty.
    const int64_t ends = (tokens < batch ? tokens : batch) + 1;
    p.tiles = (tokens + ends * (p.tile_tokens - 1)) / p.tile_tokens;
  }
  const int64_t items = p.tiles * kv_heads, slots = 2 * (int64_t)sms;
  const int64_t cut = items % slots;
  p.whole_items = items - cut;
  p.splits = 1;
  if (cut) {
    const int64_t keys = window && window + p.tile_tokens < max_keys ? window + p.tile_tokens : max_keys;
    const int64_t most = (keys / kKeys + 5) / 4;  // shares of at least four blocks
    const int64_t splits = slots / cut < most ? slots / cut : most;
    if (splits > 1) p.splits = (int)splits;
  }
  if (p.splits == 1) p.whole_items = items;
  return p;
}

// At most one share a CTA that the device holds.
size_t paged_prefill_workspace(int D, int sms) {
  return (size_t)(2 * sms) * (kTile * (size_t)(D + 2) * sizeof(float) + sizeof(Tile));
}

bool launch_paged_prefill(const AttentionArgs& a, const PrefillPlan& plan, int dtype, int D, int64_t page_size,
                          cudaStream_t stream, cudaError_t* err) {
  PrefillArgs p{};
  p.a = a;
  p.tile_tokens = plan.tile_tokens;
  p.splits = plan.splits;
  p.whole_items = (int)plan.whole_items;
  p.tiles = (int)plan.tiles;
  p.box_rows = page_size < kKeys ? (int)page_size : kKeys;
  const int64_t items = plan.tiles * a.kv_heads;
  if (items * plan.splits * (kTile / 16) >= (int64_t(1) << 31)) return false;
  CUtensorMap k_map, v_map;
  if (!encode_cache(&k_map, a.k, dtype, D, page_size, a.kv_heads, a.pages.num_pages, a.k_slot, a.k_head, a.k_page,
                    p.box_rows) ||
      !encode_cache(&v_map, a.v, dtype, D, page_size, a.kv_heads, a.pages.num_pages, a.v_slot, a.v_head, a.v_page,
                    p.box_rows))
    return false;
  if (p.splits > 1) {
    p.part_out = static_cast<float*>(a.workspace);
    const int64_t shares = (items - p.whole_items) * p.splits;
    p.part_stat = p.part_out + shares * kTile * D;
    p.joins = reinterpret_cast<Tile*>(p.part_stat + shares * kTile * 2);
  }
  if (D == 64)
    *err = dtype == 0 ? launch<__nv_bfloat16, 64>(k_map, v_map, p, items, stream)
                      : launch<__half, 64>(k_map, v_map, p, items, stream);
  else
    *err = dtype == 0 ? launch<__nv_bfloat16, 128>(k_map, v_map, p, items, stream)
                      : launch<__half, 128>(k_map, v_map, p, items, stream);
  return true;
}

cudaError_t read_paged_prefill_device_error(int* value, bool reset) {
  cudaError_t err = cudaMemcpyFromSymbol(value, g_device_error, sizeof(int));
  if (err != cudaSuccess || !reset) return err;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
}

}  // namespace flash_prologue
