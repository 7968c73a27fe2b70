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
// with a window of 1,024 keys, 16/4 heads x 64 FP16, a CTA a tile: 81 us;
// probabilities over the scores they came from, with two buffers for both: 83 us;
// one such buffer of 128 keys: 101 us.
//
// A tile is the rows (query heads x whole tokens) of one key head that fit into
// 128, and its blocks of keys (or a share of them where there are fewer tiles
// than the GPU holds; a second kernel adds the shares up). There is a CTA a tile
// in the grid, but one that runs takes over the tiles of those that have not
// started (cluster launch control), so the start of a tile -- finding its
// request, the pages' indices, the first loads and scores -- runs beside the last
// softmax and output of the one before: 2 to 3 us a tile instead of 7 (78 to
// 61 us for the chunks above). All buffers and their phases go on from tile to tile.
//   warps 0-3  one row a thread: scores from tensor memory, running maximum
//              and sum, probabilities to tensor memory, output to global memory;
//   warp 4     issues S = Q K^T (both from shared memory);
//   warp 6     issues O += P V (P from tensor memory, V read transposed from
//              shared memory);
//   warp 5     finds the tiles and loads Q, K and V by TMA, one box of a page a lane;
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
// an error of the size of the output's own rounding. Waits are bounded: where one
// runs out the error word is set, the rows that the CTA was at or had taken over
// are NaN, and it ends once its copies and products are done. (Only a tile whose
// index does not come back within twice the limit stays unwritten.) Tensor memory
// is released on every path.
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

// A tile and the split's share of its blocks.
struct Work {
  int first_token;  // packed index of its first row's token
  int r;
  int head;
  int rows;         // valid rows; -1: no more tiles
  int pos0, pos1;   // positions of the first and last token
  int lo, hi;       // keys that some row sees
  int first, blocks;  // this split's blocks (of 64 keys)
  int full0, full1;   // of them, those that every row sees whole: [full0, full1)
  int parts;        // splits that have blocks
  int share;        // where an item that is cut keeps this share
  int bad, wild;    // an index was out of range; V held infinities or NaNs in partial blocks
};

constexpr int kMaxStages = 4;
struct Barriers {
  uint64_t k_full[kMaxStages], k_empty[kMaxStages], v_full[kMaxStages], v_empty[kMaxStages];
  uint64_t s_full[2], s_read[2], p_full[2], o_done[2], clean_ask, v_clean, drain[2];
  uint64_t q_full, q_empty, work_full[2], work_empty[2], next_here;
  uint32_t tmem;
  int sums[kPrefillThreads / 32];
  int found, found_start;  // request of the CTA's first tile (-1: none), tiles before it
  Work work[2];            // the tile that the warps are at and the next
  // Where a wait ran out: the tiles that were put into work, and one that was taken over and not put there.
  uint32_t posted;
  int has_left;
  Work left;
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
  long long wait_cycles; // self-test: limit of a wait
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}
// Asks for a CTA of the grid that has not started, to do its work here; the
// answer (16 bytes) arrives at `bar`. After an answer without one, not to be called again.
__device__ __forceinline__ void ask_next_cta(void* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
// Its index, -1 if there is none.
__device__ __forceinline__ int next_cta(const void* answer) {
  uint32_t got, x;
  asm volatile(
      "{\n .reg .b128 h;\n .reg .pred p;\n ld.shared.b128 h, [%2];\n mov.u32 %1, 0;\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n selp.u32 %0, 1, 0, p;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n}\n"
      : "=r"(got), "=r"(x) : "r"(smem_u32(answer)) : "memory");
  return got ? (int)x : -1;
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
// The self-test's wait: polls that do not suspend, so that a limit of any length can run out.
__device__ __forceinline__ bool short_wait(uint64_t* bar, uint32_t parity, long long most_cycles) {
  const long long start = clock64();
  do {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (done) return true;
  } while (clock64() - start < most_cycles);
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
// Bits 15 and 31 of the result: infinity or NaN in either half of a pair of 16-bit values.
template <typename T>
__device__ __forceinline__ uint32_t non_finite(uint32_t pair) {
  constexpr uint32_t step = 0x8000u - kExponent<T>;  // carries an exponent of ones into the sign's place
  return ((pair & 0x7fff7fffu) + (step << 16 | step)) & 0x80008000u;
}
// The pair with such values replaced by zero.
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t pair) {
  const uint32_t n = non_finite<T>(pair);
  return pair & ~((n >> 15) * 0xffffu);
}

// NaN for row `row` of a tile (or of this share of it) that was not computed.
template <typename T, int D>
__device__ __noinline__ void void_row(const PrefillArgs& p, const Work& w, int row) {
  if (row >= w.rows) return;
  const float nan = __int_as_float(0x7fc00000);
  if (w.parts > 1) {
    float* stat = p.part_stat + ((int64_t)w.share * kTile + row) * 2;
    stat[0] = -INFINITY;
    stat[1] = nan;
    return;
  }
  const int token = w.first_token + row / p.a.group, h = w.head * p.a.group + row % p.a.group;
  T* out = static_cast<T*>(p.a.out) + token * p.a.out_n + (int64_t)h * p.a.out_h;
  for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(out + c) = make_uint4(~0u, ~0u, ~0u, ~0u);
  if (p.a.lse) p.a.lse[(int64_t)token * p.a.heads + h] = nan;
}

template <typename T, int D, bool kSelfTest = false>
__global__ void __launch_bounds__(kPrefillThreads, 2)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                         const __grid_constant__ CUtensorMap v_map, const __grid_constant__ PrefillArgs p) {
  using L = Layout<D>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Barriers bar;
  __shared__ __align__(16) unsigned char answer[16];
  const AttentionArgs& a = p.a;
  const auto wait_for = [&](uint64_t* b, uint32_t parity) {
    if constexpr (kSelfTest) return short_wait(b, parity, p.wait_cycles);
    else return phase_wait(b, parity);
  };
  // For copies and products under way, which end by themselves: never cut short.
  const auto drain = [](uint64_t* b, uint32_t parity) { return phase_wait(b, parity); };
  unsigned char* q_s = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* k_s = q_s + L::kQ;
  unsigned char* v_s = k_s + L::kStages * L::kBlock;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (p.splits > 1) start_next_kernel();
  const int requests = requests_of(a.pages);
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
      mbar_init(&bar.work_full[b], 1);
      mbar_init(&bar.work_empty[b], kRowThreads / 32 + 3);
      mbar_init(&bar.drain[b], 1);
    }
    mbar_init(&bar.clean_ask, 1);
    mbar_init(&bar.v_clean, 1);
    mbar_init(&bar.q_full, 1);
    mbar_init(&bar.q_empty, 1);
    mbar_init(&bar.next_here, 1);
    bar.found = -1;
    bar.has_left = 0;
    fence_mbar_init();
  }
  // The request of the first tile; later ones are found from there.
  const auto tiles_of = [&](const Request& q) { return (q.news + p.tile_tokens - 1) / p.tile_tokens; };
  // Last tiles first (they have the most keys), splits innermost.
  const auto tile_at = [&](int index) {
    return p.tiles - 1 - (index < p.whole_items ? index : p.whole_items + (index - p.whole_items) / p.splits) / a.kv_heads;
  };
  int all_tiles = 0;
  {
    const int tile = tile_at(blockIdx.x);
    for (int r0 = 0; r0 < requests; r0 += kPrefillThreads) {
      const int r = r0 + threadIdx.x;
      Request q{0, 0, 0};
      bool too_long;
      if (r < requests) q = request_at(a.pages, a.tokens, a.max_keys, r, &too_long);
      const int n = tiles_of(q);
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) bar.sums[warp] = upto;
      __syncthreads();
      int start = all_tiles + upto - n;
#pragma unroll
      for (int w = 0; w < kPrefillThreads / 32; ++w) {
        if (w < warp) start += bar.sums[w];
        all_tiles += bar.sums[w];
      }
      if (tile >= start && tile < start + n) {
        bar.found = r;
        bar.found_start = start;
      }
      __syncthreads();
    }
  }
  if (warp == 4) {
    tmem_alloc(&bar.tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem;

  // Every warp walks the CTA's tiles; `g` counts its blocks over all of them (buffers and
  // phases go on from tile to tile), `t` the tiles. Where a wait runs out a warp leaves.
  uint32_t g = 0, rows_done = 0;  // rows_done: tiles whose rows this warp has written
  const auto next_work = [&](uint32_t t) {
    return __all_sync(0xffffffffu, wait_for(&bar.work_full[t & 1], (t >> 1) & 1));
  };
  const auto done_with = [&](uint32_t t) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar.work_empty[t & 1]);
  };

  if (warp == 4) {
    // ---------------- scores ----------------
    // The issuing warps walk the blocks whole, with values the compiler knows to be the same
    // in all lanes, and one lane issues. Each has one product: a warp that issued both, with
    // its waits, took longer for a block than its softmax does.
    constexpr uint32_t idesc = idesc_of<T>(kKeys, false);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t q_desc = smem_desc_k_sw128(smem_u32(q_s));
    bool ok = true;
    uint32_t queries = 0;
    for (uint32_t t = 0; ok; ++t) {
      if (!(ok = next_work(t))) break;
      const Work& w = bar.work[t & 1];
      const int n = __shfl_sync(0xffffffffu, w.blocks, 0);
      if (w.rows < 0) break;
      if (n) ok = __all_sync(0xffffffffu, wait_for(&bar.q_full, queries++ & 1));
      for (int j = 0; j < n && ok; ++j, ++g) {
        const uint32_t s = g % L::kStages, b = g % L::kScores;
        // The last scores of this buffer are in the rows' registers, K is here.
        if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.s_read[b], ((g / L::kScores) & 1) ^ 1) &&
                                               wait_for(&bar.k_full[s], (g / L::kStages) & 1))))
          break;
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
          if (j == n - 1) umma_commit(&bar.q_empty);
        }
        __syncwarp();
      }
      done_with(t);
    }
    // Neither tensor memory nor the tiles are released under products still running.
    if (elect_one()) umma_commit(&bar.drain[0]);
    drain(&bar.drain[0], 0);
  } else if (warp == 6) {
    // ---------------- output ----------------
    constexpr uint32_t idesc = idesc_of<T>(D, true);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    bool ok = true;
    uint32_t cleaned = 0;
    for (uint32_t t = 0; ok; ++t) {
      if (!(ok = next_work(t))) break;
      const Work& w = bar.work[t & 1];
      const int n = __shfl_sync(0xffffffffu, w.blocks, 0), full0 = __shfl_sync(0xffffffffu, w.full0, 0),
                full1 = __shfl_sync(0xffffffffu, w.full1, 0);
      if (w.rows < 0) break;
      for (int j = 0; j < n; ++j, ++g) {
        const uint32_t s = g % L::kStages;
        ok = wait_for(&bar.v_full[s], (g / L::kStages) & 1);
        const bool partial = j < full0 || j >= full1;
        if (partial && lane == 0) mbar_arrive(&bar.clean_ask);  // cleaned beside the block's softmax
        ok = ok && (!partial || wait_for(&bar.v_clean, cleaned & 1)) && wait_for(&bar.p_full[g & 1], (g >> 1) & 1);
        cleaned += partial;
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
        const uint64_t v_desc = smem_desc_mn_sw128(smem_u32(v_s) + s * L::kBlock, L::kHalf);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < kKeys / 16; ++c)  // 16 keys a step: 8 columns of P, two 8-row groups of V (2,048 bytes)
            umma_ts(tm + L::kOCol, tm + L::kPCol + (g & 1) * (kKeys / 2) + 8 * c, v_desc + 128 * c, idesc, (j | c) != 0);
          umma_commit(&bar.v_empty[s]);
          umma_commit(&bar.o_done[g & 1]);
        }
        __syncwarp();
      }
      done_with(t);
    }
    if (elect_one()) umma_commit(&bar.drain[1]);
    drain(&bar.drain[1], 0);
  } else if (warp == 5) {
    // ---------------- tiles and loads ----------------
    const int in_page = (1 << a.pages.page_log2) - 1, boxes = kKeys / p.box_rows;
    const uint32_t box_bytes = (uint32_t)p.box_rows * 128;
    // The last tile's request: `r` with `before` tiles of others in front of it.
    int r = requests, before = all_tiles;
    Request q{0, 0, 0};
    bool too_long = false;
    if (bar.found >= 0) {
      r = bar.found;
      before = bar.found_start;
      q = request_at(a.pages, a.tokens, a.max_keys, r, &too_long);
    }
    // The work of CTA `index`; false where it has none.
    const auto describe = [&](int index, Work& w) {
      const int cut = index - p.whole_items, splits = cut < 0 ? 1 : p.splits, split = cut < 0 ? 0 : cut % p.splits;
      const int item = cut < 0 ? index : p.whole_items + cut / p.splits, tile = tile_at(index);
      if (tile >= before + tiles_of(q)) {  // not before the last one: from the end
        r = requests;
        before = all_tiles;
        q = Request{0, 0, 0};
      }
      while (tile < before && r > 0) {  // 32 requests back
        const int at = r - 1 - lane;
        Request mine{0, 0, 0};
        bool over = false;
        if (at >= 0) mine = request_at(a.pages, a.tokens, a.max_keys, at, &over);
        const int n = tiles_of(mine);
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const uint32_t here = __ballot_sync(0xffffffffu, tile >= before - upto && tile < before - upto + n);
        const int src = here ? __ffs(here) - 1 : 31;
        r = here ? r - 1 - src : max(r - 32, 0);
        before -= __shfl_sync(0xffffffffu, upto, src);
        q.first = __shfl_sync(0xffffffffu, mine.first, src);
        q.news = here ? __shfl_sync(0xffffffffu, mine.news, src) : 0;
        q.total = __shfl_sync(0xffffffffu, mine.total, src);
        too_long = __shfl_sync(0xffffffffu, (int)over, src);
        if (here) break;
      }
      Tile* join = splits > 1 && split == 0 && lane == 0 ? p.joins + (item - p.whole_items) : nullptr;
      if (tile < before || tile >= before + tiles_of(q)) {  // the grid has room for more tiles than there are
        if (join) join->parts = 0;
        return false;
      }
      const int token0 = (tile - before) * p.tile_tokens, tokens = min(p.tile_tokens, q.news - token0);
      w.r = r;
      w.head = item % a.kv_heads;
      w.first_token = q.first + token0;
      w.rows = tokens * a.group;
      w.pos0 = q.total - q.news + token0;
      w.pos1 = w.pos0 + tokens - 1;
      w.hi = max(w.pos1 + 1, 0);
      w.lo = a.window ? max(w.pos0 - a.window + 1, 0) : 0;
      const int first = w.lo / kKeys, blocks = max((w.hi + kKeys - 1) / kKeys - first, 0);
      // Shares of at least four blocks: a share's fixed cost is about theirs.
      int share = blocks;
      if (splits > 1) share = max((blocks + splits - 1) / splits, 4);
      w.parts = blocks && splits > 1 ? (blocks + share - 1) / share : 1;
      w.first = first + split * share;
      w.blocks = max(min(first + blocks, w.first + share) - w.first, 0);
      w.full0 = a.window ? max((max(w.pos1 - a.window + 1, 0) + kKeys - 1) / kKeys - w.first, 0) : 0;
      w.full1 = (w.pos0 + 1) / kKeys - w.first;
      w.share = cut;
      w.bad = too_long;
      w.wild = 0;
      if (join) {
        join->token0 = w.first_token;
        join->rows = w.rows;
        join->kv_head = w.head;
        join->parts = w.parts;
      }
      return split < w.parts;
    };
    // This lane has a box of the block to load.
    const auto has_box = [&](const Work& w, int j) {
      const int key = (w.first + j) * kKeys + lane * p.box_rows;
      return lane < boxes && j < w.blocks && key < w.hi && key + p.box_rows > w.lo;
    };
    // Its entry of the page table, read a block ahead and checked when the box is loaded (-1: nothing to load).
    const auto entry_of = [&](const Work& w, int j) {
      const int key = (w.first + j) * kKeys + lane * p.box_rows;
      return has_box(w, j) ? __ldg(a.pages.page_table + w.r * a.pages.table_stride + (key >> a.pages.page_log2)) : -1;
    };
    const auto page_of = [&](const Work& w, int j, int entry, int* bad) {
      if (!has_box(w, j)) return -1;
      if (entry >= 0 && entry < a.pages.num_pages) return entry;
      *bad = 1;
      return -1;
    };
    const auto load = [&](const Work& w, int j, int page, const CUtensorMap* map, unsigned char* ring, uint64_t* full) {
      const uint32_t s = g % L::kStages, count = __popc(__ballot_sync(0xffffffffu, page >= 0));
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
    const auto leave = [&](const Work& w) {
      if (lane == 0) {
        bar.left = w;
        bar.has_left = 1;
      }
    };
    bool ok = true, asking = false;
    uint32_t t = 0, queries = 0, asked = 0;
    uint32_t k_loads = 0, v_loads = 0, q_loads = 0;  // begun
    for (int index = blockIdx.x; index >= 0;) {
      Work w;
      if (describe(index, w)) {
        Work& slot = bar.work[t & 1];
        int entry = entry_of(w, 0);
        if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.work_empty[t & 1], ((t >> 1) & 1) ^ 1)))) {
          leave(w);
          break;
        }
        if (lane == 0) {
          slot = w;
          mbar_arrive(&bar.work_full[t & 1]);
        }
        __syncwarp();
        ++t;
        for (int j = 0; j < w.blocks; ++j, ++g) {
          const uint32_t s = g % L::kStages, parity = ((g / L::kStages) & 1) ^ 1;
          const int page = page_of(w, j, entry, &slot.bad);
          entry = entry_of(w, j + 1);
          if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.k_empty[s], parity)))) break;
          load(w, j, page, &k_map, k_s, bar.k_full);
          ++k_loads;
          if (j == 0) {
            // The last tile's scores have been computed: its Q can go.
            if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.q_empty, (queries & 1) ^ 1)))) break;
            ++queries;
            if (lane == 0) {
              mbar_arrive_expect_tx(&bar.q_full, p.tile_tokens * a.group * 128 * L::kHalves);
#pragma unroll
              for (int h = 0; h < L::kHalves; ++h)
                tma_load_3d(smem_u32(q_s) + h * L::kQHalf, &q_map, h * 64, w.head * a.group, w.first_token, &bar.q_full);
            }
            __syncwarp();
            ++q_loads;
          }
          if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.v_empty[s], parity)))) break;
          load(w, j, page, &v_map, v_s, bar.v_full);
          ++v_loads;
        }
        if (!ok) break;
      }
      // Asked for late, while the last blocks are computed, so that an idle CTA is not left without.
      if (lane == 0) {
        fence_proxy_async_smem();  // the last answer has been read
        mbar_arrive_expect_tx(&bar.next_here, 16);
        ask_next_cta(answer, &bar.next_here);
      }
      __syncwarp();
      asking = true;
      if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.next_here, asked++ & 1)))) break;
      asking = false;
      index = __shfl_sync(0xffffffffu, next_cta(answer), 0);
    }
    if (lane == 0) bar.posted = t;
    if (ok) {
      ok = __all_sync(0xffffffffu, wait_for(&bar.work_empty[t & 1], ((t >> 1) & 1) ^ 1));
      if (ok && lane == 0) {
        bar.work[t & 1].rows = -1;
        bar.work[t & 1].blocks = 0;
        mbar_arrive(&bar.work_full[t & 1]);
      }
      __syncwarp();
      // No product's arrival on an empty barrier lands after the CTA has gone.
      for (uint32_t e = g; e < g + L::kStages && ok; ++e) {
        const uint32_t s = e % L::kStages, parity = ((e / L::kStages) & 1) ^ 1;
        ok = __all_sync(0xffffffffu, wait_for(&bar.k_empty[s], parity) && wait_for(&bar.v_empty[s], parity));
      }
      if (ok) ok = __all_sync(0xffffffffu, wait_for(&bar.q_empty, (queries & 1) ^ 1));
    }
    if (!ok) {
      // A wait ran out: what is still on its way to shared memory has to arrive. A tile that does is not computed.
      if (asking && __all_sync(0xffffffffu, drain(&bar.next_here, (asked - 1) & 1))) {
        const int index = __shfl_sync(0xffffffffu, next_cta(answer), 0);
        Work w;
        if (index >= 0 && describe(index, w)) leave(w);
      }
      if (q_loads) drain(&bar.q_full, (q_loads - 1) & 1);
      for (uint32_t back = 1; back <= L::kStages; ++back) {
        if (k_loads >= back) drain(&bar.k_full[(k_loads - back) % L::kStages], ((k_loads - back) / L::kStages) & 1);
        if (v_loads >= back) drain(&bar.v_full[(v_loads - back) % L::kStages], ((v_loads - back) / L::kStages) & 1);
      }
    }
  } else if (warp == 7) {
    // ---------------- cleaning ----------------
    uint32_t asked = 0;
    bool ok = true;
    for (uint32_t t = 0; ok; ++t) {
      if (!(ok = next_work(t))) break;
      Work& w = bar.work[t & 1];
      if (w.rows < 0) break;
      const int n = w.blocks, full0 = w.full0, full1 = w.full1;
      for (int j = 0; j < n; ++j, ++g) {
        if (j >= full0 && j < full1) continue;
        const uint32_t s = g % L::kStages;
        // Asked by the warp that has seen the block arrive.
        if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.clean_ask, asked++ & 1) &&
                                               wait_for(&bar.v_full[s], (g / L::kStages) & 1))))
          break;
        const int kb = (w.first + j) * kKeys, lo = w.lo - kb, hi = w.hi - kb;
        uint4* v = reinterpret_cast<uint4*>(v_s + s * L::kBlock);
        bool wild = false;
        constexpr int kFlight = 8;
#pragma unroll 1
        for (int i0 = lane; i0 < kKeys * D / 8; i0 += 32 * kFlight) {
          uint4 x[kFlight];
#pragma unroll
          for (int f = 0; f < kFlight; ++f) x[f] = v[i0 + 32 * f];
#pragma unroll
          for (int f = 0; f < kFlight; ++f) {
            const int i = i0 + 32 * f, key = (i >> 3) & (kKeys - 1);
            if (key < lo || key >= hi) {
              v[i] = make_uint4(0, 0, 0, 0);
            } else if (non_finite<T>(x[f].x) | non_finite<T>(x[f].y) | non_finite<T>(x[f].z) | non_finite<T>(x[f].w)) {
              v[i] = make_uint4(finite_only<T>(x[f].x), finite_only<T>(x[f].y), finite_only<T>(x[f].z),
                                finite_only<T>(x[f].w));
              wild = true;
            }
          }
        }
        if (wild) w.wild = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.v_clean);
      }
      done_with(t);
    }
  } else {
    // ---------------- softmax and output rows ----------------
    const int row = threadIdx.x;
    const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
    const float scale = a.scale_log2;
    bool ok = true;
    for (; ok; ++rows_done) {
      const uint32_t t = rows_done;
      if (!(ok = next_work(t))) break;
      const Work& w = bar.work[t & 1];
      if (w.rows < 0) break;
      // Row state; the row's keys are [see_lo, see_hi].
      const int blocks = w.blocks, first = w.first, full0 = w.full0, full1 = w.full1;
      int see_hi = -1, see_lo = 0;
      float top = -INFINITY, sum = 0.f;
      if (row < w.rows) {
        see_hi = w.pos0 + row / a.group;
        if (a.window && see_hi - a.window + 1 > 0) see_lo = see_hi - a.window + 1;
      }
      for (int j = 0; j < blocks; ++j, ++g) {
        const uint32_t b = g % L::kScores;
        if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.s_full[b], (g / L::kScores) & 1)))) break;
        tc_fence_after();
        uint32_t s[2][32];
        tmem_ld32(mine + L::kSCol + b * kKeys, s[0]);
        tmem_ld32(mine + L::kSCol + b * kKeys + 32, s[1]);
        tmem_wait_ld();
        pin(s[0]);
        pin(s[1]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.s_read[b]);
        if (j < full0 || j >= full1) {
          const int hi = see_hi - (first + j) * kKeys, lo = see_lo - (first + j) * kKeys;
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
          if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1)))) break;
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
        if (!(ok = __all_sync(0xffffffffu, wait_for(&bar.o_done[g & 1], ((g >> 1) & 1) ^ 1)))) break;
        tc_fence_after();
        tmem_st32(mine + L::kPCol + (g & 1) * (kKeys / 2), out);
        const float2 both = __fadd2_rn(__fadd2_rn(add[0], add[1]), __fadd2_rn(add[2], add[3]));
        sum += both.x + both.y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_full[g & 1]);
      }
      if (blocks && ok) ok = wait_for(&bar.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) sum = __int_as_float(0x7fc00000);  // a wait ran out: no output that could pass for one

      // ---- the tile's output
      tc_fence_after();
      const bool bad = w.bad, wild = w.wild, whole = w.parts == 1;
      if (bad) sum = __int_as_float(0x7fc00000);
      if (bad && row == 0) atomicOr(&g_device_error, kDeviceErrorIndex);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int i_token = row / a.group, token = w.first_token + i_token;
      const int h = w.head * a.group + row - i_token * a.group;
      const bool valid = row < w.rows;
      const int64_t share = w.share;
      const float top2 = top == -INFINITY ? top : top * scale;
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
            if (j >= full0 && j < full1) continue;
            const int kb = (first + j) * kKeys;
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
          float4* out = reinterpret_cast<float4*>(p.part_out + (share * kTile + row) * D + 32 * c);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            out[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                                 __uint_as_float(o[4 * i + 3]));
        }
      }
      if (valid) {
        if (!whole) {
          p.part_stat[(share * kTile + row) * 2] = top2;
          p.part_stat[(share * kTile + row) * 2 + 1] = sum;
        } else if (a.lse) {
          a.lse[(int64_t)token * a.heads + h] = (top2 + log2f(sum) - kProbabilityShift<T>) * 0.6931471805599453f;
        }
      }
      tc_fence_before();
      done_with(t);
    }
    tmem_wait_st();  // where a wait ran out between a store and its use
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  // Tiles that were left where a wait ran out (at most the two that are in work, and one more).
  if (warp < 4) {
    for (; rows_done < bar.posted; ++rows_done) void_row<T, D>(p, bar.work[rows_done & 1], threadIdx.x);
    if (bar.has_left) void_row<T, D>(p, bar.left, threadIdx.x);
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
  // What no CTA wrote (a wait ran out) may be anything.
  if (t.parts > p.splits || t.rows > kTile || t.kv_head < 0 || t.kv_head >= a.kv_heads || t.token0 < 0 ||
      t.token0 >= a.tokens - (t.rows - 1) / a.group)
    return;
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

// The rows as {D, heads, tokens}, a box of 64 columns x the query heads of a key head x a tile's tokens.
bool encode_rows(CUtensorMap* map, const void* base, int dtype, int D, int64_t heads, int64_t tokens, int64_t s_head,
                 int64_t s_token, int64_t group, int64_t tile_tokens) {
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)heads, (uint64_t)tokens};
  const uint64_t strides[2] = {heads > 1 ? (uint64_t)(2 * s_head) : 128, tokens > 1 ? (uint64_t)(2 * s_token) : 128};
  for (uint64_t s : strides)
    if (s == 0 || (int64_t)s < 0) return false;
  const uint32_t box[3] = {64, (uint32_t)group, (uint32_t)tile_tokens};
  return encode_tensor_map(map, dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base,
                           dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, int D, bool kSelfTest = false>
cudaError_t launch(const CUtensorMap& q_map, const CUtensorMap& k_map, const CUtensorMap& v_map, const PrefillArgs& p, int64_t items,
                   cudaStream_t stream) {
  const void* fn = reinterpret_cast<const void*>(&paged_prefill_kernel<T, D, kSelfTest>);
  cudaError_t err = allow_shared_memory(fn, Layout<D>::kSmem);
  if (err != cudaSuccess) return err;
  const int64_t cut = items - p.whole_items;
  err = launch_kernel(paged_prefill_kernel<T, D, kSelfTest>, dim3((unsigned)(p.whole_items + cut * p.splits)), dim3(kPrefillThreads),
                      Layout<D>::kSmem, stream, q_map, k_map, v_map, p);
  if (err != cudaSuccess || p.splits == 1) return err;
  return launch_following(prefill_join_kernel<T, D>, dim3((unsigned)(cut * (kTile / 16))), dim3(512), stream, p);
}

}  // namespace

constexpr int kMostShares = 3;  // for each CTA that the device holds

// Tiles, and the shares that blocks are cut into. The GPU holds 2 CTAs an SM;
// the items that would leave its last round partly empty (all of them, where
// there are few) are cut where the rounds of their shares are shorter together.
// Lengths are only known on the device: the bound on the shares is the page
// table's width. 32/8 heads x 128, whole items against shares: 4,096 tokens over
// 16,384 keys (1,024 items, 3.46 rounds) 1,075 and 1,046 us; 16 requests of 4,096
// keys, 6 tokens each (128 items) 78 and 57 us, 64 tokens each (256) 96 and 84 us.
PrefillPlan plan_paged_prefill(int64_t tokens, int64_t batch, bool ragged, int64_t kv_heads, int64_t group, int D,
                               int64_t max_keys, int64_t window, int sms) {
  PrefillPlan p{};
  p.tile_tokens = (int)(kTile / group);
  p.tiles = tokens;
  if (ragged) {
    // Every request (and the padding on either side) may leave its last tile partly empty.
    const int64_t ends = tokens < batch + 2 ? tokens : batch + 2;
    p.tiles = (tokens + ends * (p.tile_tokens - 1)) / p.tile_tokens;
  }
  // Tiles that there are likely to be (requests of the same size): those beyond them come first and end at once.
  const int64_t asked = tokens < batch ? tokens : batch, each = (tokens + asked - 1) / asked;
  const int64_t likely = asked * ((each + p.tile_tokens - 1) / p.tile_tokens);
  const int64_t items = p.tiles * kv_heads, slots = 2 * (int64_t)sms;
  const int64_t real = likely < p.tiles ? likely * kv_heads : items, cut = real % slots;
  // Where all may run at once, none is left whole: it would take as long as all its keys.
  const int64_t room = real < slots ? items : cut;
  p.whole_items = items - room;
  p.splits = 1;
  if (cut) {
    const int64_t keys = window && window + p.tile_tokens < max_keys ? window + p.tile_tokens : max_keys;
    const int64_t blocks = keys / kKeys + 1, most = (blocks + 4) / 4;  // shares of at least four blocks
    // Rounds times a share's blocks, with about 3 for its start and end and 3 for the join.
    int64_t least = blocks + 3;
    for (int64_t s = 2; s <= most && room * s <= kMostShares * slots; ++s) {
      const int64_t cost = (cut * s + slots - 1) / slots * ((blocks + s - 1) / s + 3) + 3;
      if (cost < least) {
        least = cost;
        p.splits = (int)s;
      }
    }
  }
  if (p.splits == 1) p.whole_items = items;
  return p;
}

size_t paged_prefill_workspace(int D, int sms) {
  return (size_t)(kMostShares * 2 * sms) * (kTile * (size_t)(D + 2) * sizeof(float) + sizeof(Tile));
}

bool launch_paged_prefill(const AttentionArgs& a, const PrefillPlan& plan, int dtype, int D, int64_t page_size,
                          long long wait_cycles, cudaStream_t stream, cudaError_t* err) {
  PrefillArgs p{};
  p.a = a;
  p.wait_cycles = wait_cycles;
  p.tile_tokens = plan.tile_tokens;
  p.splits = plan.splits;
  p.whole_items = (int)plan.whole_items;
  p.tiles = (int)plan.tiles;
  p.box_rows = page_size < kKeys ? (int)page_size : kKeys;
  const int64_t items = plan.tiles * a.kv_heads;
  if (items * plan.splits * (kTile / 16) >= (int64_t(1) << 31)) return false;
  CUtensorMap q_map, k_map, v_map;
  if (!encode_rows(&q_map, a.q, dtype, D, a.heads, a.tokens, a.q_h, a.q_n, a.group, plan.tile_tokens) ||
      !encode_cache(&k_map, a.k, dtype, D, page_size, a.kv_heads, a.pages.num_pages, a.k_slot, a.k_head, a.k_page,
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
  if (wait_cycles)
    *err = D == 64 ? launch<__nv_bfloat16, 64, true>(q_map, k_map, v_map, p, items, stream)
                   : launch<__nv_bfloat16, 128, true>(q_map, k_map, v_map, p, items, stream);
  else if (D == 64)
    *err = dtype == 0 ? launch<__nv_bfloat16, 64>(q_map, k_map, v_map, p, items, stream)
                      : launch<__half, 64>(q_map, k_map, v_map, p, items, stream);
  else
    *err = dtype == 0 ? launch<__nv_bfloat16, 128>(q_map, k_map, v_map, p, items, stream)
                      : launch<__half, 128>(q_map, k_map, v_map, p, items, stream);
  return true;
}

cudaError_t read_paged_prefill_device_error(int* value, bool reset) {
  cudaError_t err = cudaMemcpyFromSymbol(value, g_device_error, sizeof(int));
  if (err != cudaSuccess || !reset) return err;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
}

}  // namespace flash_prologue
