// Attention of a few new tokens a request over a paged cache held in 4 bits:
// o_i = sum_j p_ij v_j with p the softmax of the scaled scores over the keys that
// row i sees, k and v the products s * (u - 8) of scales s and stored codes u.
//
// Bound by HBM in bytes (72 a row at D = 128), but each byte holds two values, so
// the instructions that bring codes to the matrix units count as much. Few are
// needed: the 16 bits u have the value u * 2^-24 as an FP16 number, and 16 u the
// value u * 2^-20, so an AND takes two codes of a word (four bits each, 16 bits
// apart) to an operand register, with no arithmetic at all. The powers of two go
// into the other operand and the results; scales and the 8 come in afterwards,
// exactly:
//   S_ij = sum_g s_jg (sum_{c in g} q_ic u_jc - 8 sum_{c in g} q_ic)
//   O_id = sum_j (p_ij s_jg) u_jd - 8 sum_j (p_ij s_jg),   g the group of d.
// The first sums start at -8 sum q instead of 0; the last one is a matrix product
// with a constant. Keys (then channels) are the 16 rows of the instructions and
// query rows their 8 columns: a group of up to 8 query heads fills them with one
// product where 16-row tiles of Q would leave half empty.
//
// Q is FP16 for the product, scaled by a power of two a row so that its largest
// value is 2^14 to 2^15, or 2^10 to 2^11 beside codes of 16 u: values below 2^-24 of these
// (2^-35 of the row's largest) lose bits to FP16's steps. The weights
// p s are rounded to FP16 once, p 2^8 times as large and s less the power of two sigma above the
// largest scales that the row has seen in this group of channels, so that they are below 2^15: an error of the size
// of a 16-bit output's rounding, and where a weight is below 2^-14, of 2^-33 of that power (with one
// sigma for all groups it was that of the largest group for all; 64 requests 98 us instead of 99). A sigma that moves goes one
// further than it has to (each time as far as it has to: 3 us more). Scores, statistics and sums are FP32. The
// maximum that scales a row of O moves only when the row's has grown by more than 2^7.
//
// Work is shared out as in paged_decode.cu (paged_runs.cuh). A warp takes 16 keys of
// one key head a step; a CTA's four warps take neighbouring heads of the same keys
// where there are such, since their rows lie next to each other. Where a page holds
// the four warps' step and the layout is one for tensor maps, a step comes by four
// copies into a ring of the CTA, else every warp loads its own with cp.async (64 requests:
// 113 us instead of 120). 16 keys a step and 3 CTAs an SM at D = 128 are what 168 registers
// hold: 32 keys 123 to 127 us, 4 CTAs 123 (at 128 registers), 2 CTAs 117 (3 took 102 to 103 then). One product's
// rows for the 8 sum p s of all groups would save 12 registers, but its sums wait for one another: 106 us instead of 102.
//
// Measured (32/8 heads x 128 BF16 unless said): 64 requests of up to 8,192 keys 99 us, 339 MB, 3.4
// TB/s (52 us at the copy rate; the same over a 16-bit cache 201 us); issue slots 51% and ALU 46%
// busy with three warps a scheduler: about 350 instructions a step, half of them products, masks of codes
// and the scales' multiplications. 2 requests of 131,071 keys, 16/2 heads FP16: 31.5 us (16-bit cache 48). 1
// request of 1,000 keys: 12.0 us, latency.
#include "paged_runs.cuh"
#include "tensor_map.h"
#include "umma_util.cuh"

namespace flash_prologue {
namespace {

// Steps of a ring, and how many a CTA's common ring is loaded ahead. (6 and 4, 6 and 3, 5 and 3: 99 to 100 us
// where 4 and 2 took 98.)
constexpr int kRing = 4;
constexpr int kAhead = 2;
constexpr int kBlockKeys = kWarpKeys * kDecodeWarps;
constexpr int kCtasPerSm = 4;
// Exponents of the powers of two above a group's scales: with these, 2^-sigma and 2^(sigma - 8) are normal numbers.
constexpr int kLeastScale = -110, kMostScale = 126;
// A probability of 1 is 2^8 here, and a row's maximum moves where one would be more than 2^15.
constexpr float kShift = 8.f, kMostWeight = 0x1p15f, kMostGrowth = 7.f;
constexpr float kNoTop = -3e38f;      // the maximum of a row that has seen no key
constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;

template <int BYTES>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, bool ok) {
  const int bytes = ok ? BYTES : 0;  // 0: zeros, src is not read
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// d = a b + c of 16 x 16 and 16 x 8 FP16 fragments.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, float c0, float c1, float c2, float c3) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%10, %11, %12, %13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {  // of an 8 x 8 matrix of 16-bit values over the warp
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 floats_of(uint32_t half2) { return __half22float2(*reinterpret_cast<__half2*>(&half2)); }
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 .. 127
// Words of two 16-bit numbers. Magnitudes of BF16 numbers compare as whole numbers do.
__device__ __forceinline__ uint32_t finite_sizes(uint32_t x) {  // |x|, zero for infinities and NaNs
  x &= 0x7fff7fffu;
  return x & ~(((x + 0x00800080u) >> 15 & 0x00010001u) * 0xffffu);
}
__device__ __forceinline__ uint32_t bf16_power(int e) { return (uint32_t)(e + 127) << 7; }
__device__ __forceinline__ __nv_bfloat162 bf16x2_of(uint32_t a) { return *reinterpret_cast<__nv_bfloat162*>(&a); }
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {  // (exact by powers of two)
  const __nv_bfloat162 x = __hmul2(bf16x2_of(a), bf16x2_of(b));
  return *reinterpret_cast<const uint32_t*>(&x);
}
// The two BF16 numbers of a word.
__device__ __forceinline__ float low_bf16(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high_bf16(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// A row's scales: G of them in G / 2 words.
template <int G>
struct Scales {
  uint32_t w[G / 2];
  __device__ __forceinline__ void load(uint32_t addr) {
    if constexpr (G == 4) {
      const uint2 v = lds64(addr);
      w[0] = v.x;
      w[1] = v.y;
    } else {
      w[0] = lds32(addr);
    }
  }
  __device__ __forceinline__ float get(int g) const { return g & 1 ? high_bf16(w[g / 2]) : low_bf16(w[g / 2]); }
};
// G words of a row's piece.
template <int G>
__device__ __forceinline__ void load_words(uint32_t (&w)[G], uint32_t addr) {
  if constexpr (G == 4) {
    const uint4 v = lds128(addr);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
    const uint2 v = lds64(addr);
    w[0] = v.x; w[1] = v.y;
  }
}

// A step's 16 keys of a head, one row of codes each. Slot k of the products (rows of S, columns of
// V^T) is key key_of(k), and a row's pieces lie as at() says, which is how a tensor map with 64-byte
// (32-byte) swizzle lays out rows of 64 (32) bytes. So the 8 lanes (16 at D = 64) that read shared memory
// at once find their pieces in different banks, both for K (4 pieces of neighbouring slots) and for V
// (few pieces of every other slot).
template <int D>
__device__ __forceinline__ int key_of(int slot) { return slot ^ (D == 128 ? slot >> 1 & 1 : slot >> 2 & 1); }
template <int D>
__device__ __forceinline__ int at(int key, int piece) {  // bytes; piece 0 .. 3 of a row
  if constexpr (D == 128) return key * 64 + ((piece ^ (key >> 1 & 3)) * 16);
  else return key * 32 + (((piece >> 1) ^ (key >> 2 & 1)) * 16) + (piece & 1) * 8;
}

template <int D>
struct Step {  // bytes of a head's step: K, V, scales of K, scales of V
  static constexpr int kCodes = kWarpKeys * D / 2, kScale = kWarpKeys * D / 16, kBytes = 2 * (kCodes + kScale);
};

// A cache as the copies of a CTA's heads see it (pages that hold a step's keys, scales next to each other along
// the heads or along the slots).
struct Maps {
  CUtensorMap k, v, k_scale, v_scale;
  int scales_by_slot;  // a step's scales lie [head][slot] in memory, else [slot][head]
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
// True when the phase is complete; false (and the error word) after about 4 s.
__device__ __forceinline__ bool phase_wait(uint64_t* bar, uint32_t parity) {
  constexpr long long kMostCycles = 8000000000ll;
  const uint32_t b = smem_u32(bar);
  const auto done = [&] {
    uint32_t d;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(d) : "r"(b), "r"(parity) : "memory");
    return d != 0;
  };
  if (done()) return true;
  const long long start = clock64();
  do {
    if (done()) return true;
  } while (clock64() - start < kMostCycles);
  atomicOr(&g_device_error, kDeviceErrorTimeout);
  return false;
}

// Shared memory of a CTA: its rings, later its warps' sums; then the warps' Q (kept there, since registers are
// what limits the warps of an SM).
template <int D, int NT>
constexpr size_t room_of() {
  constexpr size_t ring = (size_t)kDecodeWarps * kRing * Step<D>::kBytes, joined = (size_t)kDecodeWarps * 8 * NT * D * 4;
  return ring > joined ? ring : joined;
}
template <int D, int NT>
constexpr uint32_t kQueryBytes = NT * (D / 32) * (512 + 64);

struct Int4Args {
  AttentionArgs a;  // k, v: codes, strides in bytes
  const uint16_t* k_scale;
  const uint16_t* v_scale;
  int64_t ks_page, ks_slot, ks_head, vs_page, vs_slot, vs_head;  // elements
};

// CTAs of an SM by registers: 3 (D = 64: 4, two tiles of rows: 2). NT tiles of 8 rows; HEADS key heads a CTA, so 4 / HEADS warps share a head's keys. TMA: a step of all
// four warps comes by tensor copies into a ring of the CTA, issued by its warps in turn; else every warp loads
// its own with cp.async.
template <typename T, int D, int NT, int HEADS, bool TMA>
__global__ void __launch_bounds__(kDecodeThreads, NT == 1 ? D == 64 ? 4 : 3 : 2)
    paged_int4_decode_kernel(const Int4Args args, const __grid_constant__ Maps maps) {
  const AttentionArgs& a = args.a;
  constexpr int kRows = 8 * NT, kSplit = kDecodeWarps / HEADS, kStepKeys = kWarpKeys * kSplit;  // keys of a CTA's step
  constexpr int G = D / 32;  // groups of channels; words of a piece
  constexpr int kPerBlock = kBlockKeys / kStepKeys;
  using Tiles = Tiling<kRows, kBlockKeys, HEADS>;
  using S = Step<D>;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ RunScratch shared;
  __shared__ float stat[kDecodeWarps][kRows][2];
  // 2^-sigma of each group and column of a warp's tile: sigma is the power of two above the scales of V that the row has seen.
  __shared__ __align__(8) float inv_scale[kDecodeWarps][NT][G][8];
  __shared__ int bad_page;
  __shared__ uint64_t full[kRing], empty[kRing];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr uint32_t kStage = TMA ? kDecodeWarps * S::kBytes : S::kBytes;
  const uint32_t ring = smem_u32(smem) + (TMA ? 0 : warp * kRing * kStage), ring_end = ring + kRing * kStage;
  // The warp's Q fragments (16 bytes a lane and group), then what their sums start at (16 bytes a pair of columns).
  const uint32_t q_s = smem_u32(smem) + (uint32_t)room_of<D, NT>() + warp * kQueryBytes<D, NT>, start_s = q_s + NT * G * 512;

  if (!a.whole) start_next_kernel();
  if constexpr (TMA) {
    if (threadIdx.x == 0) {
      for (int s = 0; s < kRing; ++s) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], kDecodeWarps);
      }
      fence_mbar_init();
    }
  }
  const int64_t slots = 2 * (int64_t)gridDim.x, cta = blockIdx.x;
  float* part_out = static_cast<float*>(a.workspace);                            // [slots][HEADS][kRows][D]
  float* part_stat = part_out + slots * HEADS * kRows * D;                       // [slots][HEADS][kRows][2]
  Part* parts = reinterpret_cast<Part*>(part_stat + slots * HEADS * kRows * 2);  // [grid]
  Run run;
  if (!find_run<Tiles>(a, shared, parts, run)) return;

  // This lane's places in the products. K: slots j and j + 8, piece p of the row. V: piece and
  // half (even or odd channels) of the words, slots 2 p, 2 p + 1 and 8 more. In bytes of a stage.
  const int j = lane / 4, p = lane % 4;
  constexpr int kEight = kWarpKeys * D / 4;  // 8 keys on
  const int split = warp / HEADS, step_row = TMA ? (warp % HEADS) * kSplit + split : 0;  // copies: [head][key]
  const uint32_t codes_at = step_row * S::kCodes, v_codes = (TMA ? kDecodeWarps : 1) * S::kCodes + codes_at;
  const uint32_t k_at = codes_at + at<D>(key_of<D>(j), p);
  const uint32_t v_at[2] = {v_codes + at<D>(key_of<D>(2 * p), j % 4), v_codes + at<D>(key_of<D>(2 * p + 1), j % 4)};
  const uint32_t half_of = j / 4 ? 0x7632u : 0x5410u;
  const bool by_head = TMA && !maps.scales_by_slot;  // [slot][head]
  const uint32_t scale_pitch = by_head ? HEADS * D / 16 : D / 16, scale_eight = 8 * scale_pitch;
  const uint32_t ks_at = (TMA ? 2 * kDecodeWarps : 2) * S::kCodes +
                         (by_head ? split * kWarpKeys * scale_pitch + warp % HEADS * (D / 16) : step_row * S::kScale) +
                         key_of<D>(j) * scale_pitch;
  const uint32_t vs_at = ks_at + (TMA ? kDecodeWarps : 1) * S::kScale;
  const bool wide = a.pages.page_log2 >= 4;  // a step's keys are in one page
  const int in_page = (1 << a.pages.page_log2) - 1;
  [[maybe_unused]] uint32_t loads = 0;  // steps of the CTA's items before this one (stages and phases go on)
  [[maybe_unused]] bool lost = false;   // a wait ran out: no more copies or products

  for (int64_t unit = run.begin; unit < run.end;) {
    Item it;
    find_item<Tiles>(a, run, unit, it);
    const Request& q = it.q;
    const int b0 = it.b0, b1 = it.b1, row0 = it.row0, rows = it.rows, base = it.base;
    const int head = it.head + warp % HEADS;
    const bool idle = HEADS > 1 && head >= a.kv_heads;

    // Q: row 8 n + j of the tile, this lane's channels 8 (p G + g) .. + 7 of each group, times a power of two.
    float row_scale[NT][2];  // takes their sums to base-2 scores
    int see_hi[NT][2];       // last position that they see (behind the tile's rows: as its last row)
    const auto token_of = [&](int row) { return q.news == 1 ? 0 : (row0 + row) / a.group; };  // (a division)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = 8 * n + j, i = token_of(row);
      uint4 x[G];
      float most = 0.f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        x[g] = make_uint4(0, 0, 0, 0);
        if (row < rows && !idle)
          x[g] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (q.first + i) * a.q_n +
                                                      (head * a.group + (row0 + row - i * a.group)) * a.q_h + 8 * (p * G + g)));
        const T* v = reinterpret_cast<const T*>(&x[g]);
#pragma unroll
        for (int c = 0; c < 8; ++c) most = fmaxf(most, fabsf((float)v[c]));
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // (rows below 2^-113 come out smaller: the factor is an FP32 number)
      const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -113), 127);
      const float f = power_of_two(14 - e), f16 = f * 0.0625f;  // the latter beside codes of 16 u
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const T* v = reinterpret_cast<const T*>(&x[g]);
        uint32_t qf[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          qf[c] = half2_of((float)v[2 * c] * (c & 1 ? f16 : f), (float)v[2 * c + 1] * (c & 1 ? f16 : f));
        // -8 sum of q over the group, of this lane's two columns 2 p and 2 p + 1: as keys whose codes are all 8.
        float c[4];
        mma_f16(c, 0x00080008u, 0x00080008u, 0x00800080u, 0x00800080u, qf[0], qf[1], 0.f, 0.f, 0.f, 0.f);
        mma_f16(c, 0x00080008u, 0x00080008u, 0x00800080u, 0x00800080u, qf[2], qf[3], c[0], c[1], c[2], c[3]);
        sts128(q_s + (n * G + g) * 512 + lane * 16, make_uint4(qf[0], qf[1], qf[2], qf[3]));
        const uint32_t c0 = __float_as_uint(-c[0]), c1 = __float_as_uint(-c[1]);
        if (j == 0) sts128(start_s + (n * G + g) * 64 + p * 16, make_uint4(c0, c1, c0, c1));
      }
#pragma unroll
      for (int x2 = 0; x2 < 2; ++x2) {
        // 2^24 of the codes, 2^(e - 14) of the row
        const int up = __shfl_sync(0xffffffffu, e, (2 * p + x2) * 4) + 10;
        row_scale[n][x2] = a.scale_log2 * power_of_two(up / 2) * power_of_two(up - up / 2);
        const int at_row = 8 * n + 2 * p + x2;
        see_hi[n][x2] = base + token_of(min(at_row, rows - 1));
      }
    }
    // Of a column: probabilities are 2^(score - from), from = top - kShift (whole numbers: no rounding). inv: 2^-sigma of each group, sigma the least of this lane's columns, as BF16 numbers.
    float acc[NT][G][2][4], eights[NT][G][4], from[NT][2], sum[NT][2];
    uint32_t inv[G / 2];
#pragma unroll
    for (int i = 0; i < G / 2; ++i) inv[i] = bf16_power(-kLeastScale) * 0x10001u;
    for (int i = lane; i < NT * G * 8; i += 32) (&inv_scale[warp][0][0][0])[i] = power_of_two(-kLeastScale);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[n][g][0][x] = acc[n][g][1][x] = eights[n][g][x] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        from[n][x] = kNoTop;
        sum[n][x] = 0.f;
      }
    }
    if (threadIdx.x == 0) bad_page = it.too_long;
    __syncthreads();

    // Positions relative to this warp's first key, in 32 bits (a request has fewer than 2^30 keys).
    const int steps = idle ? 0 : (b1 - b0) * kPerBlock;
    const int warp_key = it.key0 + b0 * kBlockKeys + split * kWarpKeys;
    const int key_lo = it.lo - warp_key, key_hi = it.hi - warp_key;
    const int all_lo = a.window ? base + (row0 + rows - 1) / a.group - a.window + 1 - warp_key : kNone;
    const int all_hi = base + row0 / a.group - warp_key;  // every row sees keys all_lo .. all_hi
    const int32_t* table = a.pages.page_table + (int64_t)it.r * a.pages.table_stride;
    // Where a group's sigmas are the same in all columns the products take scales that have them already. With one tile of 8
    // rows that goes by the rows (one token: all see the same keys), in code of its own; with two by the sigmas. (64 requests, up to
    // 20 rows: 175 us; by the rows 185. 64 single tokens: 99 us, by the sigmas 101.)
    const bool one_token = token_of(0) == token_of(rows - 1);
    [[maybe_unused]] bool same = true;
    // A step's scores, probabilities and product; EDGE: some row does not see some key.
    const auto compute = [&](auto edge, auto one, uint32_t here, int key) {
      constexpr bool EDGE = decltype(edge)::value;
      // Sums of keys key_of(j) and 8 more (x / 2), columns 2 p and 2 p + 1 (x % 2).
      float s[NT][4] = {};
      {
        uint32_t wa[G], wb[G];
        load_words<G>(wa, here + k_at);
        load_words<G>(wb, here + k_at + kEight);
        Scales<G> sa, sb;
        sa.load(here + ks_at);
        sb.load(here + ks_at + scale_eight);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t ua = wa[g] >> 8, ub = wb[g] >> 8;
          const float fa = sa.get(g), fb = sb.get(g);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 qf = lds128(q_s + (n * G + g) * 512 + lane * 16), c0 = lds128(start_s + (n * G + g) * 64 + p * 16);
            float c[4];
            mma_f16(c, wa[g] & kLow, wb[g] & kLow, wa[g] & kHigh, wb[g] & kHigh, qf.x, qf.y, __uint_as_float(c0.x),
                    __uint_as_float(c0.y), __uint_as_float(c0.z), __uint_as_float(c0.w));
            mma_f16(c, ua & kLow, ub & kLow, ua & kHigh, ub & kHigh, qf.z, qf.w, c[0], c[1], c[2], c[3]);
#pragma unroll
            for (int x = 0; x < 4; ++x) s[n][x] = fmaf(c[x], x < 2 ? fa : fb, s[n][x]);
          }
        }
      }
      Scales<G> va, vb;
      va.load(here + vs_at);
      vb.load(here + vs_at + scale_eight);
      const auto sees = [&](int n, int x) {
        const int k = warp_key + key + key_of<D>(j) + (x / 2) * 8, hi = see_hi[n][x & 1];
        return k <= hi && (!a.window || k > hi - a.window);
      };
      float w[NT][4];  // probabilities times 2^8
      const auto weights = [&] {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            w[n][x] = EDGE && !sees(n, x) ? 0.f : exp2_approx(fmaf(s[n][x], row_scale[n][x & 1], -from[n][x & 1]));
      };
      Scales<G> ua, ub;  // the scales of V times 2^-sigma: below 1, or a sigma moves
      __nv_bfloat162 largest = bf16x2_of(0);
#pragma unroll
      for (int i = 0; i < G / 2; ++i) {
        ua.w[i] = mul_bf16x2(va.w[i], inv[i]);
        ub.w[i] = mul_bf16x2(vb.w[i], inv[i]);
        largest = __hmax2(largest, __hmax2(__habs2(bf16x2_of(ua.w[i])), __habs2(bf16x2_of(ub.w[i]))));
      }
      weights();
      const bool grown = !__hblt2(largest, __float2bfloat162_rn(1.f));
      bool move = grown;
#pragma unroll
      for (int n = 0; n < NT; ++n) move |= fmaxf(fmaxf(w[n][0], w[n][2]), fmaxf(w[n][1], w[n][3])) > kMostWeight;
      if (__any_sync(0xffffffffu, move)) {
        // A row's maximum or a group's largest scale may have moved: its O and sums follow. Each row goes by
        // the keys that it sees, so what others see does not change its bits.
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float most = kNoTop;
#pragma unroll
            for (int y = 0; y < 2; ++y)
              if (!EDGE || sees(n, x + 2 * y)) most = fmaxf(most, s[n][x + 2 * y] * row_scale[n][x]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float was = from[n][x] + kShift, top = most > was + kMostGrowth ? ceilf(most) : was;
            from[n][x] = top - kShift;
            const float f = exp2_approx(fmaxf(was - top, -300.f));
            sum[n][x] *= f;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                acc[n][g][0][2 * r + x] *= f;
                acc[n][g][1][2 * r + x] *= f;
                eights[n][g][2 * r + x] *= f;
              }
          }
        weights();
        if (__any_sync(0xffffffffu, grown)) {
          int least[G], largest_of[G];
#pragma unroll
          for (int g = 0; g < G; ++g) {
            least[g] = kMostScale;
            largest_of[g] = kLeastScale;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              uint32_t big[G / 2];  // infinities and NaNs lose their own group only
#pragma unroll
              for (int i = 0; i < G / 2; ++i) {
                big[i] = __vmaxu2(!EDGE || sees(n, x) ? finite_sizes(va.w[i]) : 0, !EDGE || sees(n, x + 2) ? finite_sizes(vb.w[i]) : 0);
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) big[i] = __vmaxu2(big[i], __shfl_xor_sync(0xffffffffu, big[i], o));
              }
#pragma unroll
              for (int g = 0; g < G; ++g) {
                float& inv_of = inv_scale[warp][n][g][2 * p + x];
                const int sigma_was = 127 - (int)(__float_as_uint(inv_of) >> 23);
                // The power of two above the largest scale; where that has grown one more, so that it seldom does again.
                const int least_of = (int)(big[g / 2] >> (g & 1 ? 23 : 7) & 0xff) - 126;
                const int sigma = least_of > sigma_was ? min(least_of + 1, kMostScale) : sigma_was;
                least[g] = min(least[g], sigma);
                largest_of[g] = max(largest_of[g], sigma);
                const float f = power_of_two(max(sigma_was - sigma, -126));
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  acc[n][g][0][2 * r + x] *= f;
                  acc[n][g][1][2 * r + x] *= f;
                  eights[n][g][2 * r + x] *= f;
                }
                __syncwarp();  // read by the eight lanes of the column
                if (j == 0) inv_of = power_of_two(-sigma);
              }
            }
          bool equal = true;
#pragma unroll
          for (int i = 0; i < G / 2; ++i) {
            inv[i] = bf16_power(-least[2 * i]) | bf16_power(-least[2 * i + 1]) << 16;
            ua.w[i] = mul_bf16x2(va.w[i], inv[i]);
            ub.w[i] = mul_bf16x2(vb.w[i], inv[i]);
            const uint32_t first = __shfl_sync(0xffffffffu, inv[i], 0);
            equal &= (first == inv[i]) & (least[2 * i] == largest_of[2 * i]) & (least[2 * i + 1] == largest_of[2 * i + 1]);
          }
          if constexpr (NT > 1) same = __all_sync(0xffffffffu, equal);
          __syncwarp();
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) sum[n][x & 1] += w[n][x];
      // Channels of this lane: words j % 4 of the four keys, even or odd ones.
      uint32_t w0[G], w1[G], w8[G], w9[G];
      load_words<G>(w0, here + v_at[0]);
      load_words<G>(w1, here + v_at[1]);
      load_words<G>(w8, here + v_at[0] + kEight);
      load_words<G>(w9, here + v_at[1] + kEight);
      const auto add_up = [&](auto alike) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t x = __byte_perm(w0[g], w1[g], half_of), y = __byte_perm(w8[g], w9[g], half_of);
          const uint32_t x8 = x >> 8, y8 = y >> 8;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float z[4];
            if constexpr (decltype(alike)::value) {
#pragma unroll
              for (int i = 0; i < 4; ++i) z[i] = w[n][i] * (i < 2 ? ua : ub).get(g);
            } else {
              const float2 by = *reinterpret_cast<const float2*>(&inv_scale[warp][n][g][2 * p]);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float2 x2 = __fmul2_rn(make_float2(w[n][2 * i], w[n][2 * i + 1]), __fmul2_rn(splat2((i ? vb : va).get(g)), by));
                z[2 * i] = x2.x;
                z[2 * i + 1] = x2.y;
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (EDGE && !sees(n, i)) z[i] = 0.f;  // whatever the scale is
            const uint32_t w_lo = transposed(half2_of(z[0], z[1])), w_hi = transposed(half2_of(z[2], z[3]));
            float (&o0)[4] = acc[n][g][0], (&o1)[4] = acc[n][g][1], (&e)[4] = eights[n][g];
            mma_f16(o0, x & kLow, x & kHigh, y & kLow, y & kHigh, w_lo, w_hi, o0[0], o0[1], o0[2], o0[3]);
            mma_f16(o1, x8 & kLow, x8 & kHigh, y8 & kLow, y8 & kHigh, w_lo, w_hi, o1[0], o1[1], o1[2], o1[3]);
            mma_f16(e, 0x00080008u, 0x00800080u, 0x00080008u, 0x00800080u, w_lo, w_hi, e[0], e[1], e[2], e[3]);
          }
        }
      };
      if constexpr (NT == 1) add_up(one);
      else if (same) add_up(std::true_type{});
      else add_up(std::false_type{});
    };
    const auto products = [&](uint32_t here, int key) {
      const bool inside = key >= all_lo && key + kWarpKeys - 1 <= all_hi;
      if (!inside && (key >= key_hi || key + kWarpKeys <= key_lo)) return;
      if (NT == 1 && one_token) {
        if (inside) compute(std::false_type{}, std::true_type{}, here, key);
        else compute(std::true_type{}, std::true_type{}, here, key);
      } else {
        if (inside) compute(std::false_type{}, std::false_type{}, here, key);
        else compute(std::true_type{}, std::false_type{}, here, key);
      }
    };
    if constexpr (TMA) {
      // Steps with keys that some row sees; warp i % 4 has the copies of step i.
      const int first = warp_key - split * kWarpKeys, step0 = max(it.lo - first, 0) / kStepKeys;
      const int count = max(min(steps, (it.hi - first + kStepKeys - 1) / kStepKeys) - step0, 0);
      const bool was_lost = lost;
      int page_of = -1;  // page of step 4 (lane + 32 n) + warp
      uint32_t issued = loads, load = loads;  // this warp's last copies, the step that is waited for
      const auto issue = [&](int i) {
        if (i >= count || (i & 3) != warp || lost) return;
        const int mine = i >> 2;
        if ((mine & 31) == 0) {
          const int step = (mine + lane) * 4 + warp;
          page_of = step < count ? __ldg(table + ((first + (step0 + step) * kStepKeys) >> a.pages.page_log2)) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, page_of, mine & 31), slot = (first + (step0 + i) * kStepKeys) & in_page;
        const uint32_t load = loads + i, s = load % kRing, dst = ring + s * kStage;
        issued = load;
        if (!(lost = !__all_sync(0xffffffffu, phase_wait(&empty[s], (load / kRing & 1) ^ 1)))) {
          if (lane == 0) {
            if (page >= 0 && page < a.pages.num_pages) {
              mbar_arrive_expect_tx(&full[s], kStage);
              tma_load_4d(dst, &maps.k, 0, slot, it.head, page, &full[s]);
              tma_load_4d(dst + kDecodeWarps * S::kCodes, &maps.v, 0, slot, it.head, page, &full[s]);
              const uint32_t scales = dst + 2 * kDecodeWarps * S::kCodes;
              const int c0 = by_head ? it.head * G : slot * G, c1 = by_head ? slot : it.head;
              tma_load_3d(scales, &maps.k_scale, c0, c1, page, &full[s]);
              tma_load_3d(scales + kDecodeWarps * S::kScale, &maps.v_scale, c0, c1, page, &full[s]);
            } else {
              bad_page = 1;
              mbar_arrive(&full[s]);
            }
          }
          __syncwarp();
        }
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) issue(i);
      for (int i = 0; i < count && !lost; ++i) {
        issue(i + kAhead);
        load = loads + i;
        const uint32_t s = load % kRing;
        if (lost || (lost = !__all_sync(0xffffffffu, phase_wait(&full[s], load / kRing & 1)))) break;
        products(ring + s * kStage, (step0 + i) * kStepKeys);
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }
      loads += count;
      if (lost) {
        bad_page = 1;  // rows without their keys are NaN
        // Copies of this warp that are under way have to arrive before the CTA goes on or ends.
        for (; !was_lost && load <= issued; ++load) phase_wait(&full[load % kRing], load / kRing & 1);
      }
    } else {
      // Its places in the loads: a 16-byte chunk of K and of V in each pass over a step's rows, a row's scales of
      // K (lanes 0 .. 15) or V. Strides of slots and pages take 31 bits (the host checks): a product and a sum
      // in one instruction.
      constexpr int kChunks = D / 32, kPasses = kChunks / 2;
      const int load_row = lane / kChunks, chunk = lane % kChunks;
      const uint32_t load_at = at<D>(load_row, chunk * (4 / kChunks));  // (a piece is half a chunk at D = 64)
      const uint32_t scale_to = 2 * S::kCodes + (lane < 16 ? 0 : S::kScale) + (lane & 15) * (D / 16);
      const unsigned char* k_lane = static_cast<const unsigned char*>(a.k) + head * a.k_head + (load_row & 7) * a.k_slot + chunk * 16;
      const unsigned char* v_lane = static_cast<const unsigned char*>(a.v) + head * a.v_head + (load_row & 7) * a.v_slot + chunk * 16;
      const unsigned char* s_lane = reinterpret_cast<const unsigned char*>(
          lane < 16 ? args.k_scale + head * args.ks_head + (lane & 7) * args.ks_slot
                    : args.v_scale + head * args.vs_head + (lane & 7) * args.vs_slot);
      const int k_page = (int)a.k_page, k_slot = (int)a.k_slot, v_page = (int)a.v_page, v_slot = (int)a.v_slot;
      const int s_page = 2 * (int)(lane < 16 ? args.ks_page : args.vs_page), s_slot = 2 * (int)(lane < 16 ? args.ks_slot : args.vs_slot);
      const auto along = [](const unsigned char* from, int n, int stride) { return from + (int64_t)n * stride; };
      // Pages of the keys of step page_step + lane, sixteen keys or (pages of 8) either half of them; -1: none.
      int page_of[2] = {-1, -1};
      int page_left = 0;  // steps that they still cover
      uint32_t to = ring;
      const auto load = [&](int step) {
        if (step < steps) {
          if (page_left == 0) {
            page_left = 32;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const int k = (step + lane) * kStepKeys + s * 8;
              page_of[s] = -1;
              if (wide && s) continue;
              if (step + lane < steps && k < key_hi && k + (wide ? 16 : 8) > key_lo) {
                const int page = __ldg(table + ((warp_key + k) >> a.pages.page_log2));
                if (page >= 0 && page < a.pages.num_pages) page_of[s] = page;
                else bad_page = 1;
              }
            }
          }
          const int from_lane = 32 - page_left--;
          const int key = step * kStepKeys, row = lane & 15;
          // Codes of slots outside the tile's keys are whatever they are: their scales are zeros.
          const int page0 = __shfl_sync(0xffffffffu, page_of[0], from_lane), slot0 = (warp_key + key) & in_page;
          const bool ok = key + row >= key_lo && key + row < key_hi;
          if (wide && page0 >= 0) {
            const unsigned char* k = along(along(k_lane, page0, k_page), slot0, k_slot);
            const unsigned char* v = along(along(v_lane, page0, v_page), slot0, v_slot);
            if constexpr (kPasses == 1) {
              k = along(k, load_row & 8, k_slot);
              v = along(v, load_row & 8, v_slot);
            }
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
              cp_async16(to + load_at + i * kEight, along(k, 8 * i, k_slot), true);
              cp_async16(to + load_at + S::kCodes + i * kEight, along(v, 8 * i, v_slot), true);
            }
            cp_async_small<D / 16>(to + scale_to, along(along(s_lane, page0, s_page), slot0 + (row & 8), s_slot), ok);
          } else {
            // Pages of 8 slots, or none.
            const int page1 = __shfl_sync(0xffffffffu, page_of[1], from_lane), slot1 = (warp_key + key + 8) & in_page;
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
              const bool second = kPasses == 1 ? load_row >= 8 : i == 1;
              const int page = second ? page1 : page0, slot = second ? slot1 : slot0, there = max(page, 0);
              cp_async16(to + load_at + i * kEight, along(along(k_lane, there, k_page), slot, k_slot), page >= 0);
              cp_async16(to + load_at + S::kCodes + i * kEight, along(along(v_lane, there, v_page), slot, v_slot), page >= 0);
            }
            const int page = row & 8 ? page1 : page0, slot = row & 8 ? slot1 : slot0;
            cp_async_small<D / 16>(to + scale_to, along(along(s_lane, max(page, 0), s_page), slot, s_slot), page >= 0 && ok);
          }
          to += kStage;
          if (to == ring_end) to = ring;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int s = 0; s < kRing - 1; ++s) load(s);
      uint32_t here = ring;
      for (int step = 0; step < steps; ++step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
        __syncwarp();
        load(step + kRing - 1);
        products(here, step * kStepKeys);
        here += kStage;
        if (here == ring_end) here = ring;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();

    // The sums of the warps that share a head's keys, joined.
    float* joined = reinterpret_cast<float*>(smem) + warp * kRows * D;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float l = sum[n][x];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int row = 8 * n + 2 * p + x;
        const float top = from[n][x] + kShift;
        if (j == 0) {
          stat[warp][row][0] = top == kNoTop ? -INFINITY : top;
          stat[warp][row][1] = l * 0x1p-8f;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float down = power_of_two(119 - (int)(__float_as_uint(inv_scale[warp][n][g][2 * p + x]) >> 23));  // 2^(sigma - 8)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int channel = 8 * (j % 4 * G + g) + 4 * t + j / 4;
            joined[row * D + channel] = (acc[n][g][t][x] - eights[n][g][x]) * 0x1p24f * down;
            joined[row * D + channel + 2] = (acc[n][g][t][2 + x] - eights[n][g][2 + x]) * 0x1p20f * down;
          }
        }
      }
    __syncthreads();
    const bool whole = b0 == 0 && b1 == it.blocks;
    const int64_t slot = 2 * cta + (b0 == 0 ? 1 : 0);
    if (threadIdx.x == 0 && bad_page) atomicOr(&g_device_error, kDeviceErrorIndex);
    // A row of a head a warp, kCols columns a lane.
    constexpr int kCols = D / 32;
    const int heads = min(HEADS, a.kv_heads - it.head);
    for (int i = warp; i < HEADS * rows; i += kDecodeWarps) {
      const int hh = i % HEADS, row = i / HEADS;
      if (hh >= heads) continue;
      float m = -INFINITY;
#pragma unroll
      for (int v = 0; v < kSplit; ++v) m = fmaxf(m, stat[v * HEADS + hh][row][0]);
      const float top_of = m == -INFINITY ? 0.f : m;
      float o[kCols] = {}, l = 0.f;
#pragma unroll
      for (int v = 0; v < kSplit; ++v) {
        const float f = exp2_approx(stat[v * HEADS + hh][row][0] - top_of);
        const float* from_warp = reinterpret_cast<const float*>(smem) + ((v * HEADS + hh) * kRows + row) * D + lane * kCols;
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[c] += f * from_warp[c];
        l += f * stat[v * HEADS + hh][row][1];
      }
      if (bad_page) {
        l = __int_as_float(0x7fc00000);
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[c] = l;
      }
      if (whole) {
        const int token = token_of(row), h = (it.head + hh) * a.group + (row0 + row - token * a.group);
        T* out = static_cast<T*>(a.out) + (q.first + token) * a.out_n + h * a.out_h + lane * kCols;
#pragma unroll
        for (int c = 0; c < kCols; ++c) out[c] = from_float<T>(l == 0.f ? 0.f : o[c] / l);
        if (a.lse && lane == 0) a.lse[(int64_t)(q.first + token) * a.heads + h] = (m + log2f(l)) * 0.6931471805599453f;
      } else {
        const int64_t to = (slot * HEADS + hh) * kRows + row;
#pragma unroll
        for (int c = 0; c < kCols; ++c) part_out[to * D + lane * kCols + c] = o[c];
        if (lane == 0) {
          part_stat[to * 2] = m;
          part_stat[to * 2 + 1] = l;
        }
      }
    }
    if (threadIdx.x == 0 && b0 == 0 && b1 < it.blocks) parts[cta] = part_of(run, it);
    unit = it.item_start + it.u1;
    if constexpr (TMA) fence_proxy_async_smem();  // the next copies come to lie where the sums were
    __syncthreads();
  }
}

template <typename T, int D, int NT, int HEADS, bool TMA>
cudaError_t launch(Int4Args args, const Maps& maps, cudaStream_t stream) {
  AttentionArgs& a = args.a;
  constexpr int kRows = 8 * NT;
  a.whole = a.max_keys <= kWholeKeys;
  constexpr size_t smem = room_of<D, NT>() + kDecodeWarps * kQueryBytes<D, NT>;
  const void* fn = reinterpret_cast<const void*>(&paged_int4_decode_kernel<T, D, NT, HEADS, TMA>);
  cudaError_t err = allow_shared_memory(fn, smem);
  if (err != cudaSuccess) return err;
  // Never more CTAs than there can be units.
  const int64_t tiles = (int64_t)a.tokens * a.group / kRows + (a.tokens < a.pages.batch + 2 ? a.tokens : a.pages.batch + 2);
  const int64_t blocks = a.whole ? 1 : a.max_keys / kBlockKeys + 1;
  int dev = 0, sms = 0;
  if ((err = cudaGetDevice(&dev)) != cudaSuccess ||
      (err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess)
    return err;
  const int64_t want = tiles * ((a.kv_heads + HEADS - 1) / HEADS) * blocks, most = (int64_t)sms * kCtasPerSm;
  const int64_t grid = persistent_grid(fn, smem, want < most ? want : most, kDecodeThreads);
  if (grid <= 0) return cudaErrorInvalidConfiguration;
  err = launch_kernel(paged_int4_decode_kernel<T, D, NT, HEADS, TMA>, dim3((unsigned)grid), dim3(kDecodeThreads), smem, stream,
                      args, maps);
  if (err != cudaSuccess || a.whole) return err;
  const unsigned rows = a.pages.cu_seqlens || a.group > kRows ? kRows : a.group;  // rows a tile can have
  const int64_t items = tiles * ((a.kv_heads + HEADS - 1) / HEADS);  // CTAs that can have begun one
  // By how many CTAs there are to an item, which is how many parts it may have (lengths are not known here, and with few items
  // the grid goes by the page table's width). Wide CTAs, of which an SM holds one; a small CTA a row; a warp a row, in us
  // with each form, 32/8 heads x 128, tables of 131,072 keys: 1 request of 1,000 keys 12.6, 12.6, 12.9; of 16,000 20.8, 25.6, 29.8;
  // of 131,071 54, 64, 72; 8 of 1,000 19.1, 17.1, 17.3; 8 of 8,000 34.4, 33.9, 33.6; 12 of 1,000 21.3, 18.4, 18.1; 16 of 8,000
  // 58.5, 53.9, 54.5; 32 of 4,000 67.8, 57.4, 56.8; 64 of 1,000 58.4, 37.6, 35.6.
  const dim3 joins((unsigned)(items < grid ? items : grid), rows, HEADS);
  if (items * 16 < grid)
    return launch_following(paged_join_kernel<T, D, kRows, false, HEADS, 16, 8, true>, joins, dim3(512), stream, a, grid);
  if (items * 8 < grid)
    return launch_following(paged_join_kernel<T, D, kRows, false, HEADS, 4, 4, true>, joins, dim3(128), stream, a, grid);
  return launch_following(paged_join_kernel<T, D, kRows, false, HEADS, 4, 8, true, 1>, dim3(joins.x, (rows + 3) / 4, HEADS),
                          dim3(128), stream, a, grid);
}

// The maps of a cache that the copies of HEADS heads can take: pages of a step's keys, a multiple of the heads, scales
// contiguous along the heads or along the slots, and what tensor maps want of strides. With scales [slot][head] that
// leaves multiples of four heads, and of two at D = 128; with [head][slot] any number but 3, 7, 11, ...
template <int HEADS>
bool make_maps(const Int4Args& args, int D, Maps* maps) {
  constexpr uint32_t kStepKeys = kWarpKeys * kDecodeWarps / HEADS;
  const AttentionArgs& a = args.a;
  const uint64_t slots = (uint64_t)1 << a.pages.page_log2, heads = (uint64_t)a.kv_heads, pages = (uint64_t)a.pages.num_pages;
  if (slots < kStepKeys || heads % HEADS || pages == 0) return false;
  const int G = D / 32;
  const bool by_slot = args.ks_slot == G && args.vs_slot == G, by_head = !(HEADS == 1 && by_slot) && args.ks_head == G && args.vs_head == G;
  if (!by_head && !by_slot) return false;
  maps->scales_by_slot = !by_head;
  // Copies are of whole 16 bytes, and so are the steps from one to the next.
  const auto whole16 = [](int64_t elements) { return (2 * elements & 15) == 0; };
  const auto along = [&](int64_t slot, int64_t head) { return by_head ? slot : heads > 1 ? head : 64; };  // (one head: no step)
  if (!whole16((by_head ? HEADS : kStepKeys) * G) || !whole16(along(args.ks_slot, args.ks_head)) ||
      !whole16(along(args.vs_slot, args.vs_head)) || (pages > 1 && (!whole16(args.ks_page) || !whole16(args.vs_page))) ||
      ((reinterpret_cast<uintptr_t>(args.k_scale) | reinterpret_cast<uintptr_t>(args.v_scale)) & 15))
    return false;
  const auto positive = [](int64_t bytes) { return bytes > 0; };
  const auto codes = [&](CUtensorMap* map, const void* base, int64_t slot, int64_t head, int64_t page) {
    const uint64_t dims[4] = {(uint64_t)D / 2, slots, heads, pages};
    const uint64_t strides[3] = {(uint64_t)slot, (uint64_t)head, pages > 1 ? (uint64_t)page : 128};
    const uint32_t box[4] = {(uint32_t)D / 2, kStepKeys, HEADS, 1};
    return positive(slot) && positive(head) && (pages == 1 || positive(page)) &&
           encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, box,
                             D == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
  };
  const auto scales = [&](CUtensorMap* map, const void* base, int64_t slot, int64_t head, int64_t page) {
    const uint64_t dims[3] = {(by_head ? heads : slots) * G, by_head ? slots : heads, pages};
    const uint64_t strides[2] = {(uint64_t)(2 * along(slot, head)), pages > 1 ? (uint64_t)(2 * page) : 128};
    const uint32_t box[3] = {(by_head ? HEADS : kStepKeys) * G, by_head ? kStepKeys : HEADS, 1};
    return positive(along(slot, head)) && (pages == 1 || positive(page)) &&
           encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
  };
  return codes(&maps->k, a.k, a.k_slot, a.k_head, a.k_page) && codes(&maps->v, a.v, a.v_slot, a.v_head, a.v_page) &&
         scales(&maps->k_scale, args.k_scale, args.ks_slot, args.ks_head, args.ks_page) &&
         scales(&maps->v_scale, args.v_scale, args.vs_slot, args.vs_head, args.vs_page);
}

// Copies of four heads at a time want pages of 16 slots, those of two or one 32 and 64: a step of
// the CTA's four warps is in one page. Key heads of a CTA: a cache line holds the scales of several heads' slots, and is fetched
// once where one CTA reads them together. Four at a time, two, or one where most of four would idle.
template <typename T, int D, int NT>
cudaError_t launch_heads(const Int4Args& args, cudaStream_t stream) {
  const int heads = args.a.kv_heads;
  Maps maps{};
  if (heads % 4 == 0 || heads % 4 == 3)
    return make_maps<4>(args, D, &maps) ? launch<T, D, NT, 4, true>(args, maps, stream) : launch<T, D, NT, 4, false>(args, maps, stream);
  if (heads % 2 == 0)
    return make_maps<2>(args, D, &maps) ? launch<T, D, NT, 2, true>(args, maps, stream) : launch<T, D, NT, 2, false>(args, maps, stream);
  return make_maps<1>(args, D, &maps) ? launch<T, D, NT, 1, true>(args, maps, stream) : launch<T, D, NT, 1, false>(args, maps, stream);
}

template <typename T, int D>
cudaError_t launch_rows(const Int4Args& args, cudaStream_t stream) {
  // Tiles of 8 rows where the requests have no more a key head on average, else of 16.
  return (int64_t)args.a.tokens * args.a.group <= 8 * (int64_t)args.a.pages.batch ? launch_heads<T, D, 1>(args, stream)
                                                                                  : launch_heads<T, D, 2>(args, stream);
}

}  // namespace

size_t paged_int4_decode_workspace(int D, int sms) {
  return (size_t)sms * kCtasPerSm * (2 * 4 * 16 * (size_t)(D + 2) * sizeof(float) + sizeof(Part));
}

cudaError_t launch_paged_int4_decode(const AttentionArgs& a, const flash_prologue_scales& s, int dtype, int D,
                                     cudaStream_t stream) {
  Int4Args args{};
  args.a = a;
  args.k_scale = static_cast<const uint16_t*>(s.k);
  args.v_scale = static_cast<const uint16_t*>(s.v);
  args.ks_page = s.k_page;
  args.ks_slot = s.k_slot;
  args.ks_head = s.k_head;
  args.vs_page = s.v_page;
  args.vs_slot = s.v_slot;
  args.vs_head = s.v_head;
  if (D == 64) return dtype == 0 ? launch_rows<__nv_bfloat16, 64>(args, stream) : launch_rows<__half, 64>(args, stream);
  return dtype == 0 ? launch_rows<__nv_bfloat16, 128>(args, stream) : launch_rows<__half, 128>(args, stream);
}

cudaError_t read_paged_int4_decode_device_error(int* value, bool reset) {
  cudaError_t err = cudaMemcpyFromSymbol(value, g_device_error, sizeof(int));
  if (err != cudaSuccess || !reset) return err;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
}

}  // namespace flash_prologue
