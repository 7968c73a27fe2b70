// Host-side arguments of the grouped-query prologue kernels (gqa_fwd.cu,
// gqa_bwd.cu): rows of Q with Hq heads, rows of K (and V) with Hk heads, the
// rotation picked per token by a position.
#pragma once

#include "../../include/flash_prologue.h"
#include "prologue_host.h"
#include "tma_util.cuh"

namespace flash_prologue {

// Device error word value: an index read from device memory (a position, a
// page, a length) was out of range; the rows it concerns were not read or written.
constexpr int kDeviceErrorIndex = 2;
constexpr int64_t kMaxGqaHeads = 512;
// Grid bound of the backward, hence its workspace: one partial row a CTA.
constexpr int kGqaBwdMaxCtasPerSm = 2;

// How the 32 / L row slots of a warp (L = D / 16 lanes a row) map to rows: HS
// heads of TP consecutive tokens, HS * TP = 32 / L. A warp's token group walks
// `iters[t]` head blocks of tensor t; `slices` warps share a token group when
// there are too few groups to fill the GPU.
struct RowsPlan {
  int log2_hs;
  int iters[3];       // head blocks of q, k, v (v: 0 without a cache)
  int slices;
  int per_slice;      // head blocks of one slice
  int64_t groups;     // token groups
};

struct GqaTables {
  const float* sin;
  const float* cos;
  int64_t sin_n, sin_j, cos_n, cos_j;  // element strides
  int64_t rows;                        // positions are in [0, rows)
  const void* positions;               // null: row n of the tables; else int32 / int64 [b, n]
  int64_t pos_b, pos_n;
  int pos_is64;
};

struct PagedTarget {
  const int32_t* page_table;  // [batch, max_pages]
  const int32_t* seq_lens;    // [batch], new tokens included
  const int32_t* cu_seqlens;  // [batch + 1], null: token i is request i's
  int64_t table_stride;
  int64_t max_pages, num_pages;
  int batch;
  int page_log2;
};

struct GqaFwdArgs {
  const void* x[3];    // q, k, v
  void* y[3];          // q_out, then k_out or the two caches
  RowStrides sx[3];
  RowStrides sy[3];    // of a cache: b = page, h = head, n = slot
  const float* w;      // [2, D] or null (rotation only)
  const float* scales; // [Hq] or null
  GqaTables tab;
  bool append;         // K and V go to the pages of `paged`, else to dense outputs
  PagedTarget paged;
  int64_t B, N;
  int H[3];
  float eps;
  RowsPlan p;
};

struct GqaBwdArgs {
  const void* x[2];
  const void* gy[2];
  void* dx[2];
  RowStrides sx[2], sgy[2], sdx[2];
  const float* w;
  const float* scales;
  GqaTables tab;
  float* partials;     // [grid, 2 * D + Hq]
  int64_t B, N;
  int H[2];
  float eps;
  RowsPlan p;
};

// A usable peer group for rows of `cols` sums and an epoch of at least 1.
inline bool valid_peers(const flash_prologue_peers* peers, int64_t epoch, int64_t cols) {
  return epoch >= 1 && epoch <= UINT32_MAX && peers->world >= 1 && peers->world <= FLASH_PROLOGUE_MAX_PEERS &&
         peers->rank >= 0 && peers->rank < peers->world && peers->max_cols % 32 == 0 && peers->max_cols >= cols &&
         peers->wait_ms >= 0 && peers->wait_ms <= 60000;
}

RowsPlan plan_rows(int64_t tokens, int Hq, int Hk, int Hv, int D, bool heads_inner, int64_t want_warps);
cudaError_t launch_gqa_fwd(const GqaFwdArgs& a, int dtype, int D, bool vec, cudaStream_t stream);
int64_t gqa_bwd_grid(const RowsPlan& p, int Hq, int D, int dtype, bool vec);
cudaError_t launch_gqa_bwd(const GqaBwdArgs& a, float* dw, float* ds, int dtype, int D, bool vec,
                           const BwdReduce& red, cudaStream_t stream);

// Copies of 16 bytes that a lane makes into shared memory for itself.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  const int bytes = ok ? 16 : 0;  // 0: the 16 bytes are filled with zeros, src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rotation row of token (b, n); -1 (and the error word) when it is out of range.
__device__ __forceinline__ int64_t rotation_row(const GqaTables& t, int64_t b, int64_t n) {
  int64_t pos = n;
  if (t.positions) {
    const int64_t i = b * t.pos_b + n * t.pos_n;
    pos = t.pos_is64 ? static_cast<const int64_t*>(t.positions)[i]
                     : (int64_t) static_cast<const int32_t*>(t.positions)[i];
  }
  if (pos < 0 || pos >= t.rows) {
    atomicOr(&g_device_error, kDeviceErrorIndex);
    return -1;
  }
  return pos;
}

template <typename T>
__device__ __forceinline__ void chunk_zero(Chunk<T>& c) {
#pragma unroll
  for (int i = 0; i < Chunk<T>::kWords; ++i) c.w[i] = 0;
}

// Columns of a half row that lane c of the row's L owns: 8 of them, in 16-byte
// pieces that lie next to the other lanes' (one piece of a 16-bit type, two of
// FP32: with 32 bytes a lane every access would touch twice the sectors).
template <typename T, int D>
struct Columns {
  static constexpr int kPieces = sizeof(T) == 4 ? 2 : 1;
  static constexpr int kPer = kChunk / kPieces;           // columns of a piece
  static constexpr int kApart = D / 2 / kPieces;          // columns from one piece to the next
  static __device__ __forceinline__ int first(int c) { return c * kPer; }
  static __device__ __forceinline__ int of(int c, int j) { return j / kPer * kApart + c * kPer + j % kPer; }
};

// The lane's chunk of a half row; `half` points at the half's first piece of the lane.
template <typename T, int D, bool VEC>
__device__ __forceinline__ void load_chunk(Chunk<T>& x, const T* half) {
  using C = Columns<T, D>;
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < C::kPieces; ++q) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(half + q * C::kApart));
      x.w[4 * q] = v.x; x.w[4 * q + 1] = v.y; x.w[4 * q + 2] = v.z; x.w[4 * q + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) x.w[j] = reinterpret_cast<const uint32_t*>(half)[C::of(0, j)];
  } else {
    load_stream<T, false>(x, half);
  }
}
template <typename T, int D, bool VEC>
__device__ __forceinline__ void store_chunk(T* half, const Chunk<T>& x) {
  using C = Columns<T, D>;
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < C::kPieces; ++q)
      *reinterpret_cast<uint4*>(half + q * C::kApart) =
          make_uint4(x.w[4 * q], x.w[4 * q + 1], x.w[4 * q + 2], x.w[4 * q + 3]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) reinterpret_cast<uint32_t*>(half)[C::of(0, j)] = x.w[j];
  } else {
    store_stream<T, false>(half, x);
  }
}
// The lane's 8 values of an FP32 table row or parameter (`half`: as above, in floats).
template <typename T, int D, bool VEC>
__device__ __forceinline__ void load_columns(float (&v)[kChunk], const float* half, int64_t stride) {
  using C = Columns<T, D>;
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(half + C::of(0, 4 * q)));
      v[4 * q] = x.x; v[4 * q + 1] = x.y; v[4 * q + 2] = x.z; v[4 * q + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) v[j] = __ldg(half + C::of(0, j) * stride);
  }
}

// A kernel for each activation type, head dimension and access width.
#define FLASH_PROLOGUE_GQA_DIMS(T, KERNEL)                                                        \
  switch (D) {                                                                                    \
    case 32: return vec ? reinterpret_cast<const void*>(&KERNEL<T, 32, true>)                     \
                        : reinterpret_cast<const void*>(&KERNEL<T, 32, false>);                   \
    case 64: return vec ? reinterpret_cast<const void*>(&KERNEL<T, 64, true>)                     \
                        : reinterpret_cast<const void*>(&KERNEL<T, 64, false>);                   \
    case 128: return vec ? reinterpret_cast<const void*>(&KERNEL<T, 128, true>)                   \
                         : reinterpret_cast<const void*>(&KERNEL<T, 128, false>);                 \
    case 256: return vec ? reinterpret_cast<const void*>(&KERNEL<T, 256, true>)                   \
                         : reinterpret_cast<const void*>(&KERNEL<T, 256, false>);                 \
    default: return nullptr;                                                                      \
  }
#define FLASH_PROLOGUE_GQA_KERNEL(KERNEL)                                                         \
  switch (dtype) {                                                                                \
    case 0: FLASH_PROLOGUE_GQA_DIMS(__nv_bfloat16, KERNEL)                                        \
    case 1: FLASH_PROLOGUE_GQA_DIMS(__half, KERNEL)                                               \
    case 2: FLASH_PROLOGUE_GQA_DIMS(float, KERNEL)                                                \
    default: return nullptr;                                                                      \
  }

}  // namespace flash_prologue
