// What the rows of a 4-bit cache stand for, as rows of a 16-bit type.
//
// Bound by HBM, mostly by the writes: a thread takes a word (8 channels, 16 bytes
// out), so a warp reads 128 and writes 512 contiguous bytes. 203,000 rows of 128 channels (15 MB of codes
// and scales, 52 MB out) take 10.4 us (11.6 with six sets of buffers in turn), 6.4 TB/s with part of both in L2.
#include "../../include/flash_prologue.h"
#include "gqa_rows.cuh"

namespace flash_prologue {
namespace {

constexpr int kUnpackThreads = 256;
constexpr int kFlight = 4;  // words of a thread

template <typename T, int D>
__global__ void __launch_bounds__(kUnpackThreads) unpack_int4_kernel(const uint32_t* __restrict__ codes,
                                                                     const uint16_t* __restrict__ scales,
                                                                     uint4* __restrict__ out, int64_t words) {
  constexpr int kWords = D / 8, kGroups = D / 32;
  const int64_t first = (int64_t)blockIdx.x * kUnpackThreads * kFlight + threadIdx.x;
  uint32_t w[kFlight];
  float s[kFlight];
#pragma unroll
  for (int f = 0; f < kFlight; ++f) {
    const int64_t i = first + f * kUnpackThreads;
    if (i < words) {
      w[f] = __ldcs(codes + i);
      s[f] = __uint_as_float((uint32_t)__ldg(scales + i / kWords * kGroups + i % kGroups) << 16);
    }
  }
#pragma unroll
  for (int f = 0; f < kFlight; ++f) {
    const int64_t i = first + f * kUnpackThreads;
    if (i >= words) return;
    Chunk<T> c;
    float v[kChunk];
#pragma unroll
    for (int p = 0; p < kPairs; ++p) {
      v[2 * p] = s[f] * (float)((int)(w[f] >> (4 * p) & 15) - 8);
      v[2 * p + 1] = s[f] * (float)((int)(w[f] >> (16 + 4 * p) & 15) - 8);
    }
    chunk_set(c, v);
    __stcs(out + i, make_uint4(c.w[0], c.w[1], c.w[2], c.w[3]));
  }
}

template <typename T, int D>
cudaError_t launch(const void* codes, const void* scales, void* out, int64_t rows, cudaStream_t stream) {
  const int64_t words = rows * (D / 8), each = kUnpackThreads * kFlight;
  return launch_kernel(unpack_int4_kernel<T, D>, dim3((unsigned)((words + each - 1) / each)), dim3(kUnpackThreads), 0,
                       stream, static_cast<const uint32_t*>(codes), static_cast<const uint16_t*>(scales),
                       static_cast<uint4*>(out), words);
}

}  // namespace
}  // namespace flash_prologue

using namespace flash_prologue;

extern "C" int flash_prologue_unpack_int4(const void* codes, const void* scales, void* out, int64_t rows, int64_t D,
                                          int64_t dtype, void* stream) {
  if (rows < 0) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if ((D != 64 && D != 128) || (dtype != FLASH_PROLOGUE_BF16 && dtype != FLASH_PROLOGUE_FP16) ||
      rows >= (int64_t(1) << 36))
    return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  if (rows == 0) return FLASH_PROLOGUE_OK;
  if (!codes || !scales || !out) return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(out)) & 15)
    return FLASH_PROLOGUE_ERR_ALIGNMENT;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  if (D == 64)
    err = dtype == 0 ? launch<__nv_bfloat16, 64>(codes, scales, out, rows, s) : launch<__half, 64>(codes, scales, out, rows, s);
  else
    err = dtype == 0 ? launch<__nv_bfloat16, 128>(codes, scales, out, rows, s)
                     : launch<__half, 128>(codes, scales, out, rows, s);
  return err == cudaSuccess ? FLASH_PROLOGUE_OK : FLASH_PROLOGUE_ERR_CUDA;
}
