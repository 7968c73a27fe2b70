// The page tables of a serving step, built on the GPU from the requests' lengths:
// ended requests' pages go on top of a stack of free ones, requests that grow take
// new ones from it, and every new token gets its request, position and slot.
//
// With held_r = ceil(len_r / page) and wanted_r = ceil((len_r + new_r) / page) the
// stack is free[0 .. count) and behind it the pages of the ended requests in
// order; the i-th new page, counted over the requests in order, is its entry
// available - 1 - i. All of it follows from three running sums over the requests
// (new tokens, pages returned, pages wanted), and nothing that the call reads is
// written by it: entries of the table are read below held_r and written from
// there on, the stack is read below `count` and written from there on (an entry
// above it is read where it comes from, the ended request's row of the table). So
// every CTA computes the sums for itself and does its share of the tokens and
// pages, in one launch without a word between CTAs.
//
// Bound by latency: 256 requests move 40 KB, a step of 60,000 prompt tokens 1 MB, in 6.2 us: reading the lengths,
// the sums, a search in them and a dependent read of the table, one after the other.
#include "../../include/flash_prologue.h"
#include "gqa_rows.cuh"

static_assert(sizeof(flash_prologue_plan_args) == 144, "argument struct layout");

namespace flash_prologue {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMostRequests = 8192;  // three sums each in shared memory
constexpr int kMostTokens = 1 << 30;

struct Growth {
  int held, wanted;  // pages before the step and after it
  int keep;          // pages that an ended request does not return
  int news, total;
  bool ended, bad;
};

__device__ __forceinline__ Growth growth_of(const flash_prologue_plan_args& a, int page_log2, int r) {
  Growth g;
  const int width = (int)a.max_pages, room = width << page_log2;  // below 2^30 (host)
  const int old = __ldg(a.seq_lens + r), news = __ldg(a.new_lens + r);
  g.ended = news < 0;
  const int len = min(max(old, 0), room);
  g.news = min(max(news, 0), kMostTokens);
  const int page = (1 << page_log2) - 1;
  g.held = (len + page) >> page_log2;
  g.total = g.ended ? 0 : len + g.news;  // below 2^31
  g.wanted = g.ended ? 0 : (min(g.total, room) + page) >> page_log2;
  g.keep = a.keep ? min(max(__ldg(a.keep + r), 0), g.held) : 0;
  g.bad = old < 0 || old > room || g.total > room || news > kMostTokens;
  return g;
}

// Sums end at kMostTokens, where two of them still fit 32 bits unsigned (new tokens may be 2^30 in many requests).
__device__ __forceinline__ int sum_of(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)kMostTokens); }

// The last request whose sum is at most i: sums[r] <= i < sums[r + 1].
__device__ __forceinline__ int request_at_sum(const int* sums, int batch, int i) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const flash_prologue_plan_args a, int page_log2) {
  extern __shared__ int sums[];  // [3][batch + 1]: new tokens, pages returned, pages wanted
  __shared__ int warp_sums[3][kPlanThreads / 32];
  const int batch = (int)a.batch, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* of[3] = {sums, sums + batch + 1, sums + 2 * (batch + 1)};
  const bool first_cta = blockIdx.x == 0;
  bool bad = false;
  int before[3] = {0, 0, 0};
  for (int r0 = 0; r0 < batch; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    int mine[3] = {0, 0, 0};
    if (r < batch) {
      const Growth g = growth_of(a, page_log2, r);
      bad |= g.bad;
      mine[0] = g.news;
      mine[1] = g.ended ? g.held - g.keep : 0;
      mine[2] = max(g.wanted - g.held, 0);
      if (first_cta) a.seq_lens_out[r] = g.total;
    }
    int upto[3];
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      upto[s] = mine[s];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto[s], o);
        if (lane >= o) upto[s] = sum_of(upto[s], v);
      }
      if (lane == 31) warp_sums[s][warp] = upto[s];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      // Every warp adds up the warps' sums for itself.
      int all = warp_sums[s][lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, all, o);
        if (lane >= o) all = sum_of(all, v);
      }
      const int in_front = warp ? __shfl_sync(0xffffffffu, all, warp - 1) : 0;
      const int start = sum_of(before[s], in_front);
      if (r < batch) of[s][r + 1] = sum_of(start, upto[s]);
      before[s] = sum_of(before[s], __shfl_sync(0xffffffffu, all, 31));
    }
    __syncthreads();
  }
  if (threadIdx.x < 3) of[threadIdx.x][0] = 0;
  __syncthreads();

  const int size = (int)a.free_size, counted = __ldg(a.free_count), count = min(max(counted, 0), size);
  const int returned = before[1], wanted = before[2];
  const int available = count + min(returned, size - count);  // what does not fit is lost
  bad |= counted < 0 || counted > size || returned > size - count || wanted > available || before[0] > a.tokens;
  // The stack's entry i below `available`.
  const auto stack_at = [&](int i) {
    if (i < count) return __ldcg(a.free_pages + i);
    const int k = i - count, r = request_at_sum(of[1], batch, k);
    const int first = a.keep ? min(max(__ldg(a.keep + r), 0), (int)a.max_pages) : 0;
    return __ldcg(a.page_table + r * a.table_stride + first + k - of[1][r]);
  };
  const auto new_page = [&](int i) { return i < available ? stack_at(available - 1 - i) : -1; };
  const int thread = blockIdx.x * kPlanThreads + threadIdx.x, threads = gridDim.x * kPlanThreads;
  if (first_cta) {
    for (int r = threadIdx.x; r <= batch; r += kPlanThreads) a.cu_seqlens[r] = of[0][r];
    if (threadIdx.x == 0) *a.free_count_out = available - min(wanted, available);
  }
  for (int i = thread; i < available - count; i += threads) a.free_pages[count + i] = stack_at(count + i);
  for (int i = thread; i < wanted; i += threads) {
    const int r = request_at_sum(of[2], batch, i);
    const Growth g = growth_of(a, page_log2, r);
    a.page_table[r * a.table_stride + g.held + i - of[2][r]] = new_page(i);
  }
  for (int t = thread; t < a.tokens; t += threads) {
    int request = -1, position = 0;
    int64_t slot = -1;
    if (t < before[0]) {
      request = request_at_sum(of[0], batch, t);
      const Growth g = growth_of(a, page_log2, request);
      position = g.total - g.news + t - of[0][request];
      const int column = position >> page_log2;
      int page = -1;
      if (column < g.held) page = __ldcg(a.page_table + request * a.table_stride + column);
      else if (column < g.wanted) page = new_page(of[2][request] + column - g.held);
      if (page >= 0) slot = ((int64_t)page << page_log2) + (position & ((1 << page_log2) - 1));
      else bad = true;
    }
    a.requests[t] = request;
    a.positions[t] = position;
    a.slots[t] = slot;
  }
  if (bad) atomicOr(&g_device_error, kDeviceErrorIndex);
}

}  // namespace

cudaError_t read_paged_plan_device_error(int* value, bool reset) {
  cudaError_t err = cudaMemcpyFromSymbol(value, g_device_error, sizeof(int));
  if (err != cudaSuccess || !reset) return err;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
}

}  // namespace flash_prologue

using namespace flash_prologue;

extern "C" int flash_prologue_plan_paged_step(const flash_prologue_plan_args* a, void* stream) {
  if (!a || a->batch < 0 || a->tokens < 0 || a->max_pages < 0 || a->free_size < 0 || a->page_size < 8 ||
      (a->page_size & (a->page_size - 1)))
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (a->batch > kMostRequests || a->page_size > (1 << 20) || a->max_pages >= kMostTokens / a->page_size ||
      a->tokens >= kMostTokens || a->free_size >= kMostTokens)
    return FLASH_PROLOGUE_ERR_UNSUPPORTED;
  if (!a->cu_seqlens || !a->free_count || !a->free_count_out || (a->free_size > 0 && !a->free_pages) ||
      (a->batch > 0 && (!a->seq_lens || !a->new_lens || !a->seq_lens_out || (a->max_pages > 0 && !a->page_table))) ||
      (a->tokens > 0 && (!a->positions || !a->slots || !a->requests)))
    return FLASH_PROLOGUE_ERR_INVALID_ARGUMENT;
  if (a->batch > 1 && a->max_pages > 0 && a->table_stride < a->max_pages) return FLASH_PROLOGUE_ERR_EXPANDED;
  int page_log2 = 0;
  while ((int64_t(1) << page_log2) < a->page_size) ++page_log2;
  // A CTA for each of its threads' tokens, and for pages that ended requests may return.
  int64_t grid = (a->tokens + kPlanThreads - 1) / kPlanThreads;
  const int64_t pages = (a->batch * a->max_pages + 16 * kPlanThreads - 1) / (16 * kPlanThreads);
  grid = grid > pages ? grid : pages;
  grid = grid < 1 ? 1 : grid > 128 ? 128 : grid;
  const size_t smem = 3 * (size_t)(a->batch + 1) * sizeof(int);
  const void* fn = reinterpret_cast<const void*>(&paged_plan_kernel);
  if (smem > 48 * 1024 && allow_shared_memory(fn, 3 * (size_t)(kMostRequests + 1) * sizeof(int)) != cudaSuccess)
    return FLASH_PROLOGUE_ERR_CUDA;
  flash_prologue_plan_args args = *a;
  void* params[] = {&args, &page_log2};
  return cudaLaunchKernel(fn, dim3((unsigned)grid), dim3(kPlanThreads), params, smem,
                          static_cast<cudaStream_t>(stream)) == cudaSuccess
             ? FLASH_PROLOGUE_OK
             : FLASH_PROLOGUE_ERR_CUDA;
}
