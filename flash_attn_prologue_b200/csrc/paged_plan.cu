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
// Entries below 0 in an ended request's row are no pages (a step ran out of them) and stay
// out. The CTAs of a cluster look through the returned entries together; where they find such
// entries, how many and the first of each row go to all of them, the pages returned are
// counted anew, and one behind a row's first such entry is found by a walk.
//
// Bound by latency: 256 requests move 40 KB in 9.1 us, a step of 60,000 prompt tokens 1 MB in 8.4 us: reading the
// lengths, the sums, a search in them and dependent reads of the table, one after the other. 3 us of both are the look
// through the returned entries (each CTA for itself, without clusters: 9.8 and 8.5 us; 256 requests that all end with 512
// pages each 27 us instead of 19, 8,192 with 128 pages 196 instead of 54).
#include <cooperative_groups.h>

#include "../../include/flash_prologue.h"
#include "gqa_rows.cuh"

static_assert(sizeof(flash_prologue_plan_args) == 144, "argument struct layout");

namespace flash_prologue {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanFlight = 8;       // entries that a lane has under way
constexpr int kPlanCluster = 8;      // CTAs that look through the returned entries together
constexpr int kMostRequests = 8192;  // five numbers each in shared memory
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

// Running sums over the requests of S values each: sums[s * (batch + 1) + r] is the sum in front of request r, all[s]
// that of all. values(r, mine) gives a request's, one request a thread at a time.
template <int S, class F>
__device__ __forceinline__ void running_sums(int batch, int* sums, int (*warp_sums)[kPlanThreads / 32], int (&all_of)[S],
                                             F values) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 0; s < S; ++s) all_of[s] = 0;
  for (int r0 = 0; r0 < batch; r0 += kPlanThreads) {
    const int r = r0 + threadIdx.x;
    int upto[S] = {};
    if (r < batch) values(r, upto);
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto[s], o);
        if (lane >= o) upto[s] = sum_of(upto[s], v);
      }
      if (lane == 31) warp_sums[s][warp] = upto[s];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; ++s) {
      // Every warp adds up the warps' sums for itself.
      int all = warp_sums[s][lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, all, o);
        if (lane >= o) all = sum_of(all, v);
      }
      const int in_front = warp ? __shfl_sync(0xffffffffu, all, warp - 1) : 0;
      const int start = sum_of(all_of[s], in_front);
      if (r < batch) sums[s * (batch + 1) + r + 1] = sum_of(start, upto[s]);
      all_of[s] = sum_of(all_of[s], __shfl_sync(0xffffffffu, all, 31));
    }
    __syncthreads();
  }
  if (threadIdx.x < S) sums[threadIdx.x * (batch + 1)] = 0;
  __syncthreads();
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const flash_prologue_plan_args a, int page_log2) {
  namespace cg = cooperative_groups;
  extern __shared__ int shared[];  // [5][batch + 1]
  __shared__ int warp_sums[3][kPlanThreads / 32];
  __shared__ int some_missing;  // an ended request's row has entries that are no pages
  const cg::cluster_group cluster = cg::this_cluster();
  const int batch = (int)a.batch, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int *const tokens_of = shared, *const returned_of = tokens_of + batch + 1, *const wanted_of = returned_of + batch + 1;
  // Of an ended request's returned entries: how many are no pages, the first of those.
  int *const missing = wanted_of + batch + 1, *const first_missing = missing + batch + 1;
  for (int r = threadIdx.x; r < batch; r += kPlanThreads) {
    missing[r] = 0;
    first_missing[r] = kMostTokens;
  }
  if (threadIdx.x == 0) some_missing = 0;
  cluster.barrier_arrive();
  const bool first_cta = blockIdx.x == 0;
  bool bad = false;
  int all[3];
  running_sums<3>(batch, shared, warp_sums, all, [&](int r, int (&mine)[3]) {
    const Growth g = growth_of(a, page_log2, r);
    bad |= g.bad;
    mine[0] = g.news;
    mine[1] = g.ended ? g.held - g.keep : 0;
    mine[2] = max(g.wanted - g.held, 0);
    if (first_cta) a.seq_lens_out[r] = g.total;
  });
  cluster.barrier_wait();  // their counts are zeros

  const auto kept = [&](int r) { return a.keep ? min(max(__ldg(a.keep + r), 0), (int)a.max_pages) : 0; };
  const auto row_of = [&](int r) { return a.page_table + r * a.table_stride; };
  {
    const int warps = cluster.num_blocks() * (kPlanThreads / 32), index = cluster.block_rank() * (kPlanThreads / 32) + warp;
    const int end = (int)((int64_t)all[1] * (index + 1) / warps);
    int i = (int)((int64_t)all[1] * index / warps), r = i < end ? request_at_sum(returned_of, batch, i) : 0;
    while (i < end) {
      if (i >= returned_of[r + 1]) r = request_at_sum(returned_of, batch, i);  // the next request returns none
      const int stop = min(end, returned_of[r + 1]), start = returned_of[r];
      const int32_t* from = row_of(r) + kept(r);
      int count = 0, first = kMostTokens;
      for (int e0 = i + lane; e0 < stop; e0 += 32 * kPlanFlight) {
        int entry[kPlanFlight];
#pragma unroll
        for (int f = 0; f < kPlanFlight; ++f) entry[f] = e0 + 32 * f < stop ? __ldcg(from + (e0 + 32 * f - start)) : 0;
#pragma unroll
        for (int f = 0; f < kPlanFlight; ++f)
          if (entry[f] < 0) {
            ++count;
            first = min(first, e0 + 32 * f - start);
          }
      }
      if (__any_sync(0xffffffffu, count)) {
        count = __reduce_add_sync(0xffffffffu, count);
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane < cluster.num_blocks()) {
          atomicAdd(cluster.map_shared_rank(missing, lane) + r, count);
          atomicMin(cluster.map_shared_rank(first_missing, lane) + r, first);
          *cluster.map_shared_rank(&some_missing, lane) = 1;
        }
      }
      i = stop;
      ++r;
    }
  }
  cluster.sync();
  if (some_missing) {
    int returned[1];
    running_sums<1>(batch, returned_of, warp_sums, returned, [&](int r, int (&mine)[1]) {
      const Growth g = growth_of(a, page_log2, r);
      mine[0] = g.ended ? max(g.held - g.keep - missing[r], 0) : 0;
    });
    all[1] = returned[0];
  }

  const int size = (int)a.free_size, counted = __ldg(a.free_count), count = min(max(counted, 0), size);
  const int returned = all[1], wanted = all[2];
  const int available = count + min(returned, size - count);  // what does not fit is lost
  bad |= counted < 0 || counted > size || returned > size - count || wanted > available || all[0] > a.tokens;
  // The stack's entry i below `available`.
  const auto stack_at = [&](int i) {
    if (i < count) return __ldcg(a.free_pages + i);
    int k = i - count;
    const int r = request_at_sum(returned_of, batch, k);
    k -= returned_of[r];
    const int32_t* row = row_of(r) + kept(r);
    int c = first_missing[r];
    if (k < c) return __ldcg(row + k);
    // Behind the row's first entry that is no page: the (k - c)-th page from there.
    k -= c;
    const int end = growth_of(a, page_log2, r).held - kept(r);
    int page = -1;
#pragma unroll 8
    for (; c < end; ++c) {
      const int entry = __ldcg(row + c);
      if (entry >= 0 && k-- == 0) page = entry;
    }
    return page;
  };
  const auto new_page = [&](int i) { return i < available ? stack_at(available - 1 - i) : -1; };
  const int thread = blockIdx.x * kPlanThreads + threadIdx.x, threads = gridDim.x * kPlanThreads;
  if (first_cta) {
    for (int r = threadIdx.x; r <= batch; r += kPlanThreads) a.cu_seqlens[r] = tokens_of[r];
    if (threadIdx.x == 0) *a.free_count_out = available - min(wanted, available);
  }
  for (int i = thread; i < available - count; i += threads) a.free_pages[count + i] = stack_at(count + i);
  for (int i = thread; i < wanted; i += threads) {
    const int r = request_at_sum(wanted_of, batch, i);
    const Growth g = growth_of(a, page_log2, r);
    row_of(r)[g.held + i - wanted_of[r]] = new_page(i);
  }
  for (int t = thread; t < a.tokens; t += threads) {
    int request = -1, position = 0;
    int64_t slot = -1;
    if (t < all[0]) {
      request = request_at_sum(tokens_of, batch, t);
      const Growth g = growth_of(a, page_log2, request);
      position = g.total - g.news + t - tokens_of[request];
      const int column = position >> page_log2;
      int page = -1;
      if (column < g.held) page = __ldcg(row_of(request) + column);
      else if (column < g.wanted) page = new_page(wanted_of[request] + column - g.held);
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
  // A CTA for each of its threads' tokens, and for pages that ended requests may return; in whole clusters.
  int64_t grid = (a->tokens + kPlanThreads - 1) / kPlanThreads;
  const int64_t pages = (a->batch * a->max_pages + 16 * kPlanThreads - 1) / (16 * kPlanThreads);
  grid = grid > pages ? grid : pages;
  const int cluster = grid > 1 ? kPlanCluster : 1;
  grid = grid < 1 ? 1 : grid > 128 ? 128 : (grid + cluster - 1) / cluster * cluster;
  const size_t smem = 5 * (size_t)(a->batch + 1) * sizeof(int);
  const void* fn = reinterpret_cast<const void*>(&paged_plan_kernel);
  if (smem > 48 * 1024 && allow_shared_memory(fn, 5 * (size_t)(kMostRequests + 1) * sizeof(int)) != cudaSuccess)
    return FLASH_PROLOGUE_ERR_CUDA;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)grid);
  config.blockDim = dim3(kPlanThreads);
  config.dynamicSmemBytes = smem;
  config.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attribute = {};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = cluster;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, paged_plan_kernel, *a, page_log2) == cudaSuccess ? FLASH_PROLOGUE_OK
                                                                                       : FLASH_PROLOGUE_ERR_CUDA;
}
