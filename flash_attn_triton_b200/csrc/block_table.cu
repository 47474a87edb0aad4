// Pages, slots and cu_seqlens of a serving step, from the lengths of its requests.
//
//   Mathematics.  have = ceil(old / page), need = ceil((old + new) / page); exclusive sums over the requests of new (cu_seqlens) and of
//   need - have (where a request's pages begin among the free ones).  Entry have + j of a row is free[first + j]; token i of request b
//   has position old + i, and its slot is page * page_size + position % page_size with the page from the row, or from the
//   free list where it is a new one, so that no token waits for the table.
//   Bound.  Launch and latency: 8 bytes a token, a page and a request, a few us at any size that a step has.  So it is one launch: every
//   CTA sums all requests itself (256 threads, a stretch of requests each; 8 bytes a request out of L2) and then writes its share of the
//   slots, the pages and the sums, each of them an even range of numbers, found again by bisection over the 256 partial sums.
//   A long prompt among short ones is shared by all CTAs that way.  Measured: 8 requests 6.8 us (launch, two reads one behind the other),
//   2048 prompts of 1 to 2048 tokens, 2.1 million slots, 17 us of a call.
#include "check_words.h"
#include "cache_dev.cuh"

namespace fa {

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 4;          // slots of a thread at a time

struct Sums {
  int64_t tokens, pages;
};

// Exclusive sums over the CTA's threads; the totals to *all.
__device__ __forceinline__ Sums exclusive(Sums x, int tid, Sums* warps, Sums* all) {
  const int lane = tid & 31, warp = tid >> 5;
  Sums s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, s.tokens, o), b = __shfl_up_sync(0xffffffffu, s.pages, o);
    if (lane >= o) {
      s.tokens += a;
      s.pages += b;
    }
  }
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  Sums before = {0, 0}, total = {0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) before = total;
    total.tokens += warps[w].tokens;
    total.pages += warps[w].pages;
  }
  *all = total;
  return Sums{before.tokens + s.tokens - x.tokens, before.pages + s.pages - x.pages};
}

// Last i with first[i] <= x (first[0] = 0).
__device__ __forceinline__ int stretch_of(const int* first, int x) {
  int lo = 0;
#pragma unroll
  for (int step = kThreads / 2; step > 0; step >>= 1)
    if (first[lo + step] <= x) lo += step;
  return lo;
}

}  // namespace

__global__ void __launch_bounds__(kThreads) block_table_kernel(const fa_block_table_args p, int page_shift, uint32_t* host) {
  __shared__ Sums warps[kThreads / 32];
  __shared__ int first_token[kThreads], first_page[kThreads];
  const int tid = threadIdx.x;
  auto pages_of = [&](int64_t n) { return page_shift >= 0 ? (n + p.page_size - 1) >> page_shift : (n + p.page_size - 1) / p.page_size; };

  const int per = (p.batch + kThreads - 1) / kThreads;
  const int b0 = (int)min((int64_t)p.batch, (int64_t)tid * per), b1 = min(p.batch, b0 + per);
  Sums mine = {0, 0};
  uint32_t bad = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t old = p.cache_seqlens[b], fresh = p.new_lens[b];
    if (old < 0 || fresh < 0) {
      bad |= FA_TABLE_LENGTHS;
      continue;
    }
    const int64_t need = pages_of(old + fresh);
    if (need > p.table_pages) bad |= FA_TABLE_ROW;
    mine.tokens += fresh;
    mine.pages += need - pages_of(old);
  }
  Sums all;
  const Sums before = exclusive(mine, tid, warps, &all);
  if (all.tokens > p.num_slots) bad |= FA_TABLE_SLOTS;
  if (all.pages > p.num_free) bad |= FA_TABLE_FREE;
  uint32_t failed = 0;
  if (__syncthreads_or(bad))
    failed = (__syncthreads_or(bad & FA_TABLE_LENGTHS) ? FA_TABLE_LENGTHS : 0u) | (__syncthreads_or(bad & FA_TABLE_SLOTS) ? FA_TABLE_SLOTS : 0u) |
             (__syncthreads_or(bad & FA_TABLE_FREE) ? FA_TABLE_FREE : 0u) | (__syncthreads_or(bad & FA_TABLE_ROW) ? FA_TABLE_ROW : 0u);
  if (tid == 0 && blockIdx.x == 0) {
    if (host) {
      *reinterpret_cast<volatile uint32_t*>(host) = failed | kCheckDone;
      __threadfence_system();
    }
    p.pages_used[0] = failed ? -1 : (int)all.pages;
  }
  const int64_t from = (int64_t)blockIdx.x * kThreads + tid, step = (int64_t)gridDim.x * kThreads;
  if (failed) {
    for (int64_t i = from; i < p.num_slots; i += step) p.slots[i] = -1;
    for (int64_t i = from; i <= p.batch; i += step) p.cu_seqlens[i] = 0;
    return;
  }
  // (sums that passed the checks are below 2^31)
  first_token[tid] = (int)before.tokens;
  first_page[tid] = (int)before.pages;
  __syncthreads();

  for (int64_t i = from; i <= p.batch; i += step) {
    int sum = (int)all.tokens;
    if (i < p.batch) {
      const int s = (int)(i / per);
      sum = first_token[s];
      for (int b = s * per; b < i; ++b) sum += p.new_lens[b];
    }
    p.cu_seqlens[i] = sum;
  }
  for (int64_t i = from; i < all.pages; i += step) {
    const int s = stretch_of(first_page, (int)i);
    int left = (int)i - first_page[s], b = s * per;
    for (;; ++b) {
      const int64_t old = p.cache_seqlens[b];
      const int have = (int)pages_of(old), taken = (int)pages_of(old + p.new_lens[b]) - have;
      if (left < taken) {
        p.block_table[(int64_t)b * p.table_stride + have + left] = p.free_pages[i];
        break;
      }
      left -= taken;
    }
  }
  // kPerThread slots of a thread follow one another: one bisection for them
  const bool pairs = (reinterpret_cast<uintptr_t>(p.slots) & 15) == 0;
  for (int64_t i0 = from * kPerThread; i0 < p.num_slots; i0 += step * kPerThread) {
    int64_t slot[kPerThread];
    int left = 0, b = 0, fresh = 0, have = 0, first = 0;
    int64_t old = 0;
    const int n = (int)max((int64_t)0, min((int64_t)kPerThread, all.tokens - i0));
    auto enter = [&]() {                         // request b; `first`: where its pages begin among the free ones
      old = p.cache_seqlens[b];
      fresh = p.new_lens[b];
      have = (int)pages_of(old);
    };
    auto leave = [&]() {
      left -= fresh;
      first += (int)pages_of(old + fresh) - have;
      ++b;
    };
    if (n > 0) {
      const int s = stretch_of(first_token, (int)i0);
      left = (int)i0 - first_token[s];
      b = s * per;
      first = first_page[s];
      enter();
    }
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
      slot[e] = -1;
      if (e < n) {
        while (left >= fresh) {
          leave();
          enter();
        }
        const int64_t pos = old + left;
        const int pi = (int)(page_shift >= 0 ? pos >> page_shift : pos / p.page_size);
        const int page = pi < have ? p.block_table[(int64_t)b * p.table_stride + pi] : p.free_pages[first + pi - have];
        slot[e] = (int64_t)page * p.page_size + (pos - (int64_t)pi * p.page_size);
        ++left;
      }
    }
#pragma unroll
    for (int e = 0; e < kPerThread; e += 2) {
      if (pairs && i0 + e + 1 < p.num_slots) {
        *reinterpret_cast<longlong2*>(p.slots + i0 + e) = make_longlong2(slot[e], slot[e + 1]);
      } else {
        if (i0 + e < p.num_slots) p.slots[i0 + e] = slot[e];
        if (i0 + e + 1 < p.num_slots) p.slots[i0 + e + 1] = slot[e + 1];
      }
    }
  }
}

static int launch(const fa_block_table_args& a, uint32_t* host, cudaStream_t st) {
  int shift = -1;
  if ((a.page_size & (a.page_size - 1)) == 0)
    for (shift = 0; (1 << shift) < a.page_size;) ++shift;
  const int64_t most = a.num_slots > a.batch ? a.num_slots : a.batch;
  const int64_t need = (most + kThreads * kPerThread - 1) / (kThreads * kPerThread), fit = 4ll * sm_count(a.device);
  const unsigned grid = (unsigned)(need < 1 ? 1 : need < fit ? need : fit);
  block_table_kernel<<<grid, kThreads, 0, st>>>(a, shift, host);
  return check_launch("block_table");
}

int block_table(const fa_block_table_args& a, cudaStream_t st) { return launch(a, nullptr, st); }

int block_table_checked(const fa_block_table_args& a, uint32_t* failed, cudaStream_t st) {
  *failed = 0;
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone) {
    cudaGetLastError();
    set_error("value checks cannot run while the stream is being captured; turn them off with set_validation(False)");
    return FA_ERR_LAUNCH;
  }
  uint32_t* host = nullptr;
  const int slot = take_check_word(false, a.device, &host);
  if (slot < 0) return FA_ERR_LAUNCH;
  int r = launch(a, host, st);
  const bool queued = r == FA_OK;
  if (queued) r = await_check_word(slot, failed, st);
  give_check_word(slot, queued);
  return r;
}

}  // namespace fa
