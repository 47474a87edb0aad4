// After a verification: the rows of accepted tokens moved together in the caches of all layers, and the pages that nobody needs any
// more given back.
//
//   Compaction.  Row len + i takes row len + path[i], i ascending, and path ascends, so path[i] >= i: a row is read before it is
//   overwritten as long as each column of it is moved in order.  A thread therefore has one 16-byte column of one (layer, K or V, request) and
//   walks the path; the reads of kBatch steps are in flight together, ahead of their writes.  One launch moves all layers.
//   Bound.  Twice the bytes that move; a step of few requests is bounded by launch and by the chain accepted -> path -> page -> row.  24 layers of 96
//   requests, 32 nodes each, 8 heads of 128: 105 MB in and as much out, 37 us, and 45 with the value checks, a kernel ahead of it (floor 32).
//   Pages.  As in block_table.cu: every CTA sums all requests, then writes an even share of the numbers, found again by bisection.
#include "cache_dev.cuh"
#include "check_words.h"

namespace fa {

namespace {

constexpr int kThreads = 128;
constexpr int kBatch = 8;              // steps whose reads are in flight together
constexpr int kSteps = 64;             // steps whose rows are worked out at a time
constexpr int kChecksInside = 512;     // path entries up to which every CTA makes the checks of all requests itself

struct Layers {
  void* p[2][FA_COMPACT_LAYERS];
};

__device__ __forceinline__ int64_t capacity_of(const fa_compact_args& p) {
  return p.block_table ? (int64_t)p.block_table_stride * p.page_size : p.page_size;
}
__device__ __forceinline__ int page_index(const fa_compact_args& p, int shift, int64_t pos) {
  return (int)(shift >= 0 ? pos >> shift : pos / p.page_size);
}

// Which checks request b fails, seen by this thread of nt.
__device__ __forceinline__ uint32_t request_checks(const fa_compact_args& p, int shift, int b, int tid, int nt) {
  const int n = p.num_accepted[b];
  if (n < 0 || n > p.path_len) return FA_COMPACT_COUNT;
  const int64_t len = p.cache_seqlens[b], pad = p.cache_leftpad ? p.cache_leftpad[b] : 0, cap = capacity_of(p);
  if (len < 0 || pad < 0) return FA_COMPACT_LENGTHS;
  uint32_t bad = 0;
  const int row = p.cache_batch_idx ? p.cache_batch_idx[b] : b;
  if (p.block_table == nullptr && (unsigned)row >= (unsigned)p.num_pages) bad |= FA_COMPACT_PAGES;
  const int32_t* path = p.path + (int64_t)b * p.path_stride;
  const int32_t* table = p.block_table ? p.block_table + (int64_t)b * p.block_table_stride : nullptr;
  for (int i = tid; i < n; i += nt) {
    const int x = path[i], before = i > 0 ? path[i - 1] : -1;
    if (x <= before || x < 0) {
      bad |= FA_COMPACT_PATH;
      continue;
    }
    // (an ascending path has x >= i, so the row that is written lies inside as well)
    const int64_t from = len + pad + x, to = len + pad + i;
    if (from >= cap || to >= cap) {
      bad |= FA_COMPACT_LENGTHS;
      continue;
    }
    if (table && ((unsigned)table[page_index(p, shift, from)] >= (unsigned)p.num_pages ||
                  (unsigned)table[page_index(p, shift, to)] >= (unsigned)p.num_pages))
      bad |= FA_COMPACT_PAGES;
  }
  return bad;
}

// Of all threads of the CTA, the same for each.
__device__ __forceinline__ uint32_t all_of(uint32_t bad) {
  if (!__syncthreads_or(bad)) return 0u;
  uint32_t all = 0;
#pragma unroll
  for (uint32_t bit = 1; bit <= FA_COMPACT_PAGES; bit <<= 1) all |= __syncthreads_or(bad & bit) ? bit : 0u;
  return all;
}

__device__ __forceinline__ void answer(uint32_t* host, uint32_t bad) {
  *reinterpret_cast<volatile uint32_t*>(host) = bad | kCheckDone;
  __threadfence_system();
}

// Of all requests, ahead of the kernel that moves: a step of a path per thread, the reads of kAtOnce of them in flight together.
__global__ void __launch_bounds__(1024) compact_check_kernel(const fa_compact_args p, int shift, uint32_t* host, uint32_t* dev) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int kAtOnce = 4;
  const int64_t cap = capacity_of(p), all = (int64_t)p.batch * p.path_len;
  uint32_t bad = 0;
  for (int b = threadIdx.x; b < p.batch; b += 1024) {
    const int n = p.num_accepted[b], row = p.cache_batch_idx ? p.cache_batch_idx[b] : b;
    if (n < 0 || n > p.path_len) bad |= FA_COMPACT_COUNT;
    if (p.cache_seqlens[b] < 0 || (p.cache_leftpad && p.cache_leftpad[b] < 0)) bad |= FA_COMPACT_LENGTHS;
    if (p.block_table == nullptr && (unsigned)row >= (unsigned)p.num_pages) bad |= FA_COMPACT_PAGES;
  }
  for (int64_t i0 = threadIdx.x; i0 < all; i0 += 1024 * kAtOnce) {
    int x[kAtOnce], before[kAtOnce], page[2 * kAtOnce];
    int64_t len[kAtOnce];
    bool in[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int64_t at = min(i0 + k * 1024, all - 1);
      const int b = (int)(at / p.path_len), i = (int)(at - (int64_t)b * p.path_len);
      const int32_t* path = p.path + (int64_t)b * p.path_stride;
      in[k] = i0 + k * 1024 < all && i < min(p.num_accepted[b], p.path_len);
      len[k] = max((int64_t)p.cache_seqlens[b] + (p.cache_leftpad ? p.cache_leftpad[b] : 0), (int64_t)0);
      x[k] = path[i];
      before[k] = i > 0 ? path[i - 1] : -1;
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int64_t at = min(i0 + k * 1024, all - 1);
      const int b = (int)(at / p.path_len), i = (int)(at - (int64_t)b * p.path_len);
      const int64_t from = len[k] + x[k], to = len[k] + i;
      if (in[k] && (x[k] <= before[k] || x[k] < 0)) bad |= FA_COMPACT_PATH;
      in[k] = in[k] && x[k] > before[k] && x[k] >= 0;
      if (in[k] && (from >= cap || to >= cap)) bad |= FA_COMPACT_LENGTHS;
      in[k] = in[k] && from < cap && to < cap;
      const int32_t* table = p.block_table ? p.block_table + (int64_t)b * p.block_table_stride : nullptr;
      page[2 * k] = table && in[k] ? table[page_index(p, shift, from)] : 0;
      page[2 * k + 1] = table && in[k] ? table[page_index(p, shift, to)] : 0;
    }
#pragma unroll
    for (int k = 0; k < 2 * kAtOnce; ++k)
      if (p.block_table && in[k / 2] && (unsigned)page[k] >= (unsigned)p.num_pages) bad |= FA_COMPACT_PAGES;
  }
  bad = all_of(bad);
  if (threadIdx.x == 0) {
    *dev = bad;
    answer(host, bad);
  }
}

// grid: (columns of kThreads chunks x tensors, requests)
__global__ void __launch_bounds__(kThreads) compact_kernel(const fa_compact_args p, const Layers layers, int shift, int stripes,
                                                           uint32_t* host, const uint32_t* dev) {
  __shared__ int64_t rows[2][kSteps];               // [from, to]
  const int tid = threadIdx.x;
  if (host) {
    uint32_t bad = 0;
    for (int b = tid >> 5; b < p.batch; b += kThreads / 32) bad |= request_checks(p, shift, b, tid & 31, 32);
    bad = all_of(bad);
    if (tid == 0 && blockIdx.x == 0 && blockIdx.y == 0) answer(host, bad);
    if (bad) return;
  } else if (dev) {
    asm volatile("griddepcontrol.wait;" ::: "memory");         // the kernel with the checks may still run
    if (*dev) return;
  }
  const int tensor = blockIdx.x / stripes, stripe = blockIdx.x - tensor * stripes;
  const int which = tensor & 1, layer = tensor >> 1;
  const int64_t* stride = which ? p.vc_stride : p.kc_stride;
  const int cpr = p.head_dim / 8, chunk = stripe * kThreads + tid;
  const bool mine = chunk < p.heads * cpr;
  const int head = mine ? chunk / cpr : 0;
  uint16_t* base = static_cast<uint16_t*>(layers.p[which][layer]) + head * stride[2] + (mine ? chunk - head * cpr : 0) * 8;
  for (int b = blockIdx.y; b < p.batch; b += gridDim.y) {
    if (!host && !dev && all_of(request_checks(p, shift, b, tid, kThreads))) continue;
    const int n = p.num_accepted[b];
    const int64_t first = (int64_t)p.cache_seqlens[b] + (p.cache_leftpad ? p.cache_leftpad[b] : 0);
    const int32_t* path = p.path + (int64_t)b * p.path_stride;
    const int32_t* table = p.block_table ? p.block_table + (int64_t)b * p.block_table_stride : nullptr;
    const int64_t own = (p.cache_batch_idx ? p.cache_batch_idx[b] : b) * stride[0];
    auto row_of = [&](int64_t pos) {
      if (!table) return own + pos * stride[1];
      const int pi = page_index(p, shift, pos);
      return table[pi] * stride[0] + (pos - (int64_t)pi * p.page_size) * stride[1];
    };
    for (int s0 = 0; s0 < n; s0 += kSteps) {
      const int steps = min(kSteps, n - s0);
      __syncthreads();
      for (int i = tid; i < 2 * steps; i += kThreads) {
        const int step = i >> 1;
        rows[i & 1][step] = row_of(first + ((i & 1) ? s0 + step : path[s0 + step]));
      }
      __syncthreads();
      if (!mine) continue;
      for (int i0 = 0; i0 < steps; i0 += kBatch) {
        uint4 x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          if (i0 + i < steps && rows[0][i0 + i] != rows[1][i0 + i]) x[i] = *reinterpret_cast<const uint4*>(base + rows[0][i0 + i]);
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
          if (i0 + i < steps && rows[0][i0 + i] != rows[1][i0 + i]) *reinterpret_cast<uint4*>(base + rows[1][i0 + i]) = x[i];
      }
    }
  }
}

bool capturing(cudaStream_t st) {
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &cap) == cudaSuccess && cap == cudaStreamCaptureStatusNone) return false;
  cudaGetLastError();
  set_error("value checks cannot run while the stream is being captured; turn them off with set_validation(False)");
  return true;
}

int shift_of(int page_size) {
  if (page_size & (page_size - 1)) return -1;
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

int launch_compact(const fa_compact_args& a, uint32_t* host, const uint32_t* dev, cudaStream_t st) {
  Layers l = {};
  for (int i = 0; i < a.layers; ++i) {
    l.p[0][i] = a.k_cache[i];
    l.p[1][i] = a.v_cache[i];
  }
  const int stripes = (a.heads * (a.head_dim / 8) + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(2 * a.layers * stripes), (unsigned)(a.batch < 65535 ? a.batch : 65535));
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr;
  lc.gridDim = grid;
  lc.blockDim = dim3(kThreads);
  lc.stream = st;
  if (dev) {
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = &attr;
    lc.numAttrs = 1;
  }
  cudaLaunchKernelEx(&lc, compact_kernel, a, l, shift_of(a.page_size), stripes, host, dev);
  return check_launch("compact");
}

}  // namespace

int compact(const fa_compact_args& a, cudaStream_t st) { return a.batch == 0 || a.layers == 0 ? FA_OK : launch_compact(a, nullptr, nullptr, st); }

size_t compact_workspace_bytes(const fa_compact_args& a) { return (int64_t)a.batch * a.path_len <= kChecksInside ? 0 : 16; }

int compact_checked(const fa_compact_args& a, uint32_t* failed, cudaStream_t st) {
  *failed = 0;
  if (capturing(st)) return FA_ERR_LAUNCH;
  if (a.batch == 0 || a.layers == 0) return FA_OK;
  const bool inside = compact_workspace_bytes(a) == 0;
  if (!inside && (a.workspace == nullptr || a.workspace_bytes < compact_workspace_bytes(a))) {
    set_error("compact workspace too small: need %zu bytes, got %zu", compact_workspace_bytes(a), a.workspace_bytes);
    return FA_ERR_WORKSPACE;
  }
  uint32_t* host = nullptr;
  const int slot = take_check_word(false, a.device, &host);
  if (slot < 0) return FA_ERR_LAUNCH;
  int r = FA_OK;
  bool queued = false;
  if (inside) {
    r = launch_compact(a, host, nullptr, st);
    queued = r == FA_OK;
  } else {
    uint32_t* dev = static_cast<uint32_t*>(a.workspace);
    compact_check_kernel<<<1, 1024, 0, st>>>(a, shift_of(a.page_size), host, dev);
    r = check_launch("compact_check");
    queued = r == FA_OK;
    if (queued) r = launch_compact(a, nullptr, dev, st);
  }
  if (queued) {
    const int w = await_check_word(slot, failed, st);
    if (r == FA_OK) r = w;
  }
  give_check_word(slot, queued);
  return r;
}

// ---------------------------------------------------------------------------------------
// pages
// ---------------------------------------------------------------------------------------
namespace {

constexpr int kPageThreads = 256;
constexpr int kFirsts = 4096;          // requests whose first pages are held in shared memory, and found by one bisection
constexpr int kPagesOfThread = 4;      // one behind the other

__global__ void __launch_bounds__(kPageThreads) release_kernel(const fa_release_args p, int shift, uint32_t* host) {
  __shared__ int64_t warps[kPageThreads / 32];
  __shared__ int first[kPageThreads], begins[kFirsts];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto pages_of = [&](int64_t n) { return shift >= 0 ? (n + p.page_size - 1) >> shift : (n + p.page_size - 1) / p.page_size; };
  const int per = (p.batch + kPageThreads - 1) / kPageThreads;
  const int b0 = (int)min((int64_t)p.batch, (int64_t)tid * per), b1 = min(p.batch, b0 + per);
  int64_t mine = 0;
  uint32_t bad = 0;
  for (int b = b0; b < b1; ++b) {
    const int held = p.held_lens[b], kept = p.kept_lens[b];
    if (kept < 0 || held < kept) {
      bad |= FA_RELEASE_LENGTHS;
      continue;
    }
    const int64_t end = pages_of(held);
    if (end > p.table_pages) bad |= FA_RELEASE_ROW;
    mine += end - pages_of(kept);
  }
  int64_t sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  if (lane == 31) warps[warp] = sum;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPageThreads / 32; ++w) {
    if (w == warp) before = all;
    all += warps[w];
  }
  before += sum - mine;
  if (all > p.num_pages) bad |= FA_RELEASE_ROOM;
  uint32_t failed = 0;
  if (__syncthreads_or(bad))
    failed = (__syncthreads_or(bad & FA_RELEASE_LENGTHS) ? FA_RELEASE_LENGTHS : 0u) | (__syncthreads_or(bad & FA_RELEASE_ROW) ? FA_RELEASE_ROW : 0u) |
             (__syncthreads_or(bad & FA_RELEASE_ROOM) ? FA_RELEASE_ROOM : 0u);
  if (tid == 0 && blockIdx.x == 0) {
    if (host) answer(host, failed);
    p.pages_released[0] = failed ? -1 : (int)all;
  }
  const int64_t from = (int64_t)blockIdx.x * kPageThreads + tid, step = (int64_t)gridDim.x * kPageThreads;
  if (failed) {
    for (int64_t i = from; i < p.num_pages; i += step) p.pages[i] = -1;
    return;
  }
  first[tid] = (int)before;            // (a sum that passed the checks is below 2^31)
  __syncthreads();
  const bool held = p.batch <= kFirsts;
  if (held) {
    int at = (int)before;
    for (int b = b0; b < b1; ++b) {
      begins[b] = at;
      at += (int)(pages_of(p.held_lens[b]) - pages_of(p.kept_lens[b]));
    }
    __syncthreads();
  }
  int log2 = 1;
  while (held && log2 < p.batch) log2 <<= 1;
  for (int64_t i0 = from * kPagesOfThread; i0 < p.num_pages; i0 += step * kPagesOfThread) {
    int page[kPagesOfThread], b = 0, left = 0;
    if (i0 < all) {
      if (held) {                      // last request that begins at i0 or before
        for (int k = log2 >> 1; k > 0; k >>= 1)
          if (b + k < p.batch && begins[b + k] <= (int)i0) b += k;
        left = (int)i0 - begins[b];
      } else {
        int s = 0;                     // last stretch of requests that does
#pragma unroll
        for (int k = kPageThreads / 2; k > 0; k >>= 1)
          if (first[s + k] <= (int)i0) s += k;
        b = s * per;
        left = (int)i0 - first[s];
      }
    }
#pragma unroll
    for (int e = 0; e < kPagesOfThread; ++e) {
      page[e] = -1;
      if (i0 + e < all) {
        int keep, gone;
        for (;; ++b, left -= gone) {
          keep = (int)pages_of(p.kept_lens[b]);
          gone = (int)pages_of(p.held_lens[b]) - keep;
          if (left < gone) break;
        }
        page[e] = p.block_table[(int64_t)b * p.table_stride + keep + left];
        ++left;
      }
    }
    if ((reinterpret_cast<uintptr_t>(p.pages) & 15) == 0 && i0 + kPagesOfThread <= p.num_pages) {
      *reinterpret_cast<int4*>(p.pages + i0) = make_int4(page[0], page[1], page[2], page[3]);
    } else {
#pragma unroll
      for (int e = 0; e < kPagesOfThread; ++e)
        if (i0 + e < p.num_pages) p.pages[i0 + e] = page[e];
    }
  }
}

int launch_release(const fa_release_args& a, uint32_t* host, cudaStream_t st) {
  const int64_t need = ((int64_t)a.num_pages + kPageThreads * kPagesOfThread - 1) / (kPageThreads * kPagesOfThread), fit = 4ll * sm_count(a.device);
  const unsigned grid = (unsigned)(need < 1 ? 1 : need < fit ? need : fit);
  release_kernel<<<grid, kPageThreads, 0, st>>>(a, shift_of(a.page_size), host);
  return check_launch("release_pages");
}

}  // namespace

int release_pages(const fa_release_args& a, cudaStream_t st) { return launch_release(a, nullptr, st); }

int release_pages_checked(const fa_release_args& a, uint32_t* failed, cudaStream_t st) {
  *failed = 0;
  if (capturing(st)) return FA_ERR_LAUNCH;
  uint32_t* host = nullptr;
  const int slot = take_check_word(false, a.device, &host);
  if (slot < 0) return FA_ERR_LAUNCH;
  int r = launch_release(a, host, st);
  const bool queued = r == FA_OK;
  if (queued) r = await_check_word(slot, failed, st);
  give_check_word(slot, queued);
  return r;
}

}  // namespace fa
