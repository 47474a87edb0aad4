// Verification of drafted tokens: which nodes of a request's tree the target model accepts, and the token that follows them.
//
//   Mathematics.  A node's children are tried in order; after a rejection the target's distribution becomes norm(max(p' - q, 0)), p' being
//   what it was.  With p' = max(p - c q, 0) / Z that is max(p - (c + Z) q, 0) / Z', because q >= 0: all that a rejection changes
//   is the number c, which grows by Z, and Z, the mass that is then left.  The first child of a node has c = 0, Z = 1 and reads two numbers; only
//   a node with a rejected child and another one behind it, and the node where the path ends, is read over its whole vocabulary.
//   Sums and products are in 64 bits: a decision next to a border then depends on the order of a sum only within 1e-16 of it.
//   Bound.  Latency for small batches, else 2 vocab words a request out of HBM; after that the passes of one request, which come one behind the
//   other: a pass of 100003 tokens takes a request 2.4 us where its CTAs have an SM each, 3.7 where two share one, most of it instructions and the
//   cluster's barrier.  A number becomes a double by an integer product and not by a conversion, of which an SM makes 16 a clock.
//   A cluster of CTAs has a request, as large as all requests leave room for: a second wave starts from the beginning (64 requests of 100003 tokens,
//   one pass each: clusters of 8 in two waves 20.2 us, of 4 in one 12.3, now 9.7).  Each CTA loads all nodes' numbers at once and walks the tree on its own (ballots
//   over 32 nodes), so that the walk takes no round trip to memory.  What fits of the node at hand stays in shared memory for the passes after the first.
//   A warp has an even, contiguous share of the vocabulary, its sums go to all CTAs of the cluster through distributed shared memory, and every
//   warp adds them up in the same order.  The share that the random number falls into is cut among the warps of its CTA in the same way, and one of
//   them finds the token.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "common.cuh"

namespace fa {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMostShared = 224 * 1024;  // dynamic shared memory of a CTA

template <typename T> __device__ __forceinline__ float wide(T x);
template <> __device__ __forceinline__ float wide(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float wide(float x) { return x; }

__device__ __forceinline__ double left_of(double p, double q, double c) { return fmax(fma(-c, q, p), 0.0); }

// Of a node: target and draft at its parent, its random number, its parent or -1.  In dynamic shared memory, ahead of the share of p and q.
struct Node {
  float p, q, u;
  int parent;
};
struct Shared {
  double part[2][kMaxCluster * kWarps];    // sums of all warps of the cluster, of one pass and the next
  double cut[kWarps];                      // of the warps' parts of one share
};

// Where `bound` falls among n sums in a row, the first of them preceded by `run`: the first one that reaches beyond it, else the last that
// holds anything (-1: none does); *before: what comes ahead of it.  By a warp, the same for each lane.
__device__ __forceinline__ int place_of(const double* part, int n, double bound, double run, int lane, double* before) {
  const int per = (n + 31) / 32, i0 = min(n, lane * per), i1 = min(n, i0 + per);
  double mine = 0.0;
  for (int i = i0; i < i1; ++i) mine += part[i];
  double inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  run += inc - mine;
  int at = -1, last = -1;
  double at_before = 0.0, last_before = 0.0;
  for (int i = i0; i < i1; ++i) {
    if (part[i] > 0.0) {
      last = i;
      last_before = run;
      if (at < 0 && run + part[i] > bound) {
        at = i;
        at_before = run;
      }
    }
    run += part[i];
  }
  const unsigned found = __ballot_sync(0xffffffffu, at >= 0), some = __ballot_sync(0xffffffffu, last >= 0);
  if (some == 0u) return -1;
  const int src = found ? __ffs(found) - 1 : 31 - __clz(some);
  *before = __shfl_sync(0xffffffffu, found ? at_before : last_before, src);
  return __shfl_sync(0xffffffffu, found ? at : last, src);
}

// NaN where an argument of max() is: fmax() would drop it.
__device__ __forceinline__ double rest_of(float p, float q, double c) {
  const double r = fma(-c, (double)q, (double)p);
  return r > 0.0 ? r : (r == r ? 0.0 : r);
}

// The bits of a positive finite x, moved up, are the double x 2^-896 exactly, the smallest and 0 too: an integer product in place of a conversion.
__device__ __forceinline__ double scaled(float x) { return __longlong_as_double((long long)(__float_as_uint(x) * (1ull << 29))); }
constexpr double kScale = 0x1p896;

// Adds up what is left over [v0, v1), by a warp, times 1 / kScale; kAtOnce numbers of a lane are in flight together.  top: at least the bits of
// all numbers; from those of infinity on, the sum is not one (NaN, infinity, negative).  kAll: c is 0.
constexpr int kAtOnce = 8;
// from(v): gives the numbers at v + 32 k.
template <bool kAll, typename F>
__device__ __forceinline__ void add_left(double (&s)[2], uint32_t& top, F from, uint32_t v0, uint32_t v1, double c, int lane) {
  auto add = [&](double& to, float2 x) {
    if (kAll) {
      top = max(top, __float_as_uint(x.x));
      to += scaled(x.x);
      return;
    }
    top = max(max(top, __float_as_uint(x.x)), __float_as_uint(x.y));
    const double r = fma(-c, scaled(x.y), scaled(x.x));
    if (__double2hiint(r) >= 0) to += r;
  };
  uint32_t v = v0 + lane;
#pragma unroll 1
  for (; v + 32 * (kAtOnce - 1) < v1; v += 32 * kAtOnce) {
    auto at = from(v);
    float2 x[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) x[k] = at(k);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) add(s[k & 1], x[k]);
  }
  if (v >= v1) return;
  auto at = from(v);
  float2 x[kAtOnce];
#pragma unroll
  for (int k = 0; k < kAtOnce - 1; ++k) x[k] = v + 32 * k < v1 ? at(k) : make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < kAtOnce - 1; ++k) add(s[k & 1], x[k]);
}

// hold: numbers at the start of a warp's share that stay in dynamic shared memory.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const fa_verify_args a, const int hold) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  Node* nodes = reinterpret_cast<Node*>(dynamic);
  float2* held = reinterpret_cast<float2*>(nodes + a.nodes);
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* target = static_cast<const T*>(a.target) + b * a.target_stride[0];
  const T* draft = static_cast<const T*>(a.draft) + b * a.draft_stride[0];
  for (int i = tid; i < a.nodes; i += kThreads) {
    const int parent = a.parents[b * a.parent_stride + i];
    const int64_t token = a.draft_tokens[b * a.token_stride + i];
    const bool used = i > 0 && parent >= 0 && parent < i;
    float p = 0.f, q = 0.f;
    if (used && token >= 0 && token < a.vocab) {
      p = wide(target[parent * a.target_stride[1] + token]);
      q = wide(draft[parent * a.draft_stride[1] + token]);
    }
    nodes[i] = Node{p, q, a.accept[(int64_t)b * a.nodes + i], used ? parent : -1};
  }
  cluster.sync();                          // all of its CTAs run: their shared memory may be written

  // this warp's share of the vocabulary
  const int slots = C * kWarps, slots_log2 = 31 - __clz(slots), slot = rank * kWarps + warp;       // (a power of two)
  auto share_at = [&](int i) { return (uint32_t)((a.vocab * i) >> slots_log2); };
  const uint32_t v0 = share_at(slot), v1 = share_at(slot + 1);
  int pass = 0, holds = -1;                                    // holds: the node that is in shared memory
  // What is left at `node` over [u0, u1) of the share that begins at w0 and has its place in shared memory at `own`.  (q is not read where
  // nothing of it is taken off.)
  auto sum_of = [&](int node, double c, uint32_t w0, float2* own, uint32_t u0, uint32_t u1) {
    const T* pr = target + node * a.target_stride[1];
    const T* qr = draft + node * a.draft_stride[1];
    double s[2] = {0.0, 0.0};
    uint32_t top = 0;
    if (c == 0.0) {
      add_left<true>(s, top, [&](uint32_t v) {
        return [p = pr + v](int k) { return make_float2(wide(p[32 * k]), 0.f); };
      }, u0, u1, c, lane);
    } else {
      const uint32_t vh = max(u0, min(u1, w0 + hold));
      if (holds == node) {
        add_left<false>(s, top, [&](uint32_t v) { return [o = own + (v - w0)](int k) { return o[32 * k]; }; }, u0, vh, c, lane);
      } else {
        add_left<false>(s, top, [&](uint32_t v) {
          return [p = pr + v, q = qr + v, o = own + (v - w0)](int k) { return o[32 * k] = make_float2(wide(p[32 * k]), wide(q[32 * k])); };
        }, u0, vh, c, lane);
      }
      add_left<false>(s, top, [&](uint32_t v) {
        return [p = pr + v, q = qr + v](int k) { return make_float2(wide(p[32 * k]), wide(q[32 * k])); };
      }, vh, u1, c, lane);
    }
    double sum = (s[0] + s[1]) * kScale;
    if (__any_sync(0xffffffffu, top >= 0x7f800000u)) {
      sum = 0.0;
      for (uint32_t v = u0 + lane; v < u1; v += 32) sum += rest_of(wide(pr[v]), c != 0.0 ? wide(qr[v]) : 0.f, c);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
  };
  // Sums of max(p - c q, 0) over the shares at `node`: in part[.] of every CTA.
  auto sums = [&](int node, double c) -> const double* {
    const double sum = sum_of(node, c, v0, held + warp * hold, v0, v1);
    if (c != 0.0) holds = node;
    double* mine = sh.part[pass & 1];
    ++pass;
    if (lane < C) *cluster.map_shared_rank(mine + slot, lane) = sum;
    // (what is written next goes to the other half, and nobody gets there before all have read this one: there is a barrier between)
    cluster.sync();
    return mine;
  };
  auto total_of = [&](const double* part) {
    double sum = 0.0;
    for (int i = lane; i < slots; i += 32) sum += part[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
  };

  // ---- the walk: every warp of the cluster on its own, all alike ----------------------------
  int node = 0, count = 1;
  double c = 0.0, mass = 1.0;
  bool fresh = true;                             // mass is that of c
  int32_t* path = a.path + (int64_t)b * a.nodes;
  if (rank == 0 && tid == 0) path[0] = 0;
  for (int i0 = 0; i0 < a.nodes; i0 += 32) {
    int from = 0;                                // of these 32, those still to be looked at
    for (;;) {
      const bool child = i0 + lane < a.nodes && lane >= from && nodes[i0 + lane].parent == node;
      const unsigned any = __ballot_sync(0xffffffffu, child);
      if (any == 0u) break;
      const int i = i0 + __ffs(any) - 1;
      from = i - i0 + 1;
      if (!fresh) {
        mass = total_of(sums(node, c));
        fresh = true;
      }
      const double p = nodes[i].p, q = nodes[i].q;
      if ((double)nodes[i].u * q * mass < left_of(p, q, c)) {
        node = i;
        c = 0.0;
        mass = 1.0;
        if (rank == 0 && tid == 0) path[count] = i;
        ++count;
      } else {
        c += mass;
        fresh = false;
      }
    }
  }
  if (rank == 0) {
    for (int i = count + tid; i < a.nodes; i += kThreads) path[i] = -1;
    if (tid == 0) a.num_accepted[b] = count;
  }

  // ---- the token that follows ----------------------------------------------------------------
  const double* part = sums(node, c);
  double sum = total_of(part);
  if (!(sum > 0.0) && sum == sum && c != 0.0) {   // nothing is left of p
    c = 0.0;
    part = sums(node, c);
    sum = total_of(part);
  }
  if (!(sum > 0.0) || sum > 1.7e308) {
    if (rank == 0 && tid == 0) a.next_token[b] = -1;
    return;
  }
  const double bound = (double)a.sample[b] * sum;
  double run = 0.0;
  const int at = place_of(part, slots, bound, 0.0, lane, &run);
  if (at < 0 || at / kWarps != rank) return;         // (at >= 0: the sum is positive)
  // that share, [w0, w1), in the CTA that has it: a part of it for each warp
  const uint32_t w0 = share_at(at), n = share_at(at + 1) - w0;
  const uint32_t u0 = w0 + (uint32_t)((uint64_t)n * warp / kWarps), u1 = w0 + (uint32_t)((uint64_t)n * (warp + 1) / kWarps);
  float2* own = held + (at - rank * kWarps) * hold;
  __syncthreads();                               // (one warp's share in shared memory, read by all: where c is not 0, it holds the node)
  const double mine = sum_of(node, c, w0, own, u0, u1);
  if (lane == 0) sh.cut[warp] = mine;
  __syncthreads();
  if (place_of(sh.cut, kWarps, bound, run, lane, &run) != warp) return;
  const T* pr = target + node * a.target_stride[1];
  const T* qr = draft + node * a.draft_stride[1];
  int64_t token = -1;
  for (uint32_t v = u0; v < u1; v += 32) {
    const uint32_t i = v + lane;
    const double r = i < u1 ? rest_of(wide(pr[i]), c != 0.0 ? wide(qr[i]) : 0.f, c) : 0.0;
    double s = r;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    const unsigned over = __ballot_sync(0xffffffffu, r > 0.0 && run + s > bound), some = __ballot_sync(0xffffffffu, r > 0.0);
    if (some) token = (int64_t)v + 31 - __clz(some);
    if (over) {
      token = (int64_t)v + __ffs(over) - 1;
      break;
    }
    run += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) a.next_token[b] = token;
}

template <typename T>
int launch_verify(const fa_verify_args& a, cudaStream_t st) {
  // shares of a few hundred tokens at least, and no more CTAs than run at a time
  const int sms = sm_count(a.device);
  int cluster = 1;
  while (cluster < kMaxCluster && a.vocab > (int64_t)cluster * kThreads * 4 && (int64_t)a.batch * cluster * 2 <= 2 * sms) cluster *= 2;
  // what fits of a share in shared memory, beside another CTA's, or alone on its SM where there are SMs enough: the nearer the CTAs come to
  // the SMs' number, the more clusters wait for another's end, for a cluster lies within one part of the GPU.  Alone and not, us, 24 children of one
  // node, 40009 tokens: 10 and 14 clusters of 8 the same, 16 53, 61; 18 56, 53; 100003 tokens: 16 63.5, 64; 18 69, 68.
  const bool alone = (int64_t)a.batch * cluster <= sms * 3 / 4;
  const size_t nodes = a.nodes * sizeof(Node), room = (alone ? kMostShared : kMostShared / 2 - 2048) - nodes;
  const int64_t share = a.vocab / (cluster * kWarps) + 1, fit = (int64_t)(room / sizeof(float2) / kWarps);
  const int hold = (int)(share < fit ? share : fit);
  // (more than half of an SM's, so that CTAs do not share an SM while others have none)
  const size_t smem = std::max(nodes + (size_t)hold * kWarps * sizeof(float2), (size_t)(alone ? 116 * 1024 : 0));
  auto kern = verify_kernel<T>;
  // Once per kernel and device, the most that any call takes (another thread's call may come between this and the launch).  By every first
  // call: without it 48 KB are the limit of dynamic and static shared memory together.
  static_assert(kMostShared + sizeof(Shared) <= 227 * 1024, "shared memory budget");
  static std::atomic<uint64_t> prepared{0};
  const uint64_t bit = a.device < 64 ? 1ull << a.device : 0;
  if ((prepared.load(std::memory_order_relaxed) & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
    if (e != cudaSuccess) {
      set_error("verify_draft_tree: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      return FA_ERR_LAUNCH;
    }
    prepared.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  lc.gridDim = dim3((unsigned)a.batch * cluster);
  lc.blockDim = dim3(kThreads);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  lc.attrs = &attr;
  lc.numAttrs = 1;
  cudaLaunchKernelEx(&lc, kern, a, hold);
  return check_launch("verify_draft_tree");
}

}  // namespace

int verify_draft_tree(const fa_verify_args& a, cudaStream_t st) {
  if (a.batch == 0) return FA_OK;
  if (a.dtype == FA_F16) return launch_verify<__half>(a, st);
  if (a.dtype == FA_BF16) return launch_verify<__nv_bfloat16>(a, st);
  return launch_verify<float>(a, st);
}

}  // namespace fa
