// Verification of drafted tokens: which nodes of a request's tree the target model accepts, and the token that follows them.
//
//   Mathematics.  A node's children are tried in order; after a rejection the target's distribution becomes norm(max(p' - q, 0)), p' being
//   what it was.  With p' = max(p - c q, 0) / Z that is max(p - (c + Z) q, 0) / Z', because q >= 0: all that a rejection changes
//   is the number c, which grows by Z, and Z, the mass that is then left.  The first child of a node has c = 0, Z = 1 and reads two numbers; only
//   a node with a rejected child and another one behind it, and the node where the path ends, is read over its whole vocabulary.
//   Sums and products are in 64 bits: a decision next to a border then depends on the order of a sum only within 1e-16 of it.
//   Bound.  Latency for small batches, else 2 vocab words a request out of HBM and the conversions to 64 bits.
//   A cluster of CTAs has a request.  Each loads all nodes' numbers at once and walks the tree on its own (ballots over 32 nodes), so
//   that the walk takes no round trip to memory; a warp has an even, contiguous share of the vocabulary, its sums go to all CTAs of the cluster
//   through distributed shared memory, and every warp adds them up in the same order.  The warp whose share the random number falls
//   into reads that share again.
#include <cooperative_groups.h>

#include "common.cuh"

namespace fa {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kNodes = 1024;
constexpr int kMaxCluster = 8;

template <typename T> __device__ __forceinline__ float wide(T x);
template <> __device__ __forceinline__ float wide(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float wide(float x) { return x; }

__device__ __forceinline__ double left_of(double p, double q, double c) { return fmax(fma(-c, q, p), 0.0); }

struct Shared {
  float p[kNodes], q[kNodes], u[kNodes];   // of a node: target and draft at its parent, its random number
  int parent[kNodes];
  double part[2][kMaxCluster * kWarps];    // sums of all warps of the cluster, of one pass and the next
};

// NaN where an argument of max() is: fmax() would drop it.
__device__ __forceinline__ double rest_of(float p, float q, double c) {
  const double r = fma(-c, (double)q, (double)p);
  return r > 0.0 ? r : (r == r ? 0.0 : r);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const fa_verify_args a) {
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
    sh.parent[i] = used ? parent : -1;
    sh.p[i] = p;
    sh.q[i] = q;
    sh.u[i] = a.accept[(int64_t)b * a.nodes + i];
  }
  cluster.sync();                          // all of its CTAs run: their shared memory may be written

  // this warp's share of the vocabulary
  const int slots = C * kWarps, slot = rank * kWarps + warp;
  const int64_t v0 = a.vocab * slot / slots, v1 = a.vocab * (slot + 1) / slots;
  int pass = 0;
  // Sums of max(p - c q, 0) over the shares at `node`: in part[.] of every CTA.
  auto sums = [&](int node, double c) -> const double* {
    const T* pr = target + node * a.target_stride[1];
    const T* qr = draft + node * a.draft_stride[1];
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    for (int64_t v = v0 + lane; v < v1; v += 128) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (v + 32 * k < v1) s[k] += rest_of(wide(pr[v + 32 * k]), c != 0.0 ? wide(qr[v + 32 * k]) : 0.f, c);
    }
    double sum = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
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
      const bool child = i0 + lane < a.nodes && lane >= from && sh.parent[i0 + lane] == node;
      const unsigned any = __ballot_sync(0xffffffffu, child);
      if (any == 0u) break;
      const int i = i0 + __ffs(any) - 1;
      from = i - i0 + 1;
      if (!fresh) {
        mass = total_of(sums(node, c));
        fresh = true;
      }
      const double p = sh.p[i], q = sh.q[i];
      if ((double)sh.u[i] * q * mass < left_of(p, q, c)) {
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
  // the first share whose running sum exceeds the bound, else the last one that holds anything
  const double bound = (double)a.sample[b] * sum;
  double run = 0.0, before = 0.0, last_before = 0.0;
  int at = -1, last = -1;
  for (int i = 0; i < slots && at < 0; ++i) {
    const double x = part[i];
    if (x > 0.0) {
      last = i;
      last_before = run;
    }
    if (x > 0.0 && run + x > bound) {
      at = i;
      before = run;
    }
    run += x;
  }
  if (at < 0) {
    at = last;
    before = last_before;
  }
  if (at != slot) return;
  const T* pr = target + node * a.target_stride[1];
  const T* qr = draft + node * a.draft_stride[1];
  int64_t token = -1, positive = -1;
  run = before;
  for (int64_t v = v0; v < v1; v += 32) {
    const double r = v + lane < v1 ? rest_of(wide(pr[v + lane]), c != 0.0 ? wide(qr[v + lane]) : 0.f, c) : 0.0;
    double s = r;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += x;
    }
    const unsigned over = __ballot_sync(0xffffffffu, r > 0.0 && run + s > bound), some = __ballot_sync(0xffffffffu, r > 0.0);
    if (some) positive = v + 31 - __clz(some);
    if (over) {
      token = v + __ffs(over) - 1;
      break;
    }
    run += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) a.next_token[b] = token >= 0 ? token : positive;
}

template <typename T>
int launch_verify(const fa_verify_args& a, cudaStream_t st) {
  // shares of a few hundred tokens at least
  int cluster = 1;
  while (cluster < kMaxCluster && a.vocab > (int64_t)cluster * kThreads * 4) cluster *= 2;
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  lc.gridDim = dim3((unsigned)a.batch * cluster);
  lc.blockDim = dim3(kThreads);
  lc.stream = st;
  lc.attrs = &attr;
  lc.numAttrs = 1;
  cudaLaunchKernelEx(&lc, verify_kernel<T>, a);
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
