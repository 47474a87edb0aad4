// RMS norm of every head of q and k with the rotation by the token's position in the same pass, and its gradients.
//
//   Mathematics.  r = rsqrt(mean(x^2) + eps), y = x r w, out = R y with R the rotation of the pairs.  R is orthogonal, so g = R^T dout; then
//   dw = sum g x r, and with h = g w:  dx = r (h - x r^2 mean(h x)).  Both means of the backward pass are sums over the head that do not wait
//   for one another.
//   Bound.  HBM: forward 2, backward 3 words an element.  D / 8 lanes have a head and 8 elements each, 16 bytes of a 16-bit type, so that a
//   head is one access, its sums are shuffles, and a pair's other half (rotate-half) comes from another lane of the head.  A group of
//   lanes takes several heads of a token, one after another, with the token's angles in registers.
//   Weight gradients: a thread's sums over its heads, those of a CTA through shared memory, those of the CTAs by a second kernel in
//   order.  The grid depends on the sizes and the GPU alone, so the result does not change from call to call.
#include "common.cuh"

namespace fa {

namespace {

constexpr int kThreads = 256;

template <typename T> struct Raw { uint4 v; };
template <> struct Raw<float> { float4 a, b; };

template <typename T> __device__ __forceinline__ Raw<T> load8(const T* p) { return Raw<T>{*reinterpret_cast<const uint4*>(p)}; }
template <> __device__ __forceinline__ Raw<float> load8(const float* p) {
  return Raw<float>{reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
}
template <typename T> __device__ __forceinline__ void widen(const Raw<T>& r, float (&x)[8]) {
  const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::unpack(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <> __device__ __forceinline__ void widen(const Raw<float>& r, float (&x)[8]) {
  x[0] = r.a.x; x[1] = r.a.y; x[2] = r.a.z; x[3] = r.a.w;
  x[4] = r.b.x; x[5] = r.b.y; x[6] = r.b.z; x[7] = r.b.w;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 v;
  v.x = Elem<T>::pack(x[0], x[1]);
  v.y = Elem<T>::pack(x[2], x[3]);
  v.z = Elem<T>::pack(x[4], x[5]);
  v.w = Elem<T>::pack(x[6], x[7]);
  *reinterpret_cast<uint4*>(p) = v;
}
template <> __device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <typename T> __device__ __forceinline__ float one(const T* p);
template <> __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
template <> __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <> __device__ __forceinline__ float one(const float* p) { return *p; }
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ __half narrow(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float narrow(float x) { return x; }

// element i of a vector of T or, `wide`, of fp32
template <typename T> __device__ __forceinline__ float at(const void* p, int wide, int64_t i) {
  return wide ? static_cast<const float*>(p)[i] : one(static_cast<const T*>(p) + i);
}

// How a call is cut: groups of lanes take `heads` heads of a token each, `chunks` of them a token.
struct Cut {
  int heads, chunks;
  int64_t items;
};

// The rotation of this lane's 8 elements d .. d + 7 of a head, as cos and sin per element; elements behind rotary_dim have cos = 1,
// sin = 0.  The sign of the sine is that of the forward rotation of the element: out = y cos + (its pair's y) sin.
template <typename T>
__device__ __forceinline__ void angles(const fa_qk_norm_args& p, int64_t pos, int d, float (&c)[8], float (&s)[8]) {
  const int half = p.rotary_dim >> 1;
  const bool turned = p.cos != nullptr && pos >= 0 && pos < p.rotary_seqlen;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int j = d + e;
    c[e] = 1.f;
    s[e] = 0.f;
    if (turned && j < p.rotary_dim) {
      const bool first = p.interleaved ? (j & 1) == 0 : j < half;
      const int64_t i = pos * half + (p.interleaved ? j >> 1 : first ? j : j - half);
      c[e] = at<T>(p.cos, p.table_wide, i);
      const float x = at<T>(p.sin, p.table_wide, i);
      s[e] = first ? -x : x;
    }
  }
}

// The other element of each pair.  row: this group's own D floats of shared memory, for pairs that do not lie whole lanes apart.
template <int D>
__device__ __forceinline__ void partners(const fa_qk_norm_args& p, int lane_in_group, const float (&y)[8], float (&z)[8], float* row) {
  constexpr int L = D / 8;
  if (p.interleaved) {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = y[e ^ 1];
    return;
  }
  const int half = p.rotary_dim >> 1, d = lane_in_group * 8;
  if (half % 8 == 0) {
    const int other = d < half ? lane_in_group + half / 8 : d < p.rotary_dim ? lane_in_group - half / 8 : lane_in_group;
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = __shfl_sync(0xffffffffu, y[e], other, L);
    return;
  }
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 8; ++e) row[d + e] = y[e];
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int j = d + e;
    z[e] = j < half ? row[j + half] : j < p.rotary_dim ? row[j - half] : y[e];
  }
}

template <int L> __device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

struct Weights {
  float q[8], k[8];
};
template <typename T> __device__ __forceinline__ Weights weights_of(const fa_qk_norm_args& p, int d) {
  Weights w;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    w.q[e] = p.q_weight ? at<T>(p.q_weight, p.weight_wide, d + e) : 1.f;
    w.k[e] = p.k_weight ? at<T>(p.k_weight, p.weight_wide, d + e) : 1.f;
  }
  return w;
}

template <typename T>
__device__ __forceinline__ const T* row_of(const void* q, const void* k, const int64_t* qs, const int64_t* ks, int heads_q, int b, int t, int h) {
  return h < heads_q ? static_cast<const T*>(q) + b * qs[0] + t * qs[1] + h * qs[2]
                     : static_cast<const T*>(k) + b * ks[0] + t * ks[1] + (h - heads_q) * ks[2];
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) qk_norm_kernel(const fa_qk_norm_args p, const Cut cut) {
  constexpr int L = D / 8, G = kThreads / L, kU = 4;
  __shared__ float rows[G][D];
  const int group = threadIdx.x / L, lane = threadIdx.x % L, d = lane * 8;
  const int heads = p.heads_q + p.heads_kv;
  const Weights w = weights_of<T>(p, d);
  // (the lanes of a warp stay together: groups without work do what their neighbours do, and store nothing)
  for (int64_t base = (int64_t)blockIdx.x * G; base < cut.items; base += (int64_t)gridDim.x * G) {
    const bool mine = base + group < cut.items;
    const int64_t item = mine ? base + group : cut.items - 1;
    const int64_t token = item / cut.chunks;
    const int h0 = (int)(item - token * cut.chunks) * cut.heads, h1 = min(heads, h0 + cut.heads);
    const int b = (int)(token / p.seqlen), t = (int)(token - (int64_t)b * p.seqlen);
    float c[8], s[8];
    angles<T>(p, p.positions ? (int64_t)p.positions[b * p.pos_stride[0] + t * p.pos_stride[1]] : t, d, c, s);
    for (int j0 = 0; j0 < cut.heads; j0 += kU) {
      Raw<T> x[kU];
#pragma unroll
      for (int j = 0; j < kU; ++j)
        if (j0 + j < cut.heads) x[j] = load8(row_of<T>(p.q, p.k, p.q_stride, p.k_stride, p.heads_q, b, t, min(h0 + j0 + j, h1 - 1)) + d);
#pragma unroll
      for (int j = 0; j < kU; ++j) {
        if (j0 + j >= cut.heads) break;
        const int h = min(h0 + j0 + j, h1 - 1);
        float y[8], z[8];
        widen<T>(x[j], y);
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sq = fmaf(y[e], y[e], sq);
        const float r = rsqrtf(group_sum<L>(sq) * (1.f / D) + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = y[e] * r * (h < p.heads_q ? w.q[e] : w.k[e]);
        partners<D>(p, lane, y, z, rows[group]);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = y[e] * c[e] + z[e] * s[e];
        if (mine && h0 + j0 + j < h1)
          store8(const_cast<T*>(row_of<T>(p.q_out, p.k_out, p.qo_stride, p.ko_stride, p.heads_q, b, t, h)) + d, y);
      }
    }
  }
}

// ws: 2 D sums of every CTA
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) qk_norm_bwd_kernel(const fa_qk_norm_args p, const Cut cut, float* ws) {
  constexpr int L = D / 8, G = kThreads / L, kU = 2;
  __shared__ float rows[G][D];
  const int group = threadIdx.x / L, lane = threadIdx.x % L, d = lane * 8;
  const int heads = p.heads_q + p.heads_kv;
  const Weights w = weights_of<T>(p, d);
  float dwq[8], dwk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dwq[e] = dwk[e] = 0.f;
  for (int64_t base = (int64_t)blockIdx.x * G; base < cut.items; base += (int64_t)gridDim.x * G) {
    const bool mine = base + group < cut.items;
    const int64_t item = mine ? base + group : cut.items - 1;
    const int64_t token = item / cut.chunks;
    const int h0 = (int)(item - token * cut.chunks) * cut.heads, h1 = min(heads, h0 + cut.heads);
    const int b = (int)(token / p.seqlen), t = (int)(token - (int64_t)b * p.seqlen);
    float c[8], s[8];
    angles<T>(p, p.positions ? (int64_t)p.positions[b * p.pos_stride[0] + t * p.pos_stride[1]] : t, d, c, s);
    for (int j0 = 0; j0 < cut.heads; j0 += kU) {
      Raw<T> xr[kU], gr[kU];
#pragma unroll
      for (int j = 0; j < kU; ++j) {
        if (j0 + j >= cut.heads) break;
        const int h = min(h0 + j0 + j, h1 - 1);
        xr[j] = load8(row_of<T>(p.q, p.k, p.q_stride, p.k_stride, p.heads_q, b, t, h) + d);
        gr[j] = load8(row_of<T>(p.d_qo, p.d_ko, p.d_qo_stride, p.d_ko_stride, p.heads_q, b, t, h) + d);
      }
#pragma unroll
      for (int j = 0; j < kU; ++j) {
        if (j0 + j >= cut.heads) break;
        const int h = min(h0 + j0 + j, h1 - 1);
        const bool live = mine && h0 + j0 + j < h1;
        float x[8], g[8], z[8];
        widen<T>(xr[j], x);
        widen<T>(gr[j], g);
        partners<D>(p, lane, g, z, rows[group]);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = g[e] * c[e] - z[e] * s[e];      // rotated back
        float sq = 0.f, hx = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sq = fmaf(x[e], x[e], sq);
          hx = fmaf(g[e] * (h < p.heads_q ? w.q[e] : w.k[e]), x[e], hx);
        }
        const float r = rsqrtf(group_sum<L>(sq) * (1.f / D) + p.eps);
        const float mean = group_sum<L>(hx) * (1.f / D) * r;               // of h x r
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float unit = x[e] * r, gu = g[e] * unit;
          if (live) (h < p.heads_q ? dwq[e] : dwk[e]) += gu;
          x[e] = r * (g[e] * (h < p.heads_q ? w.q[e] : w.k[e]) - unit * mean);
        }
        if (live) store8(const_cast<T*>(row_of<T>(p.d_q, p.d_k, p.d_q_stride, p.d_k_stride, p.heads_q, b, t, h)) + d, x);
      }
    }
  }
  if (ws == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) rows[group][d + e] = which ? dwk[e] : dwq[e];
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += kThreads) {
      float sum = 0.f;
      for (int g = 0; g < G; ++g) sum += rows[g][i];
      ws[((int64_t)blockIdx.x * 2 + which) * D + i] = sum;
    }
  }
}

// The sums of all CTAs, one warp an element.
template <typename T>
__global__ void __launch_bounds__(kThreads) qk_norm_dw_kernel(const float* ws, int ctas, int D, void* dq, void* dk, int wide) {
  const int i = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= 2 * D) return;
  float sum = 0.f;
  for (int c = lane; c < ctas; c += 32) sum += ws[(int64_t)c * 2 * D + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  void* out = i < D ? dq : dk;
  if (lane != 0 || out == nullptr) return;
  if (wide) static_cast<float*>(out)[i % D] = sum;
  else static_cast<T*>(out)[i % D] = narrow<T>(sum);
}

constexpr int kBwdPerSm = 4;

Cut cut_of(const fa_qk_norm_args& a) {
  const int heads = a.heads_q + a.heads_kv, groups = kThreads / (a.head_dim / 8);
  const int64_t tokens = (int64_t)a.batch * a.seqlen;
  // eight heads of a token, fewer while that leaves SMs idle
  Cut c;
  c.heads = 8;
  while (c.heads > 1 && tokens * ((heads + c.heads - 1) / c.heads) < (int64_t)groups * 2 * sm_count(a.device)) c.heads /= 2;
  c.chunks = (heads + c.heads - 1) / c.heads;
  c.items = tokens * c.chunks;
  return c;
}

int grid_of(const fa_qk_norm_args& a, const Cut& c, int per_sm) {
  const int64_t groups = kThreads / (a.head_dim / 8), need = (c.items + groups - 1) / groups, fit = (int64_t)per_sm * sm_count(a.device);
  return (int)(need < fit ? need : fit);
}

template <typename T, int D> int run(const fa_qk_norm_args& a, bool backward, cudaStream_t st) {
  const Cut c = cut_of(a);
  if (!backward) {
    qk_norm_kernel<T, D><<<grid_of(a, c, 64), kThreads, 0, st>>>(a, c);
    return check_launch("qk_norm");
  }
  const int grid = grid_of(a, c, kBwdPerSm);
  float* ws = a.d_q_weight || a.d_k_weight ? static_cast<float*>(a.workspace) : nullptr;
  qk_norm_bwd_kernel<T, D><<<grid, kThreads, 0, st>>>(a, c, ws);
  if (int r = check_launch("qk_norm_bwd")) return r;
  if (ws == nullptr) return FA_OK;
  qk_norm_dw_kernel<T><<<2 * D / (kThreads / 32), kThreads, 0, st>>>(ws, grid, D, a.d_q_weight, a.d_k_weight, a.weight_wide);
  return check_launch("qk_norm_dw");
}

template <typename T> int run_dim(const fa_qk_norm_args& a, bool backward, cudaStream_t st) {
  switch (a.head_dim) {
    case 16: return run<T, 16>(a, backward, st);
    case 32: return run<T, 32>(a, backward, st);
    case 64: return run<T, 64>(a, backward, st);
    case 128: return run<T, 128>(a, backward, st);
    default: return run<T, 256>(a, backward, st);
  }
}

}  // namespace

size_t qk_norm_bwd_workspace_bytes(const fa_qk_norm_args& a) {
  if ((int64_t)a.batch * a.seqlen == 0) return 0;
  return (size_t)grid_of(a, cut_of(a), kBwdPerSm) * 2 * a.head_dim * sizeof(float);
}

int qk_norm(const fa_qk_norm_args& a, bool backward, cudaStream_t st) {
  if ((int64_t)a.batch * a.seqlen == 0) {
    const size_t bytes = a.head_dim * (a.weight_wide || a.dtype == FA_F32 ? 4 : 2);
    for (void* w : {a.d_q_weight, a.d_k_weight})
      if (backward && w != nullptr && cudaMemsetAsync(w, 0, bytes, st) != cudaSuccess) {
        set_error("qk_norm: cudaMemsetAsync: %s", cudaGetErrorString(cudaGetLastError()));
        return FA_ERR_LAUNCH;
      }
    return FA_OK;
  }
  if (a.dtype == FA_F16) return run_dim<__half>(a, backward, st);
  if (a.dtype == FA_BF16) return run_dim<__nv_bfloat16>(a, backward, st);
  return run_dim<float>(a, backward, st);
}

}  // namespace fa
