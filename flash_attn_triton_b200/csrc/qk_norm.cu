// RMS norm of every head of q and k with the rotation by the token's position in the same pass, and its gradients.
//
//   Mathematics.  r = rsqrt(mean(x^2) + eps), y = x r w, out = R y with R the rotation of the pairs.  R is orthogonal, so g = R^T dout; then
//   dw = sum g x r, and with h = g w:  dx = r (h - x r^2 mean(h x)).  Both means of the backward pass are sums over the head that do not wait
//   for one another.
//   Bound.  HBM: forward 2, backward 3 words an element.  D / 8 lanes have a head and 8 elements each: the two halves of four pairs (rotate-half), 8
//   in a row otherwise.  Its sums are shuffles.  A group of lanes has an even share of all heads of all tokens, one after another, with a token's
//   angles in registers, first of q and then of k, so that a thread has one set of weights and sums at a time and divides only where its
//   share begins.  Every thread has a ring of its own in shared memory that its loads go to (cp.async, 128 bytes in flight), so that no
//   barrier is needed and registers do not bound the loads in flight.  16380 tokens of 40 heads of 128, bf16, forward 58 to 60 us, 0.86 of the copy rate,
//   backward 89, 0.86, what is left being instructions (two thirds of the issue slots): with four loads in registers and partners from another lane 69 and 110.
//   Weight gradients: a thread's sums over its heads, those of a CTA through shared memory, those of the CTAs by a second kernel in
//   order.  The grid depends on the sizes and the GPU alone, so the result does not change from call to call.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace fa {

namespace {

constexpr int kThreads = 256;

template <typename T> struct Raw { uint4 v; };
template <> struct Raw<float> { float4 a, b; };

// Two numbers of a word.  (bf16: the upper halves of fp32 numbers.  __bfloat1622float2 takes two or three instructions for each.)
template <typename T> __device__ __forceinline__ float2 pair_of(uint32_t w) { return Elem<T>::unpack(w); }
template <> __device__ __forceinline__ float2 pair_of<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ void widen(const Raw<T>& r, float (&x)[8]) {
  const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = pair_of<T>(w[i]);
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
// The same as four pairs.
template <typename T> __device__ __forceinline__ void pairs_of(const Raw<T>& r, float2 (&x)[4]) {
  const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pair_of<T>(w[i]);
}
template <> __device__ __forceinline__ void pairs_of(const Raw<float>& r, float2 (&x)[4]) {
  x[0] = make_float2(r.a.x, r.a.y);
  x[1] = make_float2(r.a.z, r.a.w);
  x[2] = make_float2(r.b.x, r.b.y);
  x[3] = make_float2(r.b.z, r.b.w);
}
// To p and, the second four, to p + off.
template <bool kApart, typename T> __device__ __forceinline__ void store_pairs(T* p, int off, const float2 (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
    *reinterpret_cast<float4*>(p + off) = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
  } else {
    const uint2 a = make_uint2(Elem<T>::pack(x[0].x, x[0].y), Elem<T>::pack(x[1].x, x[1].y));
    const uint2 b = make_uint2(Elem<T>::pack(x[2].x, x[2].y), Elem<T>::pack(x[3].x, x[3].y));
    if constexpr (kApart) {
      *reinterpret_cast<uint2*>(p) = a;
      *reinterpret_cast<uint2*>(p + off) = b;
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
}
// The other element of each pair of a lane's 8: next to it, or four further on.  unpaired: elements that are not rotated (0 times their neighbour, an
// infinity, would be no number).
template <bool kSideBySide> __device__ __forceinline__ void others_of(const float2 (&x)[4], float2 (&z)[4], bool unpaired) {
#pragma unroll
  for (int e = 0; e < 4; ++e) z[e] = kSideBySide ? make_float2(x[e].y, x[e].x) : x[e ^ 2];
  if (unpaired) {
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = make_float2(0.f, 0.f);
  }
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

// Four numbers of a table, aligned to their size.
template <typename T> __device__ __forceinline__ void entries(const void* p, int wide, int64_t i, float (&x)[8]) {
  if (wide) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else if constexpr (sizeof(T) == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const T*>(p) + i);
    const float2 a = Elem<T>::unpack(v.x), b = Elem<T>::unpack(v.y);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  }
}

// The rotation of this lane's 8 elements of a head -- from d on, or whole halves: four from d on and their partners --, as cos and sin per element; those behind rotary_dim have cos = 1,
// sin = 0.  The sign of the sine is that of the forward rotation of the element: out = y cos + (its pair's y) sin.
template <typename T>
__device__ __forceinline__ void angles(const fa_qk_norm_args& p, bool whole, int64_t pos, int d, float (&c)[8], float (&s)[8]) {
  const int half = p.rotary_dim >> 1;
  if (p.cos == nullptr || pos < 0 || pos >= p.rotary_seqlen || d >= p.rotary_dim) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = 1.f;
      s[e] = 0.f;
    }
    return;
  }
  if (whole) {                                   // 4 pairs with 4 entries in a row
    const int64_t i = pos * half + (p.interleaved ? d >> 1 : d);
    float x[8];
    entries<T>(p.cos, p.table_wide, i, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = p.interleaved ? x[e >> 1] : x[e & 3];
    entries<T>(p.sin, p.table_wide, i, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = p.interleaved ? (e & 1 ? x[e >> 1] : -x[e >> 1]) : (e & 4 ? x[e & 3] : -x[e & 3]);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int j = d + e;
    c[e] = 1.f;
    s[e] = 0.f;
    if (j < p.rotary_dim) {
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

// One of q and k.
struct Side {
  const void* x;
  const void* g;                                 // backward: the gradient of the result
  void* out;                                     // the result; backward: the gradient of x
  const void* weight;
  int64_t xs[3], gs[3], os[3];
  int heads;
  bool few;                                      // heads of all tokens: 32 bits count them
  int64_t share, more;                           // of a group, and how many groups have one more
};
struct Sides {
  Side side[2];
};

// The table rows of a position, on their way to L1.
__device__ __forceinline__ void prefetch_angles(const fa_qk_norm_args& p, int64_t pos, int d, int bytes) {
  const int half = p.rotary_dim >> 1;
  if (p.cos == nullptr || pos < 0 || pos >= p.rotary_seqlen || d >= half) return;
  const int64_t i = (pos * half + d) * bytes;
  asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const char*>(p.cos) + i));
  asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const char*>(p.sin) + i));
}

constexpr int kSlots = 8;                        // 16-byte slots of a thread's ring

// kTurn: whether a lane has four whole pairs (whole_lanes()): 8 elements in a row where a pair lies side by side, else four of the first half and
// the four that belong to them.  If it has, and with x' the other element of each pair, the forward is r (x (c w) + x' (s w')), the two products in brackets made
// once for all heads of a token, and all of it in pairs of fp32: element by element, 177 instructions for 8 elements of a lane bound the forward, 253 the
// backward.  Partners from another lane's 8 in a row took a shuffle and an unpacking more for each pair.
// kAll: the whole head is rotated.  ws: backward, D sums of every CTA for q, then for k.
enum Turn { kAnyhow, kHalves, kSideBySide };
template <typename T, int D, bool kBackward, Turn kTurn, bool kAll>
__global__ void __launch_bounds__(kThreads, kBackward ? 2 : 3) qk_norm_kernel(const fa_qk_norm_args p, const Sides sides, float* ws) {
  constexpr bool kWhole = kTurn != kAnyhow;
  constexpr int L = D / 8, G = kThreads / L;
  constexpr int W = sizeof(T) / 2, kOf = W * (kBackward ? 2 : 1), S = kSlots / kOf;      // slots of 8 elements, of a head; heads in flight
  __shared__ uint4 ring[kSlots][kThreads];
  __shared__ float rows[kWhole ? 1 : G][kWhole ? 1 : D];
  const int tid = threadIdx.x, group = tid / L, lane = tid % L;
  const int entry = p.table_wide ? 4 : (int)sizeof(T);
  // the lane's elements: d .. d + 3 and d + off .. d + off + 3
  constexpr bool kApart = kTurn == kHalves;
  const int half = p.rotary_dim >> 1;
  const int d = kApart && lane < half / 4 ? lane * 4 : kApart ? 2 * half + (lane - half / 4) * 8 : lane * 8;
  const int off = kApart && lane < half / 4 ? half : 4;
  const int64_t me = (int64_t)blockIdx.x * G + group;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const Side& a = sides.side[which];
    const int heads = a.heads;
    float2 w[4], wo[4], dw[4];                   // weights, those of the other elements of the pairs
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = d + (e & 1) * 2 + (e >> 1) * off;
      w[e] = a.weight ? make_float2(at<T>(a.weight, p.weight_wide, i), at<T>(a.weight, p.weight_wide, i + 1)) : make_float2(1.f, 1.f);
      dw[e] = make_float2(0.f, 0.f);
    }
    others_of<kTurn == kSideBySide>(w, wo, false);
    // this group's heads: `mine` of them from `begin` on; the groups of a warp stay together for `steps`
    const int64_t begin = a.share * me + (me < a.more ? me : a.more);
    const int mine = (int)a.share + (me < a.more), steps = (int)a.share + (a.more > 0);
    int b0 = 0, t0 = 0, h0 = 0;
    if (a.few) {                                 // (64-bit divisions take a hundred instructions each)
      const uint32_t token = (uint32_t)begin / (uint32_t)max(heads, 1);
      h0 = (int)((uint32_t)begin - token * heads);
      b0 = (int)(token / (uint32_t)p.seqlen);
      t0 = (int)(token - (uint32_t)b0 * p.seqlen);
    } else {
      const int64_t token = begin / heads;
      h0 = (int)(begin - token * heads);
      b0 = (int)(token / p.seqlen);
      t0 = (int)(token - (int64_t)b0 * p.seqlen);
    }

    // loading: S heads ahead of their use
    const int64_t xh = a.xs[2], gh = a.gs[2], oh = a.os[2];
    int lb = b0, lt = t0, asked = 0, ask_end = heads - h0;       // steps, the one with which the token ends
    const T* lx = static_cast<const T*>(a.x) + lb * a.xs[0] + lt * a.xs[1] + h0 * xh + d;
    const T* lg = kBackward ? static_cast<const T*>(a.g) + lb * a.gs[0] + lt * a.gs[1] + h0 * gh + d : nullptr;
    constexpr uint32_t kPitch = kThreads * 16;
    const uint32_t own = smem_u32(&ring[0][tid]);
    uint32_t turn = 0;                           // of the ring: bytes from this thread's first slot
    auto fetch = [&](uint32_t to, const T* from) {
      if constexpr (W == 2) {
        cp_async16(to, from, 16);
        cp_async16(to + kPitch, from + off, 16);
      } else if constexpr (kApart) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(to), "l"(from) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(to + 8), "l"(from + off) : "memory");
      } else {
        cp_async16(to, from, 16);
      }
    };
    auto ask = [&](uint32_t to) {
      if (asked < mine) {
        fetch(to, lx);
        if (kBackward) fetch(to + W * kPitch, lg);
        lx += xh;
        if (kBackward) lg += gh;
        if (++asked == ask_end) {
          ask_end += heads;
          if (++lt == p.seqlen) {
            lt = 0;
            ++lb;
          }
          lx = static_cast<const T*>(a.x) + lb * a.xs[0] + lt * a.xs[1] + d;
          if (kBackward) lg = static_cast<const T*>(a.g) + lb * a.gs[0] + lt * a.gs[1] + d;
        }
      }
      cp_async_commit();
    };
    auto word = [&](uint32_t from) {
      uint4 v;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
      return v;
    };
    auto read = [&](uint32_t from) {
      Raw<T> r;
      if constexpr (sizeof(T) == 2) {
        r.v = word(from);
      } else {
        const uint4 v = word(from), u = word(from + kPitch);
        r.a = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
        r.b = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
      }
      return r;
    };
#pragma unroll
    for (int k = 0; k < S; ++k) ask(own + k * kOf * kPitch);

    int b = b0, t = t0;
    auto position_of = [&](int pb, int pt) {
      return p.positions ? (int64_t)p.positions[pb * p.pos_stride[0] + pt * p.pos_stride[1]] : (int64_t)pt;
    };
    float2 c[4], s[4];                           // of the token at hand; forward, whole lanes: times the weights
    auto turn_to = [&](int64_t pos) {
      float cs[8], sn[8];
      angles<T>(p, kWhole, pos, d, cs, sn);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[e] = make_float2(cs[2 * e], cs[2 * e + 1]);
        s[e] = make_float2(sn[2 * e], sn[2 * e + 1]);
        if constexpr (kWhole && !kBackward) {
          c[e] = f2mul(c[e], w[e]);
          s[e] = f2mul(s[e], wo[e]);
        }
      }
    };
    int64_t next_pos = 0;
    T* out = static_cast<T*>(a.out) + b * a.os[0] + t * a.os[1] + h0 * oh + d;
    if (mine > 0) turn_to(position_of(b, t));
    // steps with which this token ends, and with which something is to be done: the next token's angles are asked for four heads ahead
    int end = heads - h0, event = kWhole ? max(end - 4, 1) : end;
    bool known = false;                          // the next token's position
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      cp_async_wait<S - 1>();
      const Raw<T> xr = read(own + turn);
      Raw<T> gr;
      if (kBackward) gr = read(own + turn + W * kPitch);
      ask(own + turn);
      turn = (turn + kOf * kPitch) & (kSlots * kPitch - 1);
      const bool live = step < mine;
      if constexpr (kWhole && !kBackward) {
        float2 y[4], z[4], sq = make_float2(0.f, 0.f);
        pairs_of<T>(xr, y);
        others_of<kTurn == kSideBySide>(y, z, !kAll && d >= p.rotary_dim);
#pragma unroll
        for (int e = 0; e < 4; ++e) sq = f2fma(y[e], y[e], sq);
        const float r = rsqrtf(group_sum<L>(sq.x + sq.y) * (1.f / D) + p.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = f2mul(f2fma(z[e], s[e], f2mul(y[e], c[e])), make_float2(r, r));
        if (live) store_pairs<kApart>(out, off, y);
      } else if constexpr (kWhole) {
        float2 x[4], g[4], z[4], sq = make_float2(0.f, 0.f), hx = make_float2(0.f, 0.f);
        pairs_of<T>(xr, x);
        pairs_of<T>(gr, g);
        others_of<kTurn == kSideBySide>(g, z, !kAll && d >= p.rotary_dim);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[e] = f2fma(z[e], make_float2(-s[e].x, -s[e].y), f2mul(g[e], c[e]));     // rotated back
          z[e] = f2mul(g[e], x[e]);
          sq = f2fma(x[e], x[e], sq);
          hx = f2fma(z[e], w[e], hx);
        }
        const float r = rsqrtf(group_sum<L>(sq.x + sq.y) * (1.f / D) + p.eps);
        const float k = group_sum<L>(hx.x + hx.y) * (-1.f / D) * r * r * r;
        if (live) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            dw[e] = f2fma(z[e], make_float2(r, r), dw[e]);
            x[e] = f2fma(x[e], make_float2(k, k), f2mul(f2mul(g[e], w[e]), make_float2(r, r)));
          }
          store_pairs<kApart>(out, off, x);
        }
      } else {
        float x[8], g[8], z[8], sq = 0.f, hx = 0.f;
        widen<T>(xr, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) sq = fmaf(x[e], x[e], sq);
        const float r = rsqrtf(group_sum<L>(sq) * (1.f / D) + p.eps);
        auto one_of = [](const float2& v, int e) { return e & 1 ? v.y : v.x; };
        if constexpr (!kBackward) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] * r * one_of(w[e >> 1], e);
          partners<D>(p, lane, x, z, rows[kWhole ? 0 : group]);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] * one_of(c[e >> 1], e) + z[e] * one_of(s[e >> 1], e);
        } else {
          widen<T>(gr, g);
          partners<D>(p, lane, g, z, rows[kWhole ? 0 : group]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            g[e] = g[e] * one_of(c[e >> 1], e) - z[e] * one_of(s[e >> 1], e);      // rotated back
            hx = fmaf(g[e] * one_of(w[e >> 1], e), x[e], hx);
          }
          const float mean = group_sum<L>(hx) * (1.f / D) * r;                     // of h x r
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float unit = x[e] * r, gu = live ? g[e] * unit : 0.f;
            if (e & 1) dw[e >> 1].y = live ? dw[e >> 1].y + gu : dw[e >> 1].y;
            else dw[e >> 1].x = live ? dw[e >> 1].x + gu : dw[e >> 1].x;
            x[e] = r * (g[e] * one_of(w[e >> 1], e) - unit * mean);
          }
        }
        if (live) store8(out, x);
      }
      // on to the next head
      out += oh;
      if (step + 1 == event && event < mine) {
        const bool wraps = t + 1 == p.seqlen;
        if (event < end) {
          if (end < mine) {
            next_pos = position_of(b + wraps, wraps ? 0 : t + 1);
            known = true;
            prefetch_angles(p, next_pos, d, entry);
          }
          event = end;
        } else {
          t = wraps ? 0 : t + 1;
          b += wraps;
          out = static_cast<T*>(a.out) + b * a.os[0] + t * a.os[1] + d;
          turn_to(known ? next_pos : position_of(b, t));
          known = false;
          event = kWhole ? max(end + heads - 4, end + 1) : end + heads;
          end += heads;
        }
      }
      __syncwarp();
    }
    cp_async_wait<0>();
    if (!kBackward || ws == nullptr) continue;
    // over the ring: every group's sums, 8 KB
    __syncthreads();
    float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(sums + group * D + d + (e & 1) * 2 + (e >> 1) * off) = dw[e];
    __syncthreads();
    for (int i = tid; i < D; i += kThreads) {
      float sum = 0.f;
      for (int g = 0; g < G; ++g) sum += sums[g * D + i];
      ws[((int64_t)which * gridDim.x + blockIdx.x) * D + i] = sum;
    }
    __syncthreads();
  }
}

// The sums of all CTAs, one warp an element.
template <typename T>
__global__ void __launch_bounds__(kThreads) qk_norm_dw_kernel(const float* ws, int ctas, int D, void* dq, void* dk, int wide) {
  const int i = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= 2 * D) return;
  float sum = 0.f;
  for (int c = lane; c < ctas; c += 32) sum += ws[((int64_t)(i / D) * ctas + c) * D + i % D];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  void* out = i < D ? dq : dk;
  if (lane != 0 || out == nullptr) return;
  if (wide) static_cast<float*>(out)[i % D] = sum;
  else static_cast<T*>(out)[i % D] = narrow<T>(sum);
}

// As many CTAs as run at a time, fewer where there is not a head for every group of lanes.
int grid_of(const fa_qk_norm_args& a, bool backward) {
  const int groups = kThreads / (a.head_dim / 8);
  const int64_t need = ((int64_t)a.batch * a.seqlen * std::max(a.heads_q, a.heads_kv) + groups - 1) / groups, fit = (backward ? 2ll : 3ll) * sm_count(a.device);
  return (int)(need < fit ? need : fit);
}
// The 8 elements of a lane are four pairs: see angles().
bool whole_lanes(const fa_qk_norm_args& a) {
  const int half = a.rotary_dim / 2;
  return half % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) & 15) == 0 &&
         (a.dtype != FA_F32 || a.table_wide);
}

template <typename T, int D> int run(const fa_qk_norm_args& a, bool backward, cudaStream_t st) {
  Sides sides = {};
  for (int i = 0; i < 2; ++i) {
    Side& s = sides.side[i];
    s.heads = i ? a.heads_kv : a.heads_q;
    s.x = i ? a.k : a.q;
    s.g = i ? a.d_ko : a.d_qo;
    s.out = backward ? (i ? a.d_k : a.d_q) : (i ? a.k_out : a.q_out);
    s.weight = i ? a.k_weight : a.q_weight;
    for (int d = 0; d < 3; ++d) {
      s.xs[d] = (i ? a.k_stride : a.q_stride)[d];
      s.gs[d] = (i ? a.d_ko_stride : a.d_qo_stride)[d];
      s.os[d] = backward ? (i ? a.d_k_stride : a.d_q_stride)[d] : (i ? a.ko_stride : a.qo_stride)[d];
    }
  }
  const bool whole = whole_lanes(a);
  const int grid = grid_of(a, backward);
  for (Side& s : sides.side) {
    const int64_t all = (int64_t)a.batch * a.seqlen * s.heads, groups = (int64_t)grid * (kThreads / (D / 8));
    s.few = all <= UINT32_MAX;
    s.share = all / groups;
    s.more = all % groups;
  }
  float* ws = backward && (a.d_q_weight || a.d_k_weight) ? static_cast<float*>(a.workspace) : nullptr;
  auto launch = [&](auto kernel) { kernel<<<grid, kThreads, 0, st>>>(a, sides, ws); };
  auto turned = [&](auto direction) {
    constexpr bool kBackward = decltype(direction)::value;
    const bool all = a.rotary_dim == D;
    if (!whole) launch(qk_norm_kernel<T, D, kBackward, kAnyhow, true>);
    else if (a.interleaved) all ? launch(qk_norm_kernel<T, D, kBackward, kSideBySide, true>) : launch(qk_norm_kernel<T, D, kBackward, kSideBySide, false>);
    else all ? launch(qk_norm_kernel<T, D, kBackward, kHalves, true>) : launch(qk_norm_kernel<T, D, kBackward, kHalves, false>);
  };
  if (backward) turned(std::true_type{});
  else turned(std::false_type{});
  if (int r = check_launch(backward ? "qk_norm_bwd" : "qk_norm")) return r;
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
  return (size_t)grid_of(a, true) * 2 * a.head_dim * sizeof(float);
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
