// Codes of the 8-bit KV cache: to 16-bit floats for the tensor cores, and from floats.
#pragma once
#include "cache8_host.h"
#include "cache_dev.cuh"
#include "cache_geo.cuh"

namespace fa {

// Every code of either kind is a 16-bit float exactly: whole numbers up to 255, or 4 significant bits from 2^-9 to 448.  (The products are
// therefore taken in fp16 whatever the type of the queries; bf16 queries are brought into its range by a power of two.)
template <int kCode> struct Code;

template <> struct Code<FA_CODE_INT8> {
  static constexpr float kLargest = 127.f;
  // Keys of the decode kernel (neighbours): a byte in the low half of a 16-bit float is u * 2^-24 (u = code + 128), one byte permutation per
  // pair.  The products are then 2^-24 of the true ones and too large by those with kBias.
  static constexpr float kUnit = 0x1p-24f;
  static constexpr uint32_t kBias = 0x00800080u;
  static __device__ __forceinline__ uint32_t pair(uint32_t x, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(sel));
    return r;
  }
  // bytes (0, 1) and (2, 3) of x as pairs
  static __device__ __forceinline__ void neighbours(uint32_t x, uint32_t& a, uint32_t& b) {
    x ^= 0x80808080u;
    a = pair(x, 0x4140);
    b = pair(x, 0x4342);
  }
  // bytes as they are, without the factor and the bias: 0x6400 | u is 1024 + u
  static __device__ __forceinline__ uint32_t whole(uint32_t x, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0x64646464u), "r"(sel));
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64806480u));
    return r;
  }
  // (0, 1) and (2, 3)
  static __device__ __forceinline__ void integers(uint32_t x, uint32_t& a, uint32_t& b) {
    x ^= 0x80808080u;
    a = whole(x, 0x4140);
    b = whole(x, 0x4342);
  }
  // (0, 2) and (1, 3)
  static __device__ __forceinline__ void alternate(uint32_t x, uint32_t& a, uint32_t& b) {
    x ^= 0x80808080u;
    a = whole(x, 0x4240);
    b = whole(x, 0x4341);
  }
  // four codes of x[i] * m.  Adding 1.5 * 2^23 leaves the number rounded half to even in the low byte.
  static __device__ __forceinline__ uint32_t four(float a, float b, float c, float d, float m) {
    const float magic = 12582912.f;
    const uint32_t ia = __float_as_uint(__fadd_rn(__fmul_rn(a, m), magic)), ib = __float_as_uint(__fadd_rn(__fmul_rn(b, m), magic));
    const uint32_t ic = __float_as_uint(__fadd_rn(__fmul_rn(c, m), magic)), id = __float_as_uint(__fadd_rn(__fmul_rn(d, m), magic));
    return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
  }
  static __device__ __forceinline__ void floats(uint32_t x, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(x >> (8 * i));
  }
};

template <> struct Code<FA_CODE_E4M3> {
  static constexpr float kLargest = 448.f;
  static constexpr float kUnit = 1.f;
  static constexpr uint32_t kBias = 0u;
  static __device__ __forceinline__ uint32_t pair(uint16_t x) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(x));
    return r;
  }
  static __device__ __forceinline__ void neighbours(uint32_t x, uint32_t& a, uint32_t& b) {
    a = pair((uint16_t)x);
    b = pair((uint16_t)(x >> 16));
  }
  static __device__ __forceinline__ void integers(uint32_t x, uint32_t& a, uint32_t& b) { neighbours(x, a, b); }
  static __device__ __forceinline__ void alternate(uint32_t x, uint32_t& a, uint32_t& b) {
    neighbours(__byte_perm(x, 0u, 0x3120), a, b);
  }
  static __device__ __forceinline__ uint32_t four(float a, float b, float c, float d, float m) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(__fmul_rn(a, m)), "f"(__fmul_rn(b, m)));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(__fmul_rn(c, m)), "f"(__fmul_rn(d, m)));
    return (uint32_t)lo | ((uint32_t)hi << 16);
  }
  static __device__ __forceinline__ void floats(uint32_t x, float (&f)[4]) {
    uint32_t a, b;
    neighbours(x, a, b);
    const float2 p = Elem<__half>::unpack(a), q = Elem<__half>::unpack(b);
    f[0] = p.x; f[1] = p.y; f[2] = q.x; f[3] = q.y;
  }
};

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src));
}

// log2 of a power of two, else -1
inline int log2_of(int n) {
  if (n <= 0 || (n & (n - 1)) != 0) return -1;
  int s = 0;
  while ((1 << s) < n) ++s;
  return s;
}
// x / n for 0 <= x < 2^31 by one product: m = ceil(2^(31 + l) / n) with 2^l >= n is too large by less than n / 2^31 of itself.
__device__ __forceinline__ int divided(int x, const Div32& d) { return (int)(((uint64_t)(uint32_t)x * d.m) >> d.shift); }
__device__ __forceinline__ int divided(int x, int n, int shift) { return shift >= 0 ? x >> shift : x / n; }

// Chunks of tokens: pieces that `all` key tiles of a unit are cut into.  A piece has the tiles that an SM would have if all work were
// shared evenly, so that sequences longer than that do not set the time (32 heads over 8 of 128, whole units -> cut: 100 tokens behind
// 30000 563 -> 146 us, 3 x 256 behind 300 to 30000 571 -> 534, 4 x 256 behind 1024 to 8192 197 -> 201).  Every warp works it out from
// the lengths; units: of a sequence.
__device__ __forceinline__ int chunk_pieces(const fa_decode_args& p, const ScoreCfg& cfg, const CacheGeo& geo, int units, int all, int lane) {
  if (geo.parts == 1) return 1;
  int64_t tiles = 0;
  for (int b = lane; b < p.batch; b += 32) {
    const int cap = seq_capacity(p, b);
    int keys = min(max(0, min(geo.seqlens[b], cap)) + geo.n_new, cap);
    if (cfg.wl >= 0) keys = min(keys, cfg.wl + geo.tokens + 127);
    tiles += (keys + 127) / 128;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
  const int even = max(4, (int)((tiles * units + geo.sms - 1) / geo.sms));
  return max(1, min(min(geo.parts, all), (all + even - 1) / even));
}

}  // namespace fa
