// New keys and values into the 8-bit KV cache: packed tokens by slot, or the new tokens of a cache call.
//
//   Mathematics.  For each block of tokens and head: need = largest |x| / Q, s' = s where |s| >= need, else need, codes rn(x / s'), and where
//   the scale grows the codes that the block keeps are rounded again to it.  (fa_b200.h has the exact form.)
//   Bound.  HBM: 2 bytes read and 1 written per element.  A sum over rows is not needed, only a maximum, so the values of a block and
//   head stay in registers between the maximum and the codes and are read once.
//   Split.  A run is the tokens of a call that fall into one block.  A CTA looks at `span` tokens, lists the runs that begin among
//   them, and its warps take (run, head, key or value) one by one; 1 to 8 warps share one by the size of a block, so that each lane
//   has at most 8 or 16 16-byte pieces of it.  Nothing is left to atomics: a block belongs to one run, and a run and head to one group of warps.
//   Measured: 302 k tokens of 8 heads of 128, int8, blocks of 32: 318 us, 5.8 TB/s of 6.5 (rounding and packing are 13 instructions
//   per element); 22 k, e4m3, blocks of 64: 34 us (floor 21); 32 single tokens: 5.5 us, all latency.
#include <type_traits>

#include "cache8.cuh"
#include "cache8_host.h"
#include "check_words.h"

namespace fa {

namespace {

constexpr int kThreads = 256;
constexpr int kSpanMost = 256, kBlockMost = 1024;
constexpr int kHeadWords = 4;          // of the value checks, in front of the bits of the blocks

// Row of a slot: page, block of the page, row of the block.
struct Place {
  int64_t page;
  int row, block, in_block;
};
__device__ __forceinline__ Place place_of(const Append8& p, int64_t slot) {
  Place w;
  w.page = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
  w.row = (int)(slot - w.page * p.page_size);
  w.block = divided(w.row, p.block, p.block_shift);
  w.in_block = w.row - w.block * p.block;
  return w;
}
// Packed tokens: the slot of token t, -1 for one that is passed over.
__device__ __forceinline__ int64_t slot_of(const Append8& p, int64_t t) {
  const int64_t s = p.slots[t];
  return s < (int64_t)p.num_pages * p.page_size ? s : -1;
}
// Whether token t (slot s) carries on the run of the token before it.
__device__ __forceinline__ bool carries_on(const Append8& p, int64_t t, int64_t s) {
  return s >= 0 && t > 0 && slot_of(p, t - 1) == s - 1 && place_of(p, s).in_block != 0;
}

// Cache call: position of token t = (b, tok) and its slot.
struct CallToken {
  int b, tok, old, pos;                // tokens of its sequence before the call; position, padding included
  int64_t slot;
};
__device__ __forceinline__ CallToken call_token(const Append8& p, const fa_decode_args& d, int64_t t) {
  CallToken c;
  c.b = (int)(t / d.seqlen_new);
  c.tok = (int)(t - (int64_t)c.b * d.seqlen_new);
  c.old = max(0, min(d.cache_seqlens[c.b], seq_capacity(d, c.b)));
  c.pos = c.old + c.tok + (d.cache_leftpad ? max(0, d.cache_leftpad[c.b]) : 0);
  c.slot = -1;
  if (c.pos < cache_capacity(d)) {
    const int pi = d.block_table ? divided(c.pos, p.page_size, p.page_shift) : 0;
    const int page = d.block_table ? d.block_table[(int64_t)c.b * d.block_table_stride + pi] : d.cache_batch_idx ? d.cache_batch_idx[c.b] : c.b;
    if ((unsigned)page < (unsigned)p.num_pages) c.slot = (int64_t)page * p.page_size + (c.pos - pi * p.page_size);
  }
  return c;
}

struct Run {
  int64_t token, slot;
  int n, kept;                         // tokens; those of the block that stay
};

}  // namespace

// kSlots: packed tokens; else those of the cache call d.  g.per_y (head, key or value) per CTA along y, 2^g.warps_log2 warps for one.
// kHeld: 16-byte pieces that a lane holds; a larger share of a block is read twice.
template <typename T, int kCode, bool kSlots, int kHeld>
__global__ void __launch_bounds__(kThreads, kHeld == 16 ? 2 : kSlots ? 4 : 3)
    cache8_append_kernel(const Append8 p, const fa_decode_args d, const AppendGeom g, uint32_t* host, uint32_t* dev, bool check_here) {
  using C = Code<kCode>;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (check_here) {
    const uint32_t bad = decode_checks(d, tid, kThreads);
    if (tid == 0 && blockIdx.x == 0 && blockIdx.y == 0) {
      *dev = bad;
      *reinterpret_cast<volatile uint32_t*>(host) = bad | kCheckDone;
      __threadfence_system();
    }
    if (bad) return;
  } else if (!kSlots && dev && *dev) {
    return;
  }
  __shared__ Run runs[kSpanMost];
  __shared__ uint32_t breaks[(kSpanMost + kBlockMost) / 32];
  __shared__ uint32_t part[2][8];
  __shared__ int nruns;
  if (tid == 0) nruns = 0;

  // ---- the runs that begin here --------------------------------------------------------------
  const int64_t t0 = (int64_t)blockIdx.x * g.span;
  const int here = (int)min((int64_t)g.span, p.tokens - t0);
  if (kSlots) {
    const int reach = (int)min((int64_t)here + p.block, p.tokens - t0);   // a run may end behind the span
    bool begins = false;
    int64_t mine = -1;
    for (int i = tid; i - lane < reach; i += kThreads) {
      int64_t s = -1;
      bool brk = true;
      if (i < reach) {
        s = slot_of(p, t0 + i);
        brk = !carries_on(p, t0 + i, s);
      }
      if (i < here) {
        begins = brk && s >= 0;
        mine = s;
      }
      const uint32_t word = __ballot_sync(0xffffffffu, brk);
      if (lane == 0) breaks[i >> 5] = word;
    }
    __syncthreads();
    if (begins) {
      // the next break behind this token
      int w = tid >> 5;
      uint32_t word = lane == 31 ? 0u : breaks[w] >> (lane + 1) << (lane + 1);
      while (word == 0u && ++w * 32 < reach) word = breaks[w];
      const int end = word ? min(reach, w * 32 + __ffs(word) - 1) : reach;
      runs[atomicAdd(&nruns, 1)] = Run{t0 + tid, mine, end - tid, place_of(p, mine).in_block};
    }
  } else {
    __syncthreads();
    if (tid < here) {
      const CallToken c = call_token(p, d, t0 + tid);
      if (c.slot >= 0) {
        const int at = place_of(p, c.slot).in_block;
        if (at == 0 || c.tok == 0)
          runs[atomicAdd(&nruns, 1)] = Run{t0 + tid, c.slot, min(min(p.block - at, d.seqlen_new - c.tok), cache_capacity(d) - c.pos),
                                           min(at, c.old + c.tok)};
      }
    }
  }
  __syncthreads();
  if (kSlots && dev) {
    // behind the checks (a programmatic launch): the runs were listed meanwhile (a call of 22 k tokens 46 us, 42.5)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (*dev) return;
  }

  // ---- (run, head, key or value) by groups of warps ---------------------------------------------
  const int wlog = g.warps_log2, group = warp >> wlog, groups = 8 >> wlog;
  const int gl = tid & ((32 << wlog) - 1), gsize = 32 << wlog;
  const int dshift = p.dim_log2 - 3;   // log2 of a row's 16-byte pieces
  const int hv0 = blockIdx.y * g.per_y, items = nruns * g.per_y;
  int turn = 0;
  for (int i = group; i < items; i += groups) {
    const int r = i / g.per_y, hv = hv0 + i - r * g.per_y;
    if (hv >= 2 * p.heads) continue;
    const Run run = runs[r];
    const int which = hv >= p.heads, h = hv - which * p.heads;
    const Place at = place_of(p, run.slot);
    const int pieces = run.n << dshift;
    const T* x;
    int64_t row_stride;
    int pos = 0;
    if (kSlots) {
      row_stride = p.x_stride[which][1];
      x = reinterpret_cast<const T*>(p.x[which]) + run.token * row_stride + h * p.x_stride[which][2];
    } else {
      const int b = (int)(run.token / d.seqlen_new), tok = (int)(run.token - (int64_t)b * d.seqlen_new);
      row_stride = p.x_stride[which][1];
      x = reinterpret_cast<const T*>(p.x[which]) + b * p.x_stride[which][0] + tok * row_stride + h * p.x_stride[which][2];
      pos = max(0, min(d.cache_seqlens[b], seq_capacity(d, b))) + tok + (d.cache_leftpad ? max(0, d.cache_leftpad[b]) : 0);
    }
    float* scale = p.scale[which] + at.page * p.s_stride[which][0] + at.block * p.s_stride[which][1] + h * p.s_stride[which][2];
    unsigned char* codes = static_cast<unsigned char*>(p.cache[which]) + at.page * p.c_stride[which][0] +
                           (int64_t)at.row * p.c_stride[which][1] + h * p.c_stride[which][2];
    const int64_t code_stride = p.c_stride[which][1];
    const bool rotate = !kSlots && which == 0 && d.rotary_cos != nullptr;
    // piece gl + k * gsize of a lane: the same column, gsize >> dshift rows on
    const int row0 = gl >> dshift, col = (gl & ((1 << dshift) - 1)) * 8, rstep = gsize >> dshift;
    const T* xl = x + row0 * row_stride + col;
    const int64_t xstep = rstep * row_stride;
    auto load = [&](int k) {
      if (rotate)
        return rotary_chunk<T, true>(xl - col + k * xstep, col, reinterpret_cast<const T*>(d.rotary_cos),
                                     reinterpret_cast<const T*>(d.rotary_sin), pos + row0 + k * rstep, d.rotary_dim, d.rotary_interleaved,
                                     d.rotary_seqlen);
      return *reinterpret_cast<const uint4*>(xl + k * xstep);
    };
    // bit patterns without their sign order magnitudes, NaN above infinity above numbers
    uint32_t most = 0u;
    auto widen = [&](const uint4& v) {
      most = __vmaxu2(__vmaxu2(most, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu)), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    };
    uint4 held[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int j = gl + k * gsize;
      held[k] = j < pieces ? load(k) : make_uint4(0u, 0u, 0u, 0u);
    }
    float old = run.kept > 0 ? *scale : 0.f;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) widen(held[k]);
    for (int k = kHeld; gl + k * gsize < pieces; ++k) widen(load(k));
    most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
    if (wlog > 0) {
      if (lane == 0) part[turn][warp] = most;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(gsize) : "memory");
      for (int k = 0; k < (1 << wlog); ++k) most = max(most, part[turn][(group << wlog) + k]);
      turn ^= 1;                       // (written again behind the next barrier but one)
    }
    const unsigned short bits = (unsigned short)most;
    float need = __fdiv_rn(Elem<T>::to_f(*reinterpret_cast<const T*>(&bits)), C::kLargest);
    if (need < 1.17549435e-38f) need = 0.f;
    if (fabsf(old) < 1.17549435e-38f) old = 0.f;          // (its reciprocal may be infinite)
    const bool raised = need > fabsf(old);
    const float now = old != old ? old : raised || need != need ? need : old;
    // A scale that is no number or infinite makes every value of the block and head one that is none: its new codes are 0, since e4m3 codes of
    // NaN would reach rows that do not see the key (0 times NaN in the products).
    const bool spoilt = !(fabsf(now) <= 3.402823466e38f);
    const float inv = now != 0.f && !spoilt ? __frcp_rn(now) : 0.f;
    if (spoilt) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) held[k] = make_uint4(0u, 0u, 0u, 0u);
    }
    unsigned char* cl = codes + row0 * code_stride + col;
    const int64_t cstep = rstep * code_stride;
    auto store = [&](int k, const uint4& v) {
      const float2 a = Elem<T>::unpack(v.x), b = Elem<T>::unpack(v.y), c = Elem<T>::unpack(v.z), e = Elem<T>::unpack(v.w);
      *reinterpret_cast<uint2*>(cl + k * cstep) = make_uint2(C::four(a.x, a.y, b.x, b.y, inv), C::four(c.x, c.y, e.x, e.y, inv));
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (gl + k * gsize < pieces) store(k, held[k]);
    for (int k = kHeld; gl + k * gsize < pieces; ++k) store(k, spoilt ? make_uint4(0u, 0u, 0u, 0u) : load(k));
    if (run.kept > 0 && raised) {
      const float m = __fmul_rn(old, inv), least = m < 0.f ? -127.f : -128.f;            // int8: -128 has no opposite
      for (int j = gl; j < run.kept << (dshift - 1); j += gsize) {
        const int row = j >> (dshift - 1), col = (j & ((1 << (dshift - 1)) - 1)) * 16;
        uint4* q = reinterpret_cast<uint4*>(codes - (int64_t)(row + 1) * code_stride + col);
        uint4 v = *q;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float f[4];
          C::floats(w[k], f);
          if (kCode == FA_CODE_INT8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = fmaxf(f[e], least);
          }
          w[k] = C::four(f[0], f[1], f[2], f[3], m);
        }
        *q = v;
      }
    }
    if (gl == 0) *scale = now;         // (every lane has read the old one: it is behind the maximum)
  }
}

// ---------------------------------------------------------------------------------------
// value checks of packed tokens: a run takes the bit of its block, and finds it taken where the call writes the block in two places
// ---------------------------------------------------------------------------------------
// words: result, CTAs that are done, then the bits; zero before the launch, or by the one CTA of a small call itself.
__global__ void __launch_bounds__(1024) append8_check_kernel(const Append8 p, uint32_t* words, int64_t bit_words, uint32_t* host) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint32_t* bits = words + kHeadWords;
  if (gridDim.x == 1) {
    for (int64_t i = threadIdx.x; i < bit_words; i += 1024) bits[i] = 0u;
    __syncthreads();
  }
  uint32_t bad = 0;
  for (int64_t t = (int64_t)blockIdx.x * 1024 + threadIdx.x; t < p.tokens; t += (int64_t)gridDim.x * 1024) {
    const int64_t s = slot_of(p, t);
    if (s < 0) {
      if (p.slots[t] >= 0) bad |= FA_SLOT_RANGE;
    } else if (!carries_on(p, t, s)) {
      const Place w = place_of(p, s);
      const int64_t block = w.page * (p.page_size / p.block) + w.block;
      const uint32_t bit = 1u << (block & 31);
      if (atomicOr(bits + (block >> 5), bit) & bit) bad |= FA_SLOT_TWICE;
    }
  }
  const uint32_t all = (__syncthreads_or(bad & FA_SLOT_RANGE) ? FA_SLOT_RANGE : 0u) | (__syncthreads_or(bad & FA_SLOT_TWICE) ? FA_SLOT_TWICE : 0u);
  if (threadIdx.x != 0) return;
  if (gridDim.x == 1) {
    words[0] = all;
    *reinterpret_cast<volatile uint32_t*>(host) = all | kCheckDone;
  } else {
    if (all) atomicOr(words, all);
    __threadfence();
    if (atomicAdd(words + 1, 1u) == gridDim.x - 1) {
      __threadfence();
      *reinterpret_cast<volatile uint32_t*>(host) = *reinterpret_cast<volatile uint32_t*>(words) | kCheckDone;
    }
  }
  __threadfence_system();
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
static AppendGeom append_geometry(const Append8& p, int device) {
  AppendGeom g;
  const int64_t ctas = 4ll * sm_count(device);
  // warps of a (run, head): as many as hold a full block
  const int longest = (int)(p.longest_run < p.block ? p.longest_run : p.block);
  const int64_t pieces = (int64_t)longest * (p.head_dim / 8);
  // 8 pieces per lane and four CTAs per SM, except where 16 let one warp hold a block (no barrier: 302 k tokens of 8 heads of 128 in blocks
  // of 32, 350 -> 338 us) or 8 warps one that is read twice otherwise (blocks of 256: 210 -> 163); else they only cost CTAs (blocks of 64:
  // 48 -> 50; of 16: 46 -> 59).
  g.held = (pieces > 256 && pieces <= 512) || pieces > 2048 ? 16 : 8;
  g.warps_log2 = 0;
  while (g.warps_log2 < 3 && pieces > (32ll * g.held << g.warps_log2)) ++g.warps_log2;
  const int groups = 8 >> g.warps_log2;
  // A CTA per block and few heads where the tokens are few (a span shorter than a block leaves CTAs without a run, which is cheap as
  // long as all run at once), all heads of a block where there are more blocks than CTAs.  2048 tokens, 8 heads of 128, blocks of 64: 30 us
  // with spans of 2 tokens and all heads, 12 now; 22 k tokens: 52, 34.
  int64_t ny = (2 * p.heads + groups - 1) / groups;
  const int64_t most = p.block > 32 ? (p.block < kSpanMost ? p.block : kSpanMost) : 32;
  g.span = 1;
  while (g.span * 2 <= most && (p.tokens + 2 * g.span - 1) / (2 * g.span) * ny >= ctas) g.span *= 2;
  const int64_t nx = (p.tokens + g.span - 1) / g.span;
  while (ny > 1 && nx * ny > 4 * ctas) ny = (ny + 1) / 2;
  g.per_y = (int)((2 * p.heads + ny - 1) / ny);
  g.grid_x = (unsigned)nx;
  g.grid_y = (unsigned)((2 * p.heads + g.per_y - 1) / g.per_y);
  return g;
}

int append8_launch(const Append8& p, const fa_decode_args* call, int dtype, int code, int device, uint32_t* host, uint32_t* dev,
                   bool check_here, cudaStream_t st) {
  const AppendGeom g = append_geometry(p, device);
  fa_decode_args d = {};
  if (call) d = *call;
  auto go = [&](auto* t, auto c, auto slots) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int kCode = decltype(c)::value;
    constexpr bool kSlots = decltype(slots)::value;
    auto kern = g.held == 8 ? cache8_append_kernel<T, kCode, kSlots, 8> : cache8_append_kernel<T, kCode, kSlots, 16>;
    cudaLaunchConfig_t lc = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    lc.gridDim = dim3(g.grid_x, g.grid_y);
    lc.blockDim = dim3(kThreads);
    lc.stream = st;
    lc.attrs = &attr;
    lc.numAttrs = kSlots && dev ? 1 : 0;
    cudaLaunchKernelEx(&lc, kern, p, d, g, host, dev, check_here);
  };
  auto by_source = [&](auto* t, auto c) {
    if (call) go(t, c, std::false_type{});
    else go(t, c, std::true_type{});
  };
  auto by_code = [&](auto* t) {
    if (code == FA_CODE_INT8) by_source(t, std::integral_constant<int, FA_CODE_INT8>{});
    else by_source(t, std::integral_constant<int, FA_CODE_E4M3>{});
  };
  if (dtype == FA_BF16) by_code(static_cast<__nv_bfloat16*>(nullptr));
  else by_code(static_cast<__half*>(nullptr));
  return check_launch("cache8_append");
}

static Append8 append_of(const fa_append8_args& a) {
  Append8 p = {};
  p.tokens = a.tokens;
  p.heads = a.heads;
  p.head_dim = a.head_dim;
  p.dim_log2 = log2_of(a.head_dim);
  p.block = a.cache.block;
  p.block_shift = log2_of(p.block);
  p.page_size = a.page_size;
  p.page_shift = log2_of(p.page_size);
  p.num_pages = a.num_pages;
  p.slots = a.slots;
  p.longest_run = a.tokens;
  p.x[0] = a.k;
  p.x[1] = a.v;
  p.cache[0] = a.k_cache;
  p.cache[1] = a.v_cache;
  p.scale[0] = a.cache.k_scale;
  p.scale[1] = a.cache.v_scale;
  for (int i = 0; i < 3; ++i) {
    p.x_stride[0][i] = i ? a.k_stride[i - 1] : 0;
    p.x_stride[1][i] = i ? a.v_stride[i - 1] : 0;
    p.c_stride[0][i] = a.kc_stride[i];
    p.c_stride[1][i] = a.vc_stride[i];
    p.s_stride[0][i] = a.cache.ks_stride[i];
    p.s_stride[1][i] = a.cache.vs_stride[i];
  }
  return p;
}

Append8 append_of(const fa_decode_args& a, const fa_cache8& c) {
  Append8 p = {};
  p.tokens = (int64_t)a.batch * a.seqlen_new;
  p.heads = a.heads_kv;
  p.head_dim = a.head_dim;
  p.dim_log2 = log2_of(a.head_dim);
  p.block = c.block;
  p.block_shift = log2_of(p.block);
  p.page_size = a.page_size;
  p.page_shift = log2_of(p.page_size);
  p.num_pages = a.num_pages;
  p.longest_run = a.seqlen_new;
  p.x[0] = a.k_new;
  p.x[1] = a.v_new;
  p.cache[0] = a.k_cache;
  p.cache[1] = a.v_cache;
  p.scale[0] = c.k_scale;
  p.scale[1] = c.v_scale;
  for (int i = 0; i < 3; ++i) {
    p.x_stride[0][i] = a.kn_stride[i];
    p.x_stride[1][i] = a.vn_stride[i];
    p.c_stride[0][i] = a.kc_stride[i];
    p.c_stride[1][i] = a.vc_stride[i];
    p.s_stride[0][i] = c.ks_stride[i];
    p.s_stride[1][i] = c.vs_stride[i];
  }
  return p;
}

constexpr int64_t kOneCta = 4096;      // tokens, and words of bits, up to which one CTA makes the checks

static int64_t bit_words(const fa_append8_args& a) { return ((int64_t)a.num_pages * (a.page_size / a.cache.block) + 31) / 32; }
size_t append8_workspace_bytes(const fa_append8_args& a) {
  if (a.tokens <= 0 || a.cache.block <= 0 || a.page_size <= 0) return 0;
  return (kHeadWords + (size_t)bit_words(a)) * sizeof(uint32_t);
}

int append8(const fa_append8_args& a, cudaStream_t st) {
  if (a.tokens == 0) return FA_OK;
  return append8_launch(append_of(a), nullptr, a.dtype, a.cache.code, a.device, nullptr, nullptr, false, st);
}

int append8_checked(const fa_append8_args& a, uint32_t* failed, cudaStream_t st) {
  *failed = 0;
  if (a.tokens == 0) return FA_OK;
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone) {
    cudaGetLastError();
    set_error("value checks cannot run while the stream is being captured; turn them off with set_validation(False)");
    return FA_ERR_LAUNCH;
  }
  const size_t need = append8_workspace_bytes(a);
  if (a.workspace == nullptr || a.workspace_bytes < need) {
    set_error("fa_append8_checked: workspace too small: need %zu bytes, got %zu", need, a.workspace_bytes);
    return FA_ERR_WORKSPACE;
  }
  uint32_t* words = static_cast<uint32_t*>(a.workspace);
  const Append8 p = append_of(a);
  uint32_t* host = nullptr;
  const int slot = take_check_word(false, a.device, &host);
  if (slot < 0) return FA_ERR_LAUNCH;
  int r = FA_OK;
  unsigned grid = 1;
  if (a.tokens > kOneCta || bit_words(a) > kOneCta) {
    const int64_t ctas = (a.tokens + 1023) / 1024, fit = 2ll * sm_count(a.device);
    grid = (unsigned)(ctas < 2 ? 2 : ctas < fit ? ctas : fit);
    const cudaError_t e = cudaMemsetAsync(words, 0, need, st);
    if (e != cudaSuccess) {
      set_error("append8: cudaMemsetAsync: %s", cudaGetErrorString(e));
      r = FA_ERR_LAUNCH;
    }
  }
  if (r == FA_OK) {
    append8_check_kernel<<<grid, 1024, 0, st>>>(p, words, bit_words(a), host);
    r = check_launch("append8_check");
  }
  const bool queued = r == FA_OK;
  if (r == FA_OK) r = append8_launch(p, nullptr, a.dtype, a.cache.code, a.device, nullptr, words, false, st);
  if (queued) {
    const int w = await_check_word(slot, failed, st);
    if (r == FA_OK) r = w;
  }
  give_check_word(slot, queued);
  return r;
}

}  // namespace fa
