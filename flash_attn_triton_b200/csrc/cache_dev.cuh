// What the kernels over a KV cache share: value checks, rotary embedding of a row, where a row of the cache lies, the tiles of a
// sequence, the merge of its pieces.
#pragma once
#include "common.cuh"

namespace fa {

constexpr int kTile = 64;             // keys per work tile
constexpr int kMaxBalanced = 512;     // sequences up to which every warp sums the lengths itself
constexpr int kOneWave = 64;          // largest piece, in tiles, that is still run in one wave of CTAs
constexpr int kWaves = 4;             // waves of CTAs beyond that

struct DecodeGeom {
  int shares;      // pieces the grid has room for
  int splits;      // 0: pieces sized on the device; else that many pieces of every sequence
  int resident;    // CTAs the GPU runs at a time
  int max_tiles;   // tiles of a full cache
  int row_groups;  // ceil(seqlen_q * group / rows of a unit)
  int page_shift;  // log2(page_size) or -1
};

// The value checks of one call: their result goes to a word in mapped host memory (bit 31 = done, low
// bits = fa_decode_check of the checks that failed), and to a word of the call's own workspace for the kernels
// behind them.  The host word is handed to the next call once the host has read it; the kernels read theirs until the
// last CTA has started, long after the call has returned, so no other call may write to it.
constexpr uint32_t kCheckDone = 0x80000000u;
constexpr int kInlineCheck = 1024;   // table entries up to which every attention CTA makes the checks itself
struct DecodeCheck {
  uint32_t* host;       // null = no checks in this kernel
  const uint32_t* dev;  // null, or the result of decode_check_kernel
};

// All checks, by the threads of one CTA; every thread gets the mask of those that failed.
__device__ __forceinline__ uint32_t decode_checks(const fa_decode_args& p, int tid, int nt) {
  uint32_t bad = 0;
  if (p.block_table) {
    const int n = p.batch * p.block_table_stride;
    for (int i = tid; i < n; i += nt)
      if ((unsigned)p.block_table[i] >= (unsigned)p.num_pages) bad |= FA_CHECK_PAGES;
  }
  const long long cap = p.block_table ? (long long)p.block_table_stride * p.page_size : p.page_size;
  for (int b = tid; b < p.batch; b += nt) {
    if (p.cache_batch_idx && (unsigned)p.cache_batch_idx[b] >= (unsigned)p.num_pages) bad |= FA_CHECK_ROWS;
    const int pad = p.cache_leftpad ? p.cache_leftpad[b] : 0;
    if (pad < 0) bad |= FA_CHECK_LEFTPAD;
    const int old = p.cache_seqlens[b];
    const long long last = (long long)old + (p.k_new ? p.seqlen_new : 0) + pad;
    if (old < 0 || last > cap) bad |= FA_CHECK_LENGTHS;
    if (p.rotary_cos && last > p.rotary_seqlen) bad |= FA_CHECK_ROTARY;
  }
  if (!__syncthreads_or(bad)) return 0u;
  return (__syncthreads_or(bad & FA_CHECK_PAGES) ? FA_CHECK_PAGES : 0u) |
         (__syncthreads_or(bad & FA_CHECK_ROWS) ? FA_CHECK_ROWS : 0u) |
         (__syncthreads_or(bad & FA_CHECK_LEFTPAD) ? FA_CHECK_LEFTPAD : 0u) |
         (__syncthreads_or(bad & FA_CHECK_LENGTHS) ? FA_CHECK_LENGTHS : 0u) |
         (__syncthreads_or(bad & FA_CHECK_ROTARY) ? FA_CHECK_ROTARY : 0u);
}

template <typename T> __device__ __forceinline__ T hmul_rn(T a, T b);
template <> __device__ __forceinline__ __half hmul_rn(__half a, __half b) { return __hmul_rn(a, b); }
template <> __device__ __forceinline__ __nv_bfloat16 hmul_rn(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmul_rn(a, b); }
template <typename T> __device__ __forceinline__ T hadd_rn(T a, T b);
template <> __device__ __forceinline__ __half hadd_rn(__half a, __half b) { return __hadd_rn(a, b); }
template <> __device__ __forceinline__ __nv_bfloat16 hadd_rn(__nv_bfloat16 a, __nv_bfloat16 b) { return __hadd_rn(a, b); }
template <typename T> __device__ __forceinline__ T hsub_rn(T a, T b);
template <> __device__ __forceinline__ __half hsub_rn(__half a, __half b) { return __hsub_rn(a, b); }
template <> __device__ __forceinline__ __nv_bfloat16 hsub_rn(__nv_bfloat16 a, __nv_bfloat16 b) { return __hsub_rn(a, b); }

// Rotary on element d of a head vector x (read through `get`), every product and sum
// rounded to T like the reference's eager arithmetic (flash_attn_interface.py:57-66).
// A position outside the table [0, rotary_seqlen) leaves the element unrotated (the host checks
// the lengths when validation is on; this keeps the read in bounds when it is off).
template <typename T, typename F>
__device__ __forceinline__ T rotary_elem(F get, int d, const T* cos, const T* sin, int pos,
                                         int rotary_dim, int interleaved, int rotary_seqlen) {
  if (d >= rotary_dim || pos < 0 || pos >= rotary_seqlen) return get(d);
  const int half = rotary_dim >> 1;
  int i, partner;
  bool first;
  if (interleaved) {
    i = d >> 1;
    first = (d & 1) == 0;
    partner = d ^ 1;
  } else {
    first = d < half;
    i = first ? d : d - half;
    partner = first ? d + half : d - half;
  }
  const T c = cos[(int64_t)pos * half + i], s = sin[(int64_t)pos * half + i];
  const T x = get(d), y = get(partner);
  // first: x*c - y*s ; second: y*s + x*c  (y = first element of the pair)
  return first ? hsub_rn(hmul_rn(x, c), hmul_rn(y, s)) : hadd_rn(hmul_rn(y, s), hmul_rn(x, c));
}

// Whether rotary_chunk() can read 16 (pairs side by side: 8) bytes of the tables at a time.
template <typename T>
__device__ __forceinline__ bool rotary_in_chunks(const T* cos, const T* sin, int rotary_dim, int interleaved) {
  return (rotary_dim & (interleaved ? 7 : 15)) == 0 &&
         ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & (interleaved ? 7 : 15)) == 0;
}

// The others: halves that are multiples of 4 by 8 bytes, the rest element by element.
template <typename T>
__device__ __forceinline__ uint4 rotary_chunk_any(const T* x, int d, const T* cos, const T* sin, int pos, int rotary_dim,
                                                  int interleaved, int rotary_seqlen) {
  union { uint4 v; uint2 h[2]; T e[8]; } out;
  const int half = rotary_dim >> 1;
  if (!interleaved && half % 4 == 0 && ((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 7) == 0) {
    union Four { uint2 v; T e[4]; };
    out.v = *reinterpret_cast<const uint4*>(x + d);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = d + 4 * h;
      if (at >= rotary_dim) break;
      const bool first = at < half;
      const int64_t i = (int64_t)pos * half + (first ? at : at - half);
      Four self, other, c, s;
      self.v = out.h[h];
      other.v = *reinterpret_cast<const uint2*>(x + (first ? at + half : at - half));
      c.v = *reinterpret_cast<const uint2*>(cos + i);
      s.v = *reinterpret_cast<const uint2*>(sin + i);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        self.e[k] = first ? hsub_rn(hmul_rn(self.e[k], c.e[k]), hmul_rn(other.e[k], s.e[k]))
                          : hadd_rn(hmul_rn(other.e[k], s.e[k]), hmul_rn(self.e[k], c.e[k]));
      out.h[h] = self.v;
    }
    return out.v;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    out.e[k] = rotary_elem<T>([&](int j) { return x[j]; }, d + k, cos, sin, pos, rotary_dim, interleaved, rotary_seqlen);
  return out.v;
}
template <typename T>
__device__ __noinline__ uint4 rotary_chunk_call(const T* x, int d, const T* cos, const T* sin, int pos, int rotary_dim,
                                                int interleaved, int rotary_seqlen) {
  return rotary_chunk_any(x, d, cos, sin, pos, rotary_dim, interleaved, rotary_seqlen);
}

// 8 elements of a head row, rotated like rotary_elem.  kCall: the general case out of line.  In the main loop of decode_kernel
// it cost registers and the order of the loads (head_dim 256, 32 x 8000 tokens, 16 heads over 4: 268 us, 233 as a call); a
// kernel that only rotates and copies is better off without the call (4 x 256 tokens behind 300, 32 heads over 8 of 128, with
// their attention: 42 us, 46).  Pairs side by side need no row beside the one at hand and half as much of the tables: 8 x 900
// tokens, 4 new, 16 heads over 4 of 128: a thread per element 30.4 us, eight elements of a thread one by one 20.6, now 16.6.
template <typename T, bool kCall>
__device__ __forceinline__ uint4 rotary_chunk(const T* x, int d, const T* cos, const T* sin, int pos, int rotary_dim,
                                              int interleaved, int rotary_seqlen) {
  union { uint4 v; T e[8]; } out, self, other, c, s;
  self.v = *reinterpret_cast<const uint4*>(x + d);
  if (cos == nullptr || d >= rotary_dim || pos < 0 || pos >= rotary_seqlen) return self.v;
  if (!rotary_in_chunks(cos, sin, rotary_dim, interleaved)) {
    if (kCall) return rotary_chunk_call(x, d, cos, sin, pos, rotary_dim, interleaved, rotary_seqlen);
    return rotary_chunk_any(x, d, cos, sin, pos, rotary_dim, interleaved, rotary_seqlen);
  }
  const int half = rotary_dim >> 1;
  if (interleaved) {
    *reinterpret_cast<uint2*>(c.e) = *reinterpret_cast<const uint2*>(cos + (int64_t)pos * half + (d >> 1));
    *reinterpret_cast<uint2*>(s.e) = *reinterpret_cast<const uint2*>(sin + (int64_t)pos * half + (d >> 1));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const T x0 = self.e[2 * k], x1 = self.e[2 * k + 1];
      out.e[2 * k] = hsub_rn(hmul_rn(x0, c.e[k]), hmul_rn(x1, s.e[k]));
      out.e[2 * k + 1] = hadd_rn(hmul_rn(x0, s.e[k]), hmul_rn(x1, c.e[k]));
    }
    return out.v;
  }
  const bool first = d < half;
  const int i = first ? d : d - half;
  other.v = *reinterpret_cast<const uint4*>(x + (first ? d + half : d - half));
  c.v = *reinterpret_cast<const uint4*>(cos + (int64_t)pos * half + i);
  s.v = *reinterpret_cast<const uint4*>(sin + (int64_t)pos * half + i);
#pragma unroll
  for (int k = 0; k < 8; ++k)
    out.e[k] = first ? hsub_rn(hmul_rn(self.e[k], c.e[k]), hmul_rn(other.e[k], s.e[k]))
                     : hadd_rn(hmul_rn(other.e[k], s.e[k]), hmul_rn(self.e[k], c.e[k]));
  return out.v;
}

__device__ __forceinline__ int64_t cache_row_offset(const fa_decode_args& p, int b, int pos,
                                                    int page_shift, const int64_t* stride) {
  int page, row;
  if (p.block_table) {
    int pi;
    if (page_shift >= 0) {
      pi = pos >> page_shift;
      row = pos & (p.page_size - 1);
    } else {
      pi = pos / p.page_size;
      row = pos - pi * p.page_size;
    }
    page = p.block_table[(int64_t)b * p.block_table_stride + pi];
  } else {
    page = p.cache_batch_idx ? p.cache_batch_idx[b] : b;
    row = pos;
  }
  return (int64_t)page * stride[0] + (int64_t)row * stride[1];
}

// Tiles of a sequence: nt work tiles from tile lo on.  Keys that no query row sees (left of the window)
// are skipped, new tokens never are: somebody has to append them.  An empty sequence has one
// (empty) tile, which writes its zeros.
struct SeqTiles {
  int len_old, len, lo, nt;
};
// Rows a sequence can hold behind its left padding: lengths are taken up to here and new tokens stored up to here, so
// that a call whose values are not checked stays inside its rows of the cache and of the table.
__host__ __device__ __forceinline__ int cache_capacity(const fa_decode_args& p) {
  const int64_t cap = p.block_table ? (int64_t)p.block_table_stride * p.page_size : p.page_size;
  return (int)(cap < (1 << 30) ? cap : (1 << 30));
}
__device__ __forceinline__ int seq_capacity(const fa_decode_args& p, int b) {
  return cache_capacity(p) - (p.cache_leftpad ? max(0, p.cache_leftpad[b]) : 0);
}
__device__ __forceinline__ SeqTiles seq_tiles(const fa_decode_args& p, const ScoreCfg& cfg, int max_tiles, int b) {
  SeqTiles s;
  s.len_old = max(0, min(p.cache_seqlens[b], seq_capacity(p, b)));
  s.len = s.len_old + (p.k_new ? p.seqlen_new : 0);
  const int first = cfg.wl >= 0 ? min(max(0, s.len - p.seqlen_q - cfg.wl), s.len_old) : 0;
  s.lo = first / kTile;
  s.nt = min(max(1, (s.len + kTile - 1) / kTile - s.lo), max_tiles);
  return s;
}

// What a CTA works on: tiles [tile0, tile0 + count) of sequence b, counted from the first one that is work; base is the first of
// the `parts` pieces of the sequence.  tiles(i): work tiles of sequence i; U: units of a sequence.  False: nothing.
struct Piece {
  int b, tile0, count, parts, base;
};
template <typename Tiles>
__device__ __forceinline__ bool piece_of(const DecodeGeom& geo, int batch, int share, int U, int lane, Tiles tiles, Piece& out) {
  int b, parts, base;
  if (geo.splits == 0) {
    // Every warp does this on its own, without shared memory or barriers (which cost a small step 2 to 4
    // us); lane i looks after the sequences [i per, (i + 1) per).
    const int per = (batch + 31) / 32, b0 = min(lane * per, batch), b1 = min(b0 + per, batch);
    int sum = 0, longest = 0;
    for (int i = b0; i < b1; ++i) {
      const int nt = tiles(i);
      sum += nt;
      longest = max(longest, nt);
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    longest = __reduce_max_sync(0xffffffffu, longest);
    const int64_t work = (int64_t)sum * U;
    int size = (int)((work + geo.resident - 1) / geo.resident), mine = 0;
    auto count_pieces = [&]() {
      mine = 0;
      for (int i = b0; i < b1; ++i) mine += (tiles(i) + size - 1) / size;
    };
    if (size > kOneWave) {
      size = max(kOneWave / 2, (int)((work + kWaves * geo.resident - 1) / (kWaves * geo.resident)));
      count_pieces();
    } else {
      size = max(size, (int)ceilf((float)longest / ceilf(sqrtf(7.f * longest))));
      for (; size < longest; size += max(1, size >> 3)) {
        count_pieces();
        if (__reduce_add_sync(0xffffffffu, mine) * U <= geo.resident) break;
      }
    }
    if (size >= longest) {                       // every sequence in one piece
      if (share >= batch) return false;
      b = base = share;
      parts = 1;
    } else {
      int inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      const bool owner = share >= inc - mine && share < inc;
      const unsigned who = __ballot_sync(0xffffffffu, owner);
      if (who == 0u) return false;                       // the grid is sized for a full cache
      base = inc - mine;
      b = b0;
      parts = 0;
      if (owner) {
        for (;; ++b) {
          parts = (tiles(b) + size - 1) / size;
          if (share < base + parts) break;
          base += parts;
        }
      }
      const int src = __ffs(who) - 1;
      b = __shfl_sync(0xffffffffu, b, src);
      base = __shfl_sync(0xffffffffu, base, src);
      parts = __shfl_sync(0xffffffffu, parts, src);
    }
  } else {
    b = share / geo.splits;
    base = b * geo.splits;
    parts = min(geo.splits, tiles(b));
    if (share - base >= parts) return false;
  }
  const int nt = tiles(b);
  out.b = b;
  out.parts = parts;
  out.base = base;
  out.tile0 = (int)((int64_t)(share - base) * nt / parts);
  out.count = (int)((int64_t)(share - base + 1) * nt / parts) - out.tile0;
  return true;
}

// Elements [d, d + 4) of one output row, merged from the `parts` workspace rows r0, r0 + step, ...  Eight
// pieces are loaded at a time, their common maximum taken first.  (Sixteen: longer code in front of few rows, -1 to
// +7 % of a step's time at every head size -- 2 x 411 tokens, one head of 64: 9.7 -> 10.6 us.)
constexpr int kMergeBatch = 8;
template <typename T, int D>
__device__ __forceinline__ void merge_pieces(const float* ws_o, const float* ws_l, int64_t r0, int64_t step, int parts, int d,
                                             T* og) {
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float wsum = 0.f, m = -INFINITY;
  for (int i0 = 0; i0 < parts; i0 += kMergeBatch) {
    float l[kMergeBatch];
    float4 x[kMergeBatch];
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) {
      const int i = i0 + j;
      const int64_t r = r0 + i * step;
      l[j] = i < parts ? ws_l[r] : -INFINITY;
      x[j] = i < parts ? *reinterpret_cast<const float4*>(ws_o + r * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) mn = fmaxf(mn, l[j]);
    // pieces without a finite score weigh 0, which a NaN in them survives
    const float mf = mn == -INFINITY ? 0.f : mn;
    const float sc = exp2f(m - mf);
    acc.x *= sc; acc.y *= sc; acc.z *= sc; acc.w *= sc;
    wsum *= sc;
    m = mn;
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) {
      const float w = exp2f(l[j] - mf);
      wsum += w;
      acc.x += w * x[j].x; acc.y += w * x[j].y; acc.z += w * x[j].z; acc.w += w * x[j].w;
    }
  }
  const float inv = wsum > 0.f ? 1.f / wsum : 0.f;
  uint2 pk;
  pk.x = Elem<T>::pack(acc.x * inv, acc.y * inv);
  pk.y = Elem<T>::pack(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(og + d) = pk;
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

inline int page_shift_of(const fa_decode_args& a) {
  if (a.page_size <= 0 || (a.page_size & (a.page_size - 1)) != 0) return -1;
  int s = 0;
  while ((1 << s) < a.page_size) ++s;
  return s;
}

// Room for the pieces the kernel may make.  It picks their size so that
//   * one wave of CTAs (two per SM, one at head_dim 256) takes all of them, while that needs no more
//     than kOneWave tiles each: every CTA costs about 3.5 us beside its tiles (16 sequences of 4000 keys,
//     8 heads: one wave of 32-tile pieces 55 us, two of 16 61 us, 68 us without pieces);
//   * a sequence has no more than sqrt(7 nt) pieces of its nt tiles: a tile costs about 0.7 us and a piece
//     0.1 us in the merge (one sequence of 8000 keys, two heads: 126 pieces 20 us, 32 pieces 16.4 us);
//   * more work than that runs as kWaves waves, which the hardware balances over SMs of unequal speed
//     (64 sequences of 16000 keys: one wave of equal shares 688 us, 3.5 waves 656 us = 0.98 of the copy
//     bandwidth).
// An explicit num_splits, and batches too large to sum in every warp, cut every sequence into the
// same number of pieces.
inline DecodeGeom decode_geometry(const fa_decode_args& a, int row_groups, int ctas_per_sm) {
  DecodeGeom g;
  g.row_groups = row_groups;
  const int64_t cap = a.block_table ? (int64_t)a.block_table_stride * a.page_size : a.page_size;
  const int64_t nt = cap > 0 ? (cap + kTile - 1) / kTile : 1;
  const int64_t U = (int64_t)a.heads_kv * g.row_groups;
  g.max_tiles = (int)nt;
  g.splits = 0;
  g.resident = sm_count(a.device) * ctas_per_sm;
  if (a.num_splits > 0 || a.batch > kMaxBalanced || a.batch * nt > (1 << 30)) {
    g.splits = a.num_splits > 0 ? (int)(a.num_splits < nt ? a.num_splits : nt) : 1;
    g.shares = a.batch * g.splits;
  } else {
    const int64_t most = a.batch * nt, whole = a.batch;
    int64_t n = most * U <= (int64_t)kOneWave * g.resident ? g.resident / U : kWaves * g.resident / U + 1;
    n += whole;                                // rounding up adds less than a piece per sequence
    g.shares = (int)(n < most ? n : most);
  }
  g.page_shift = page_shift_of(a);
  return g;
}

}  // namespace fa
