// Decode over the 8-bit KV cache.  The kernel of decode.cu (units of 8 or 16 query rows of a KV head, pieces cut by length, products
// taken transposed on mma.sync, a cp.async ring per warp) on half the bytes per key; what differs is below.
//
//   Mathematics.  With codes k8, v8 and scales ks, vs of the block a key j is in:
//     t_j = scale * ks_j * (q . k8_j),   out = sum_j p_j vs_j v8_j / sum_j p_j,   p_j = 2^(t_j - M).
//   M is the running maximum of t_j + log2 |vs_j|, so that the weights p_j vs_j that go to the tensor cores as fp16 are at most about 1,
//   however much the scales of the blocks differ; the sum of the p_j is in fp32, whose range takes the offset.
//   Operands.  Codes are fp16 exactly.  bf16 queries are multiplied by the power of two that brings the largest of a unit to [2^14, 2^15);
//   elements more than 2^32 below it lose bits, nothing else does.
//   Fragments.  Both tiles are read by ldmatrix in units of two bytes.  The head dimension of q . k8 may come in any order: a lane takes
//   the 4 neighbouring codes that it is given as columns (2t, 2t+1, 2t+8, 2t+9) and the queries are arranged to match.  For V the
//   transposing form gives a lane 2 dims of 2 keys; one byte permutation sorts them by dim, and rows g and g + 8 of the product are dims
//   2g and 2g + 1.
//   int8 keys go to the tensor cores as (code + 128) * 2^-24, which is a byte permutation; what the 128 adds is the same for all keys of a row,
//   and the accumulators start from its negative.  Values go as the codes themselves, one subtraction per pair more: 128 times the weights left
//   the outputs off by 2^-21 of the largest value, however small they were (fp16, 120 k keys of equal weight: error 6.8e-4 of the outputs' rms
//   instead of 2.9e-4; 64 sequences of 1024 to 32768: 427 -> 428 us, heads of 64 291 -> 296).
//   Scales travel with their tile, by 4-byte cp.async.
//   Split: see the ranges in the kernel.
//   Bound.  HBM: one byte per code.  Measured: 64 sequences of 1024 to 32768, 32 heads over 8 of 128: 386 to 398 us (int8 and
//   e4m3), 5.2 TB/s of 6.5; heads of 64 285 us, 3.6 TB/s; whole calls over other inputs in turn 434 to 457.  What is left is the chain of a tile
//   with 12 warps per SM: 840 instructions for 32 keys (int8), issue active about half; with the loads taken out of the loop it takes 235 us, with all of them from L2 346.  A TMA
//   copy per warp and tile in place of 16 cp.async was slower (437 us; heads of 64: 425 instead of 295), so were 16 keys per warp and 16
//   warps (469), three stages and 8 warps (434).
#pragma once
#include <atomic>

#include "cache8.cuh"
#include "cache8_host.h"

namespace fa {

template <int D, int kRows> struct Decode8 {
  static constexpr int kKeys = D == 256 ? 16 : 32;     // of a warp's tile
  static constexpr int kTile8 = 4 * kKeys;
  static constexpr int P = D;                          // bytes of a staged row
  static constexpr int NS = D == 128 && kRows == 8 ? 2 : 3, QP = D + 8, OP = D + 4;
  static constexpr size_t ring = (size_t)2 * NS * kTile8 * P;
  static constexpr size_t scales = (size_t)NS * 4 * 2 * kKeys * 4;
  // Query fragments stay in registers, their rows pass through the last stage of the ring (two CTAs per SM would not fit otherwise); where
  // there are too many, they are read again for each tile.
  static constexpr bool kQueriesHeld = D * kRows < 4096;
  static constexpr size_t q_bytes = (size_t)kRows * QP * 2;
  static constexpr size_t q_at = kQueriesHeld ? ring / NS * (NS - 1) : ring + scales;
  static constexpr size_t rows_at = ring + scales + (kQueriesHeld ? 0 : q_bytes);
  static constexpr size_t smem = rows_at + 4 * kRows * 2 * 4;
  static_assert((size_t)4 * kRows * OP * 4 <= ring, "the warps' outputs, over the ring");
  static_assert(!kQueriesHeld || q_bytes <= ring / NS, "the queries, over a stage");
  static constexpr int kResident = D <= 64 || (D == 128 && kRows == 8) ? 3 : 2;   // CTAs per SM
  // 16-byte chunks of a row lie in another order, so that 8 rows of ldmatrix meet 8 bank groups: chunk c is at c ^ turn(row).
  static constexpr int kChunks = D / 16;
  static __device__ __forceinline__ int turn(int row) {
    return kChunks >= 8 ? row & 7 : kChunks == 4 ? (row >> 1) & 3 : kChunks == 2 ? (row >> 2) & 1 : 0;
  }
};
constexpr int kLongest8 = 32;          // tiles of the largest range that is still run in one wave of CTAs
constexpr int kWaves8 = 4;             // waves of CTAs beyond that
// Ranges that the `all` tiles of a unit are cut into, of U units; the host's grid is for a full cache.
__host__ __device__ __forceinline__ int ranges8(int resident, int U, int64_t all, int longest) {
  const int once = resident / U;
  if (once == 0 || all > (int64_t)kLongest8 * once) {
    const int n = kWaves8 * resident / U;
    return (int)(n < 1 ? 1 : n < all ? n : all);
  }
  const float most = ceilf(sqrtf(7.f * longest));
  const int size = (int)ceilf((float)longest / most);
  const int64_t n = (all + size - 1) / size;
  return (int)(n < once ? n : once);
}

// Sequence b after the append: keys the cache holds of it, positions of its tokens, the tiles that any query row sees.
struct Seq8 {
  int keys, len, lo, nt;
};
template <int kTile8>
__device__ __forceinline__ Seq8 seq8(const fa_decode_args& p, const ScoreCfg& cfg, int max_tiles, int b) {
  Seq8 s;
  const int cap = seq_capacity(p, b);
  s.len = max(0, min(p.cache_seqlens[b], cap)) + (p.k_new ? p.seqlen_new : 0);
  s.keys = min(s.len, cap);
  const int first = cfg.wl >= 0 ? min(max(0, s.len - p.seqlen_q - cfg.wl), s.keys) : 0;
  s.lo = first / kTile8;
  s.nt = min(max(1, (s.keys + kTile8 - 1) / kTile8 - s.lo), max_tiles);
  return s;
}

template <typename T, int kCode, int D, int kRows>
__global__ void __launch_bounds__(128, Decode8<D, kRows>::kResident)
    decode8_kernel(const fa_decode_args p, const fa_cache8 c8, const ScoreCfg cfg, const Geom8 geo,
                   const DecodeCheck chk, const bool behind) {
  using SM = Decode8<D, kRows>;
  using C = Code<kCode>;
  constexpr int P = SM::P, QP = SM::QP, NT = 128, NS = SM::NS, OP = SM::OP, NB = kRows / 8;
  constexpr int KW = SM::kKeys, KB = KW / 16, kTile8 = SM::kTile8;
  constexpr int CPR = D / 16, RPW = 32 / CPR < KW ? 32 / CPR : KW, PASSES = KW / RPW;  // a warp's loads: KW rows of CPR 16-byte chunks
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char* ring = smem_raw;                // [stage][warp][K, V][KW][P]
  float* sO = reinterpret_cast<float*>(smem_raw); // over the ring, when it is done with: 4 x kRows x OP
  float* sS = reinterpret_cast<float*>(smem_raw + SM::ring);                       // [stage][warp][K, V][KW]
  __half* sQ = reinterpret_cast<__half*>(smem_raw + SM::q_at);                     // kRows x QP
  float* sM = reinterpret_cast<float*>(smem_raw + SM::rows_at);                    // 4 x kRows
  float* sL = sM + 4 * kRows;                    // 4 x kRows
  __shared__ uint32_t sMost[4];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (chk.host) {
    const uint32_t bad = decode_checks(p, tid, NT);
    if (tid == 0 && blockIdx.x == 0) {
      *reinterpret_cast<volatile uint32_t*>(chk.host) = bad | kCheckDone;
      __threadfence_system();
    }
    if (bad) return;
  }
  const int G = p.heads_q / p.heads_kv;
  const int R = p.seqlen_q * G;                  // query rows of a kv head: r = sq * G + gi
  const int U = p.heads_kv * geo.row_groups;     // units of a sequence
  const int u = blockIdx.x % U, share = blockIdx.x / U;
  const int hk = u / geo.row_groups, rg = u % geo.row_groups;

  // ---- this CTA's range of tiles -----------------------------------------------------------------
  // The tiles of the unit in all sequences, one after another, are cut into n equal ranges, however the sequences lie in them: one wave of
  // CTAs while that needs no more than kLongest8 tiles each (but no sequence is cut into more than sqrt(7 nt) pieces), else kWaves8
  // full waves.  (Pieces of equal size within each sequence, as decode.cu has them, leave the last wave partly empty: 1 x 1900 tokens,
  // 32 heads over 8 of 128, calls with an append behind an L2 that was written over: 30 us, 26 in ranges; batches that fill the GPU several times take as long either way.)  Every warp works its range out; lane i sums
  // the sequences [i per, (i + 1) per).
  auto tiles = [&](int i) { return seq8<kTile8>(p, cfg, geo.max_tiles, i).nt; };
  int b = 0, n = 1;                              // sequence; ranges
  int64_t all = 0, off = 0, pos = 0, end = 0;    // tiles in all; before sequence b; the range that is left
  if (geo.splits == 0) {
    const int per = (p.batch + 31) / 32, b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
    int sum = 0, longest = 0;
    for (int i = b0; i < b1; ++i) {
      const int nt = tiles(i);
      sum += nt;
      longest = max(longest, nt);
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    all = __shfl_sync(0xffffffffu, inc, 31);
    longest = __reduce_max_sync(0xffffffffu, longest);
    n = ranges8(geo.resident, U, all, longest);
    if (share < n) {
      pos = share * all / n;
      end = (share + 1) * all / n;
      const int src = __ffs(__ballot_sync(0xffffffffu, pos >= inc - sum && pos < inc)) - 1;
      b = __shfl_sync(0xffffffffu, b0, src);
      off = __shfl_sync(0xffffffffu, inc - sum, src);
      for (;; ++b) {
        const int nt = tiles(b);
        if (pos < off + nt) break;
        off += nt;
      }
    }
  } else {
    // pieces of equal size of sequence b; a range is one of them
    b = share / geo.splits;
    const int nt = tiles(b), part = share - b * geo.splits;
    n = min(geo.splits, nt);
    all = nt;
    if (part < n) {
      pos = (int64_t)part * nt / n;
      end = (int64_t)(part + 1) * nt / n;
    }
  }
  // Behind the append or the checks (a programmatic launch): what the caller brought may be read before they are done, the cache and
  // their result may not.
  if (behind) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (chk.dev && *chk.dev) return;

  for (; pos < end; __syncthreads()) {
  const Seq8 w = seq8<kTile8>(p, cfg, geo.max_tiles, b);
  const int len = w.len, keys = w.keys, tile0 = w.lo + (int)(pos - off), count = (int)(min(end, off + w.nt) - pos);
  // pieces of the sequence: the ranges that it lies in; they have rows first, first + 1, ... of the workspace
  const int64_t in0 = geo.splits ? 0 : ((off + 1) * n + all - 1) / all - 1, in1 = geo.splits ? n - 1 : ((off + w.nt) * n + all - 1) / all - 1;
  const int parts = (int)(in1 - in0) + 1;
  const int64_t first = geo.splits ? (int64_t)b * geo.splits : in0 + b, mine = geo.splits ? share : share + b;

  // ---- loading --------------------------------------------------------------------------
  const int lc = (lane % CPR) * 16, lr = lane / CPR;        // this lane's 16-byte column and first row
  const int pad = p.cache_leftpad ? max(0, p.cache_leftpad[b]) : 0;
  const int* table = p.block_table ? p.block_table + (int64_t)b * p.block_table_stride : nullptr;
  const bool whole = table == nullptr || p.page_size % 16 == 0;       // 16 keys lie inside one page
  int page[KB], row16[KB];                                  // of each 16 keys of the next tile
  int ld = tile0;                                           // next tile to load
  auto ld_page = [&]() {                                    // read one tile ahead of its use
#pragma unroll
    for (int h = 0; h < KB; ++h) {
      const int key = ld * kTile8 + warp * KW + h * 16;
      const int pi = table ? divided(key, geo.page) : 0;
      page[h] = table == nullptr ? (p.cache_batch_idx ? p.cache_batch_idx[b] : b) : key < keys ? table[pi] : 0;
      row16[h] = table ? key - pi * p.page_size : key + pad;
    }
  };
  const unsigned char* kb = static_cast<const unsigned char*>(p.k_cache) + (int64_t)hk * p.kc_stride[2] + lc;
  const unsigned char* vb = static_cast<const unsigned char*>(p.v_cache) + (int64_t)hk * p.vc_stride[2] + lc;
  // Addresses by products of 32 bits into 64: with general strides and divisions, and a path of its own for whole tiles, a tile had a
  // seventh more instructions (64 sequences of 1024 to 32768, 32 heads over 8 of 128: 424 us, 416 now).
  auto row_of = [&](bool value, int pg, int row) {
    const uint64_t at = (uint64_t)(uint32_t)pg * (value ? geo.v_page : geo.k_page) + (uint64_t)(uint32_t)row * (value ? geo.v_row : geo.k_row);
    return (value ? vb : kb) + at * 16;
  };
  const float* ksb = c8.k_scale + (int64_t)hk * c8.ks_stride[2];
  const float* vsb = c8.v_scale + (int64_t)hk * c8.vs_stride[2];
  if (whole) ld_page();
  // Keys (with the scales of both) or values of tile `ld` to a stage; a tile is one cp.async group.  (Groups of their own for keys and values,
  // so that a stage's keys make room as soon as the scores are computed, had half as much again on its way and were 5 to 10 % slower:
  // 1 x 1900 tokens, timed as above, 26 -> 30 us, 64 of 1024 to 32768 with heads of 64 302 -> 319.)
  auto load_half = [&](int st, bool value) {
    if (ld < tile0 + count) {
      const int key00 = ld * kTile8 + warp * KW;
      // (row at + lr; at is a multiple of a power of two above lr)
      const uint32_t dst = smem_u32(ring) + (uint32_t)(((st * 4 + warp) * 2 + value) * KW + lr) * P;
      auto column = [&](int at) { return (uint32_t)(lc ^ (SM::turn(lr) << 4) ^ (SM::turn(at) << 4)); };
      const unsigned char* base = value ? vb : kb;
      float* dS = sS + (st * 4 + warp) * 2 * KW;
      if (whole) {
        if (!value && (KW == 32 || lane < KW)) {
          const int h = KB > 1 ? lane >> 4 : 0;
          const int pg = KB > 1 && h ? page[KB - 1] : page[0], row = (KB > 1 && h ? row16[KB - 1] : row16[0]) + (lane & 15);
          const int blk = divided(row, geo.block), bytes = key00 + lane < keys ? 4 : 0;
          cp_async4(smem_u32(dS + lane), bytes ? ksb + pg * c8.ks_stride[0] + blk * c8.ks_stride[1] : ksb, bytes);
          cp_async4(smem_u32(dS + KW + lane), bytes ? vsb + pg * c8.vs_stride[0] + blk * c8.vs_stride[1] : vsb, bytes);
        }
        if (RPW <= 16) {               // a pass lies inside 16 keys
#pragma unroll
          for (int h = 0; h < KB; ++h) {
            const unsigned char* src = row_of(value, page[h], row16[h] + lr);
            const uint64_t unit = value ? geo.v_row : geo.k_row;                 // (of 16 bytes, up to 2^32 - 1: products of them are wider)
#pragma unroll
            for (int i = 0; i < PASSES / KB; ++i) {
              const int at = (h * (PASSES / KB) + i) * RPW;
              const unsigned char* x = src + unit * (uint32_t)(16 * RPW * i);
              cp_async16(dst + at * P + column(at), x, key00 + at + lr < keys ? 16 : 0);     // zeros past the last key
            }
          }
        } else if (lr < KW) {          // one pass takes them all
          const bool up = KB > 1 && lr >= 16;
          const int pg = up ? page[KB - 1] : page[0], row = (up ? row16[KB - 1] : row16[0]) + (lr & 15), bytes = key00 + lr < keys ? 16 : 0;
          cp_async16(dst + column(0), bytes ? row_of(value, pg, row) : base, bytes);
        }
      } else {                         // pages of any size: every row is looked up
        auto where = [&](int key, int& pg, int& row) {
          const int pi = divided(key, geo.page);
          row = key - pi * p.page_size;
          pg = table[pi];
        };
        if (!value && (KW == 32 || lane < KW)) {
          int pg = 0, row = 0;
          const int bytes = key00 + lane < keys ? 4 : 0;
          if (bytes) where(key00 + lane, pg, row);
          const int blk = divided(row, geo.block);
          cp_async4(smem_u32(dS + lane), ksb + pg * c8.ks_stride[0] + blk * c8.ks_stride[1], bytes);
          cp_async4(smem_u32(dS + KW + lane), vsb + pg * c8.vs_stride[0] + blk * c8.vs_stride[1], bytes);
        }
        if (lr < KW) {
#pragma unroll 1
          for (int i = 0; i < PASSES; ++i) {
            const int key = key00 + i * RPW + lr, bytes = key < keys ? 16 : 0;
            int pg = 0, row = 0;
            if (bytes) where(key, pg, row);
            cp_async16(dst + i * RPW * P + column(i * RPW), row_of(value, pg, row), bytes);
          }
        }
      }
      if (value) {
        ++ld;
        if (whole) ld_page();
      }
    }
  };
  auto load_tile = [&](int st) {
    load_half(st, false);
    load_half(st, true);
    cp_async_commit();
  };

#pragma unroll
  for (int i = 0; i < NS - 1; ++i) load_tile(i);

  float* ws_o = reinterpret_cast<float*>(p.workspace);
  float* ws_l = ws_o + (int64_t)geo.rows * p.heads_kv * R * D;
  int stage = 0;

  // ---- Q rows (rotary fused) -> shared memory as fp16 -> B fragments held in registers ------------
  constexpr int QC = D / 8, NQ = (kRows * QC + NT - 1) / NT;
  float qinv = 1.f;                              // what the scores are multiplied by in turn
  {
    const T* cos = reinterpret_cast<const T*>(p.rotary_cos);
    const T* sin = reinterpret_cast<const T*>(p.rotary_sin);
    uint4 val[NQ];
    uint32_t most = 0u;
#pragma unroll
    for (int k = 0; k < NQ; ++k) {
      const int i = k * NT + tid, r = i / QC, d = i % QC * 8, gr = rg * kRows + r;
      val[k] = make_uint4(0u, 0u, 0u, 0u);
      if (r < kRows && gr < R) {
        const int sq = gr / G, gi = gr % G;
        const T* qrow = reinterpret_cast<const T*>(p.q) + b * p.q_stride[0] + sq * p.q_stride[1] + (int64_t)(hk * G + gi) * p.q_stride[2];
        val[k] = rotary_chunk<T, true>(qrow, d, cos, sin, len - p.seqlen_q + sq + pad, p.rotary_dim, p.rotary_interleaved, p.rotary_seqlen);
      }
      if (std::is_same<T, __nv_bfloat16>::value) {
        const uint32_t* x = reinterpret_cast<const uint32_t*>(&val[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t m = (x[e >> 1] >> (16 * (e & 1))) & 0x7fffu;
          most = max(most, m < 0x7f80u ? m : 0u);     // the largest number
        }
      }
    }
    float qmul = 1.f;
    if (std::is_same<T, __nv_bfloat16>::value) {
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) sMost[warp] = most;
      __syncthreads();
      most = max(max(sMost[0], sMost[1]), max(sMost[2], sMost[3]));
      const int e = 14 - ((int)(most >> 7) - 127);    // exponent of the factor
      if (most != 0u) {
        qmul = __int_as_float((min(e, 126) + 127) << 23);
        qinv = __int_as_float((127 - min(e, 126)) << 23);
      }
    }
#pragma unroll
    for (int k = 0; k < NQ; ++k) {
      const int i = k * NT + tid, r = i / QC, d = i % QC * 8;
      if (r >= kRows) break;
      if (std::is_same<T, __nv_bfloat16>::value) {
        uint32_t* x = reinterpret_cast<uint32_t*>(&val[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Elem<T>::unpack(x[e]);
          x[e] = Elem<__half>::pack(f.x * qmul, f.y * qmul);
        }
      }
      *reinterpret_cast<uint4*>(sQ + r * QP + d) = val[k];
    }
  }
  __syncthreads();
  auto query = [&](int n, int kk) { return *reinterpret_cast<const uint2*>(sQ + (n * 8 + g) * QP + kk * 16 + 4 * t); };
  uint2 bq[NB][SM::kQueriesHeld ? D / 16 : 1];
  if (SM::kQueriesHeld) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) bq[n][SM::kQueriesHeld ? kk : 0] = query(n, kk);
    }
    __syncthreads();                             // the stage is free
  }
  // the scores of a tile start from what the bias of its codes adds to them
  float s0[NB][2];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    if (C::kBias) {
      const uint32_t less = C::kBias | 0x80008000u, a[4] = {less, less, less, less};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint2 x = SM::kQueriesHeld ? bq[n][SM::kQueriesHeld ? kk : 0] : query(n, kk);
        mma16816<__half>(c, a, x.x, x.y);
      }
    }
    s0[n][0] = c[0];
    s0[n][1] = c[1];
  }
  // this thread's score columns: query rows 8 n + 2 t and 8 n + 2 t + 1
  int qpos[NB][2];
  float slope[NB][2];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int gr = min(rg * kRows + n * 8 + 2 * t + i, R - 1);
      const int sq = gr / G, gi = gr % G;
      qpos[n][i] = len - p.seqlen_q + sq;
      slope[n][i] = cfg.has_alibi ? p.alibi_slopes[b * p.heads_q + hk * G + gi] : 0.f;
    }
  }
  const int qmin = len - p.seqlen_q + rg * kRows / G, qmax = len - p.seqlen_q + min(rg * kRows + kRows - 1, R - 1) / G;
  float o[NB][D / 16][4];
  float mrow[NB][2], lrow[NB][2];                // M; sums of this lane's keys
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    mrow[n][0] = mrow[n][1] = -INFINITY;
    lrow[n][0] = lrow[n][1] = 0.f;
  }
  const float kmul = qinv * (1.f / C::kUnit);

  for (int ti = 0; ti < count; ++ti) {
    const int keyw = (tile0 + ti) * kTile8 + warp * KW;  // this warp's first key
    cp_async_wait<NS - 2>();
    __syncwarp();
    load_tile(stage == 0 ? NS - 1 : stage - 1);
    // this lane's row and chunk of both tiles for ldmatrix
    const uint32_t tK = smem_u32(ring) + (uint32_t)(stage * 4 + warp) * 2 * KW * P + (lane & 15) * P, tV = tK + KW * P;
    const uint32_t turned = (uint32_t)((D > 16 ? lane >> 4 : 0) ^ SM::turn(lane & 15)) << 4;
    const float* tS = sS + (stage * 4 + warp) * 2 * KW;
    if (++stage == NS) stage = 0;
    if (keyw >= keys) continue;
    // scales of this lane's keys keyw + 16 h + g and + 8; log2 of those of V: a block of zeros has a small one
    float ks[KB][2], vs[KB][2], lv[KB][2];
#pragma unroll
    for (int h = 0; h < KB; ++h) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ks[h][j] = tS[h * 16 + j * 8 + g] * kmul;
        vs[h][j] = tS[KW + h * 16 + j * 8 + g];
        lv[h][j] = __log2f(fmaxf(fabsf(vs[h][j]), 0x1p-60f));
      }
    }

    // ---- S^T = K Q^T ----------------------------------------------------------------------
    float s[KB][NB][4];
#pragma unroll
    for (int h = 0; h < KB; ++h) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        s[h][n][0] = s[h][n][2] = s0[n][0];
        s[h][n][1] = s[h][n][3] = s0[n][1];
      }
    }
#pragma unroll
    for (int kk = 0; kk < (D + 31) / 32; ++kk) {
#pragma unroll
      for (int h = 0; h < KB; ++h) {
        uint32_t r[4];
        ldsm_x4(tK + h * 16 * P + (turned ^ (kk * 32)), r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int half = 0; half < (D > 16 ? 2 : 1); ++half) {
          uint32_t a[4];
          C::neighbours(r[2 * half], a[0], a[2]);
          C::neighbours(r[2 * half + 1], a[1], a[3]);
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const uint2 x = SM::kQueriesHeld ? bq[n][SM::kQueriesHeld ? 2 * kk + half : 0] : query(n, 2 * kk + half);
            mma16816<__half>(s[h][n], a, x.x, x.y);
          }
        }
      }
    }
    // ---- softmax --------------------------------------------------------------------------
    const bool full = !cfg.has_alibi && keyw + KW <= keys && (!cfg.causal || keyw + KW - 1 <= qmin) &&
                      (cfg.wl < 0 || keyw >= qmax - cfg.wl) && (cfg.wr < 0 || keyw + KW - 1 <= qmin + cfg.wr);
    if (full) {
#pragma unroll
      for (int h = 0; h < KB; ++h) {
        const float mul[2] = {ks[h][0] * cfg.scale_log2, ks[h][1] * cfg.scale_log2};
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][n][e] *= mul[e >> 1];
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < KB; ++h) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = e & 1, j = e >> 1, key = keyw + h * 16 + j * 8 + g;
            float th;
            const float v = score_log2(cfg, slope[n][i], s[h][n][e] * ks[h][j], qpos[n][i], key, th);
            const bool seen = visible(cfg, qpos[n][i], key, keys);
            s[h][n][e] = seen ? v : -INFINITY;
          }
        }
      }
    }
    // (Raised whenever it grows.  Only past 2^8 there were 1 % fewer instructions and no time, but errors against float64 of 2.6e-4 instead of
    // 2.1e-4 in fp16: the largest weights are then rounded like the others.)
    bool grow = false;
#pragma unroll
    for (int h = 0; h < KB; ++h) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) grow |= s[h][n][e] + lv[h][e >> 1] > mrow[n][e & 1];
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float m = -INFINITY;
#pragma unroll
          for (int h = 0; h < KB; ++h) m = fmax3(m, s[h][n][i] + lv[h][0], s[h][n][2 + i] + lv[h][1]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          const bool up = m > mrow[n][i];
          alpha[i] = up ? exp2f(mrow[n][i] - m) : 1.f;           // from -inf: 0
          if (up) mrow[n][i] = m;
          lrow[n][i] *= alpha[i];
        }
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
          o[n][db][0] *= alpha[0]; o[n][db][1] *= alpha[1];
          o[n][db][2] *= alpha[0]; o[n][db][3] *= alpha[1];
        }
      }
    }
    uint32_t pb[KB][NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      // no finite score yet: exponents relative to 0, so that -inf gives 0 and NaN stays NaN
      const float m[2] = {mrow[n][0] == -INFINITY ? 0.f : mrow[n][0], mrow[n][1] == -INFINITY ? 0.f : mrow[n][1]};
#pragma unroll
      for (int h = 0; h < KB; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pe = ex2(s[h][n][e] - m[e & 1]);
          lrow[n][e & 1] += pe;
          s[h][n][e] = !full && pe == 0.f ? 0.f : pe * vs[h][e >> 1];      // a hidden key weighs 0 whatever its scale is
        }
        // P^T[key][row] as the accumulator holds it -> B fragment [keys] x [rows]
        pb[h][n][0] = transpose_8x8(Elem<__half>::pack(s[h][n][0], s[h][n][1]));
        pb[h][n][1] = transpose_8x8(Elem<__half>::pack(s[h][n][2], s[h][n][3]));
      }
    }
    // ---- O^T += V^T P^T -----------------------------------------------------------------
#pragma unroll
    for (int d2 = 0; d2 < (D + 31) / 32; ++d2) {
#pragma unroll
      for (int h = 0; h < KB; ++h) {
        uint32_t r[4];
        ldsm_x4_t(tV + h * 16 * P + (turned ^ (d2 * 32)), r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int half = 0; half < (D > 16 ? 2 : 1); ++half) {
          uint32_t a[4];
          C::alternate(r[2 * half], a[0], a[1]);
          C::alternate(r[2 * half + 1], a[2], a[3]);
#pragma unroll
          for (int n = 0; n < NB; ++n) mma16816<__half>(o[n][2 * d2 + half], a, pb[h][n][0], pb[h][n][1]);
        }
      }
    }
  }

  // ---- merge the 4 warps (each saw a quarter of every tile) -----------------------------------
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float l = lrow[n][i];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      if (g == 0) {
        sM[warp * kRows + n * 8 + 2 * t + i] = mrow[n][i];
        sL[warp * kRows + n * 8 + 2 * t + i] = l;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = n * 8 + 2 * t + i;
      const float mstar = fmaxf(fmaxf(sM[r], sM[kRows + r]), fmaxf(sM[2 * kRows + r], sM[3 * kRows + r]));
      const float wgt = mstar == -INFINITY ? 0.f : exp2f(mrow[n][i] - mstar);
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        *reinterpret_cast<float2*>(sO + (warp * kRows + r) * OP + db * 16 + 2 * g) = make_float2(wgt * o[n][db][i], wgt * o[n][db][2 + i]);
    }
  }
  __syncthreads();

  // ---- output, or a piece of it -----------------------------------------------------------
  // workspace: the R query rows of every (piece, kv head), not padded to units
  const int64_t ws_row = (mine * p.heads_kv + hk) * R + rg * kRows;
  for (int i = tid; i < kRows * (D / 4); i += NT) {
    const int r = i / (D / 4), c4 = (i % (D / 4)) * 4;
    const int gr = rg * kRows + r;
    if (gr >= R) continue;
    const float mstar = fmaxf(fmaxf(sM[r], sM[kRows + r]), fmaxf(sM[2 * kRows + r], sM[3 * kRows + r]));
    float lsum = 0.f;
    if (mstar != -INFINITY) {
#pragma unroll
      for (int wv = 0; wv < 4; ++wv) lsum += exp2f(sM[wv * kRows + r] - mstar) * sL[wv * kRows + r];
    }
    float4 acc = *reinterpret_cast<const float4*>(sO + r * OP + c4);
#pragma unroll
    for (int wv = 1; wv < 4; ++wv) {
      const float4 x = *reinterpret_cast<const float4*>(sO + (wv * kRows + r) * OP + c4);
      acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    }
    const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
    acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    const int sq = gr / G, h = hk * G + gr % G;
    if (parts == 1) {
      T* og = reinterpret_cast<T*>(p.o) + b * p.o_stride[0] + sq * p.o_stride[1] + (int64_t)h * p.o_stride[2] + c4;
      uint2 pk;
      pk.x = Elem<T>::pack(acc.x, acc.y);
      pk.y = Elem<T>::pack(acc.z, acc.w);
      *reinterpret_cast<uint2*>(og) = pk;
    } else {
      *reinterpret_cast<float4*>(ws_o + (ws_row + r) * D + c4) = acc;
      if (c4 == 0) ws_l[ws_row + r] = lsum == 0.f ? -INFINITY : mstar + log2f(lsum);
    }
  }
  if (parts > 1) {
    // the CTA that comes last merges; the pieces are ordered before the count by each writer's fence
    __shared__ int last;
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      uint32_t* ctr = p.counters + ((int64_t)b * U + u);
      last = atomicAdd(ctr, 1u) == (uint32_t)(parts - 1);
      if (last) *ctr = 0u;
    }
    __syncthreads();
    if (last) {
      __threadfence();
      const int rows = min(kRows, R - rg * kRows);
      for (int i = tid; i < rows * (D / 4); i += NT) {
        const int r = i / (D / 4), gr = rg * kRows + r;
        const int sq = gr / G, h = hk * G + gr % G;
        merge_pieces<T, D>(ws_o, ws_l, (first * p.heads_kv + hk) * R + gr, (int64_t)p.heads_kv * R, parts, (i % (D / 4)) * 4,
                           reinterpret_cast<T*>(p.o) + b * p.o_stride[0] + sq * p.o_stride[1] + (int64_t)h * p.o_stride[2]);
      }
    }
  }
  // the next sequence of the range
  cp_async_wait<0>();
  pos += count;
  off += w.nt;
  ++b;
  }
}

template <typename T, int kCode, int D, int kRows>
static int launch_decode8_rows(const fa_decode_args& a, const fa_cache8& c, const ScoreCfg& cfg, const Geom8& g, const DecodeCheck& chk,
                               bool behind, cudaStream_t st) {
  auto kern = decode8_kernel<T, kCode, D, kRows>;
  const size_t smem = Decode8<D, kRows>::smem;
  static std::atomic<uint64_t> prepared{0};      // once per kernel and device
  const uint64_t bit = a.device < 64 ? 1ull << a.device : 0;
  if ((prepared.load(std::memory_order_relaxed) & bit) == 0) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) {
      set_error("decode8: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
      return FA_ERR_LAUNCH;
    }
    prepared.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr;
  lc.gridDim = dim3((unsigned)g.ranges * a.heads_kv * g.row_groups);
  lc.blockDim = dim3(128);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  if (behind) {
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = &attr;
    lc.numAttrs = 1;
  }
  cudaLaunchKernelEx(&lc, kern, a, c, cfg, g, chk, behind);
  return check_launch("decode8");
}

template <typename T, int kCode, int D>
static int launch_decode8_dim(const fa_decode_args& a, const fa_cache8& c, const ScoreCfg& cfg, int unit_rows, const Geom8& g,
                              const DecodeCheck& chk, bool behind, cudaStream_t st) {
  return unit_rows == 8 ? launch_decode8_rows<T, kCode, D, 8>(a, c, cfg, g, chk, behind, st)
                        : launch_decode8_rows<T, kCode, D, 16>(a, c, cfg, g, chk, behind, st);
}

template <typename T, int kCode>
static int launch_decode8(const fa_decode_args& a, const fa_cache8& c, const ScoreCfg& cfg, int unit_rows, const Geom8& g,
                          const DecodeCheck& chk, bool behind, cudaStream_t st) {
  switch (a.head_dim) {
    case 16: return launch_decode8_dim<T, kCode, 16>(a, c, cfg, unit_rows, g, chk, behind, st);
    case 32: return launch_decode8_dim<T, kCode, 32>(a, c, cfg, unit_rows, g, chk, behind, st);
    case 64: return launch_decode8_dim<T, kCode, 64>(a, c, cfg, unit_rows, g, chk, behind, st);
    case 128: return launch_decode8_dim<T, kCode, 128>(a, c, cfg, unit_rows, g, chk, behind, st);
    case 256: return launch_decode8_dim<T, kCode, 256>(a, c, cfg, unit_rows, g, chk, behind, st);
  }
  set_error("head_dim %d not in {16,32,64,128,256}", a.head_dim);
  return FA_ERR_UNSUPPORTED;
}

}  // namespace fa
