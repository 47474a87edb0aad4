// Decode over the 8-bit KV cache.  The kernel of decode.cu (units of 8 or 16 query rows of a KV head, pieces cut by length, products
// taken transposed on mma.sync, a cp.async ring per warp) on half the bytes per key; what differs is below.
//
//   Mathematics.  With codes k8, v8 and scales ks, vs of the block a key j is in:
//     t_j = scale * ks_j * (q . k8_j),   out = sum_j p_j vs_j v8_j / sum_j p_j,   p_j = 2^(t_j - M).
//   M is the running maximum of t_j + log2 vs_j, so that the weights p_j vs_j that go to the tensor cores as fp16 are at most about 1,
//   however much the scales of the blocks differ; the sum of the p_j is in fp32, whose range takes the offset.
//   Operands.  Codes are fp16 exactly.  bf16 queries are multiplied by the power of two that brings the largest of a unit to [2^14, 2^15);
//   elements more than 2^32 below it lose bits, nothing else does.
//   Fragments.  Both tiles are read by ldmatrix in units of two bytes.  The head dimension of q . k8 may come in any order: a lane takes
//   the 4 neighbouring codes that it is given as columns (2t, 2t+1, 2t+8, 2t+9) and the queries are arranged to match.  For V the
//   transposing form gives a lane 2 dims of 2 keys; one byte permutation sorts them by dim, and rows g and g + 8 of the product are dims
//   2g and 2g + 1.
//   Scales travel with their tile: 32 words per warp and stage by 4-byte cp.async.
//   Bound.  HBM: one byte per code.
#pragma once
#include <atomic>

#include "cache8.cuh"
#include "cache8_host.h"

namespace fa {

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes));
}

template <int D, int kRows> struct Decode8 {
  static constexpr int P = D == 16 ? 16 : D + 16;      // bytes of a staged row: 8 rows of ldmatrix meet 8 bank groups
  static constexpr int NS = 3, QP = D + 8, OP = D + 4;
  static constexpr size_t ring = (size_t)2 * NS * kTile * P;
  static constexpr size_t scales = (size_t)NS * 4 * 32 * 4;
  static constexpr size_t q_bytes = (size_t)kRows * QP * 2;
  static constexpr size_t smem = ring + scales + q_bytes + 4 * kRows * 2 * 4;
  static_assert((size_t)4 * kRows * OP * 4 <= ring, "the warps' outputs, over the ring");
  // CTAs per SM: accumulators and query fragments are D * kRows * 3 / 64 registers
  static constexpr int kCtas = D * kRows <= 1024 ? 4 : D * kRows <= 2048 ? 3 : 2;
  static constexpr int kResident = D == 256 ? 2 : kCtas;
};

// Sequence b after the append: keys the cache holds of it, positions of its tokens, the tiles that any query row sees.
struct Seq8 {
  int keys, len, lo, nt;
};
__device__ __forceinline__ Seq8 seq8(const fa_decode_args& p, const ScoreCfg& cfg, int max_tiles, int b) {
  Seq8 s;
  const int cap = seq_capacity(p, b);
  s.len = max(0, min(p.cache_seqlens[b], cap)) + (p.k_new ? p.seqlen_new : 0);
  s.keys = min(s.len, cap);
  const int first = cfg.wl >= 0 ? min(max(0, s.len - p.seqlen_q - cfg.wl), s.keys) : 0;
  s.lo = first / kTile;
  s.nt = min(max(1, (s.keys + kTile - 1) / kTile - s.lo), max_tiles);
  return s;
}

template <typename T, int kCode, int D, int kRows>
__global__ void __launch_bounds__(128, Decode8<D, kRows>::kResident)
    decode8_kernel(const fa_decode_args p, const fa_cache8 c8, const int block_shift, const ScoreCfg cfg, const DecodeGeom geo,
                   const DecodeCheck chk, const bool behind) {
  using SM = Decode8<D, kRows>;
  using C = Code<kCode>;
  constexpr int P = SM::P, QP = SM::QP, NT = 128, NS = SM::NS, OP = SM::OP, NB = kRows / 8;
  constexpr int CPR = D / 16, RPW = 32 / CPR, PASSES = RPW >= 16 ? 1 : 16 / RPW;     // a warp's loads: 16 rows of CPR 16-byte chunks
  extern __shared__ __align__(16) unsigned char smem_raw[];
  unsigned char* ring = smem_raw;                // [stage][warp][K, V][16][P]
  float* sO = reinterpret_cast<float*>(smem_raw); // over the ring, when it is done with: 4 x kRows x OP
  float* sS = reinterpret_cast<float*>(smem_raw + SM::ring);                       // [stage][warp][K, V][16]
  __half* sQ = reinterpret_cast<__half*>(smem_raw + SM::ring + SM::scales);        // kRows x QP
  float* sM = reinterpret_cast<float*>(smem_raw + SM::ring + SM::scales + SM::q_bytes); // 4 x kRows
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

  // Behind the append or the checks (a programmatic launch): what the caller brought may be read before they are done, the cache and
  // their result may not.
  Piece piece;
  const bool work = piece_of(geo, p.batch, share, U, lane, [&](int i) { return seq8(p, cfg, geo.max_tiles, i).nt; }, piece);
  if (behind) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!work || (chk.dev && *chk.dev)) return;
  const int b = piece.b, parts = piece.parts, base = piece.base, count = piece.count;
  const Seq8 w = seq8(p, cfg, geo.max_tiles, b);
  const int len = w.len, keys = w.keys, tile0 = w.lo + piece.tile0;

  // ---- loading --------------------------------------------------------------------------
  const int lc = (lane % CPR) * 16, lr = lane / CPR;        // this lane's 16-byte column and first row
  const bool one_page = p.block_table == nullptr || geo.page_shift >= 4;   // a warp's 16 keys lie inside one page
  const int pad = p.cache_leftpad ? max(0, p.cache_leftpad[b]) : 0;
  const int* table = p.block_table ? p.block_table + (int64_t)b * p.block_table_stride : nullptr;
  int page = table ? 0 : (p.cache_batch_idx ? p.cache_batch_idx[b] : b);
  int ld = tile0;                                           // next tile to load
  auto ld_page = [&]() {                                    // read one tile ahead of its use
    if (table && one_page) {
      const int key = ld * kTile + warp * 16;
      if (key < keys) page = table[key >> geo.page_shift];
    }
  };
  // page and row of a key
  auto where = [&](int key, int& pg, int& row) {
    if (one_page) {
      pg = page;
      row = table ? key & (p.page_size - 1) : key + pad;
    } else {
      const int pi = divided(key, p.page_size, geo.page_shift);
      row = key - pi * p.page_size;
      pg = table[pi];
    }
  };
  const unsigned char* kb = static_cast<const unsigned char*>(p.k_cache) + (int64_t)hk * p.kc_stride[2] + lc;
  const unsigned char* vb = static_cast<const unsigned char*>(p.v_cache) + (int64_t)hk * p.vc_stride[2] + lc;
  // lanes 0-15: scales of K, lanes 16-31: of V
  const float* sb = (lane < 16 ? c8.k_scale + (int64_t)hk * c8.ks_stride[2] : c8.v_scale + (int64_t)hk * c8.vs_stride[2]);
  const int64_t sb_page = lane < 16 ? c8.ks_stride[0] : c8.vs_stride[0], sb_block = lane < 16 ? c8.ks_stride[1] : c8.vs_stride[1];
  ld_page();
  auto load_tile = [&](int st) {
    if (ld == tile0 + count) return;
    const int key00 = ld * kTile + warp * 16;
    {
      const int key = key00 + (lane & 15);
      const bool in = key < keys;
      int pg = 0, row = 0;
      if (in) where(key, pg, row);
      cp_async4(smem_u32(sS + (st * 4 + warp) * 32 + lane), sb + pg * sb_page + divided(row, c8.block, block_shift) * sb_block, in ? 4 : 0);
    }
    if (RPW <= 16 || lr < 16) {
      unsigned char* dK = ring + (size_t)((st * 4 + warp) * 2 * 16 + lr) * P + lc;
      unsigned char* dV = dK + 16 * P;
      const int key0 = key00 + lr;
      if (one_page) {
        int pg, row0;
        where(key0, pg, row0);
        const unsigned char* ks = kb + (int64_t)pg * p.kc_stride[0] + (int64_t)row0 * p.kc_stride[1];
        const unsigned char* vs = vb + (int64_t)pg * p.vc_stride[0] + (int64_t)row0 * p.vc_stride[1];
        const int64_t kstep = RPW * p.kc_stride[1], vstep = RPW * p.vc_stride[1];
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int bytes = key0 + i * RPW < keys ? 16 : 0;      // rows past the last key are zero-filled
          cp_async16(smem_u32(dK + i * RPW * P), bytes ? ks + i * kstep : kb, bytes);
          cp_async16(smem_u32(dV + i * RPW * P), bytes ? vs + i * vstep : vb, bytes);
        }
      } else {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int key = key0 + i * RPW;
          const int bytes = key < keys ? 16 : 0;
          int pg = 0, row = 0;
          if (bytes) where(key, pg, row);
          cp_async16(smem_u32(dK + i * RPW * P), kb + (int64_t)pg * p.kc_stride[0] + (int64_t)row * p.kc_stride[1], bytes);
          cp_async16(smem_u32(dV + i * RPW * P), vb + (int64_t)pg * p.vc_stride[0] + (int64_t)row * p.vc_stride[1], bytes);
        }
      }
    }
    ++ld;
    ld_page();
  };

#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    load_tile(i);
    cp_async_commit();
  }

  float* ws_o = reinterpret_cast<float*>(p.workspace);
  float* ws_l = ws_o + (int64_t)(gridDim.x / U) * p.heads_kv * R * D;
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
  uint32_t bq[NB][D / 16][2];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint2 x = *reinterpret_cast<const uint2*>(sQ + (n * 8 + g) * QP + kk * 16 + 4 * t);
      bq[n][kk][0] = x.x;
      bq[n][kk][1] = x.y;
    }
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

  for (int ti = 0; ti < count; ++ti) {
    const int keyw = (tile0 + ti) * kTile + warp * 16;   // this warp's first key
    cp_async_wait<NS - 2>();
    __syncwarp();
    load_tile(stage == 0 ? NS - 1 : stage - 1);
    cp_async_commit();
    unsigned char* tK = ring + (size_t)(stage * 4 + warp) * 2 * 16 * P;
    unsigned char* tV = tK + 16 * P;
    const float* tS = sS + (stage * 4 + warp) * 32;
    if (++stage == NS) stage = 0;
    if (keyw >= keys) continue;
    const float ks[2] = {tS[g] * qinv, tS[g + 8] * qinv}, vs[2] = {tS[16 + g], tS[24 + g]};
    // log2 of the V scales; a block of zeros has a small one
    const float lv[2] = {__log2f(fmaxf(vs[0], 0x1p-60f)), __log2f(fmaxf(vs[1], 0x1p-60f))};

    // ---- S^T = K Q^T: keys keyw + g and keyw + g + 8 ------------------------------------
    float s[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < (D + 31) / 32; ++kk) {
      uint32_t r[4];
      ldsm_x4(smem_u32(tK + (lane & 15) * P + kk * 32 + (D > 16 ? (lane >> 4) * 16 : 0)), r[0], r[1], r[2], r[3]);
#pragma unroll
      for (int half = 0; half < (D > 16 ? 2 : 1); ++half) {
        uint32_t a[4];
        C::neighbours(r[2 * half], a[0], a[2]);
        C::neighbours(r[2 * half + 1], a[1], a[3]);
#pragma unroll
        for (int n = 0; n < NB; ++n) mma16816<__half>(s[n], a, bq[n][2 * kk + half][0], bq[n][2 * kk + half][1]);
      }
    }
    // ---- softmax --------------------------------------------------------------------------
    const bool full = !cfg.has_alibi && keyw + 16 <= keys && (!cfg.causal || keyw + 15 <= qmin) &&
                      (cfg.wl < 0 || keyw >= qmax - cfg.wl) && (cfg.wr < 0 || keyw + 15 <= qmin + cfg.wr);
    if (full) {
      const float mul[2] = {ks[0] * cfg.scale_log2, ks[1] * cfg.scale_log2};
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] *= mul[e >> 1];
      }
    } else {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = e & 1, key = keyw + g + (e >> 1) * 8;
          float th;
          const float v = score_log2(cfg, slope[n][i], s[n][e] * ks[e >> 1], qpos[n][i], key, th);
          s[n][e] = visible(cfg, qpos[n][i], key, keys) ? v : -INFINITY;
        }
      }
    }
    float mx[NB][2];
    bool grow = false;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float m = fmaxf(s[n][i] + lv[0], s[n][2 + i] + lv[1]);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        mx[n][i] = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        grow |= mx[n][i] > mrow[n][i];
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool up = mx[n][i] > mrow[n][i];
          alpha[i] = up ? exp2f(mrow[n][i] - mx[n][i]) : 1.f;    // from -inf: 0
          if (up) mrow[n][i] = mx[n][i];
          lrow[n][i] *= alpha[i];
        }
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
          o[n][db][0] *= alpha[0]; o[n][db][1] *= alpha[1];
          o[n][db][2] *= alpha[0]; o[n][db][3] *= alpha[1];
        }
      }
    }
    uint32_t pb[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // no finite score yet: exponents relative to 0, so that -inf gives 0 and NaN stays NaN
        const float m = mrow[n][e & 1] == -INFINITY ? 0.f : mrow[n][e & 1];
        const float pe = ex2(s[n][e] - m);
        lrow[n][e & 1] += pe;
        s[n][e] = pe == 0.f ? 0.f : pe * vs[e >> 1];             // a hidden key weighs 0 whatever its scale is
      }
      // P^T[key][row] as the accumulator holds it -> B fragment [keys] x [rows]
      pb[n][0] = transpose_8x8(Elem<__half>::pack(s[n][0], s[n][1]));
      pb[n][1] = transpose_8x8(Elem<__half>::pack(s[n][2], s[n][3]));
    }
    // ---- O^T += V^T P^T -----------------------------------------------------------------
#pragma unroll
    for (int d2 = 0; d2 < (D + 31) / 32; ++d2) {
      uint32_t r[4];
      ldsm_x4_t(smem_u32(tV + (lane & 15) * P + d2 * 32 + (D > 16 ? (lane >> 4) * 16 : 0)), r[0], r[1], r[2], r[3]);
#pragma unroll
      for (int half = 0; half < (D > 16 ? 2 : 1); ++half) {
        uint32_t a[4];
        C::alternate(r[2 * half], a[0], a[1]);
        C::alternate(r[2 * half + 1], a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NB; ++n) mma16816<__half>(o[n][2 * d2 + half], a, pb[n][0], pb[n][1]);
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
  const int64_t ws_row = ((int64_t)share * p.heads_kv + hk) * R + rg * kRows;
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
        merge_pieces<T, D>(ws_o, ws_l, ((int64_t)base * p.heads_kv + hk) * R + gr, (int64_t)p.heads_kv * R, parts, (i % (D / 4)) * 4,
                           reinterpret_cast<T*>(p.o) + b * p.o_stride[0] + sq * p.o_stride[1] + (int64_t)h * p.o_stride[2]);
      }
    }
  }
}

template <typename T, int kCode, int D, int kRows>
static int launch_decode8_rows(const fa_decode_args& a, const fa_cache8& c, const ScoreCfg& cfg, const DecodeGeom& g, const DecodeCheck& chk,
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
  lc.gridDim = dim3((unsigned)g.shares * a.heads_kv * g.row_groups);
  lc.blockDim = dim3(128);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  if (behind) {
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = &attr;
    lc.numAttrs = 1;
  }
  cudaLaunchKernelEx(&lc, kern, a, c, log2_of(c.block), cfg, g, chk, behind);
  return check_launch("decode8");
}

template <typename T, int kCode, int D>
static int launch_decode8_dim(const fa_decode_args& a, const fa_cache8& c, const ScoreCfg& cfg, int unit_rows, const DecodeGeom& g,
                              const DecodeCheck& chk, bool behind, cudaStream_t st) {
  return unit_rows == 8 ? launch_decode8_rows<T, kCode, D, 8>(a, c, cfg, g, chk, behind, st)
                        : launch_decode8_rows<T, kCode, D, 16>(a, c, cfg, g, chk, behind, st);
}

template <typename T, int kCode>
static int launch_decode8(const fa_decode_args& a, const fa_cache8& c, const ScoreCfg& cfg, int unit_rows, const DecodeGeom& g,
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
