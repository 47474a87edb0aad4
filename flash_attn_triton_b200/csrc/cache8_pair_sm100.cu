// Chunks of tokens against the 8-bit KV cache on the 5th-generation tensor cores, two tiles of 128 query rows per CTA (256 rows of a KV
// head): every unit of K or V that is converted serves both.  head_dim 64 and 128; the mathematics and the conversion are those of
// cache8_chunk_sm100.cu, which keeps head_dim 256, ALiBi, chunks of at most 128 rows and scales of less than 16 tokens.
//
//   warps 0-3, 4-7   softmax of query tiles 0 and 1 ("streams"): a thread has a row, its maximum and its sum
//   warp  8          TMA producer of codes, and the scales of the tiles' keys
//   warp  9          MMA issuer: S_x = Q_x K_j^T;  O_x += P_x V_j (A = P_x from tensor memory), the streams out of phase
//   warps 10, 11     converters
//
// Tensor memory: S_0 | S_1 | O_0 | O_1.  P_x overwrites S_x, and Q_x K_(j+1)^T is issued behind P_x V_j, which reads it, in the in-order pipe.
// With 12 warps the softmax warps have 216 registers, and all scores of a row fit (16 warps with one query tile: 184 and two readings).
// Why two tiles: with one, the converters have 1100 (e4m3) to 1800 (int8) cycles of work for 1024 of the tensor pipe.  2 x 1537 tokens behind
// 5000 to 11000, 32 heads over 8 of 128, int8: fp16 1249 us with one, 856 with two (660 TFLOP/s of a call over other inputs in turn), bf16 1134,
// 778; 16 x 64 behind 1024 to 8192, e4m3: 218, 210; 4 x 256: 195, 199.
// Bound: the chain of a tile (fp16, before maxima were raised at once): 1.5 k cycles from the last of P to the next scores, 0.7 k load and maximum, 2.2 k exponentials and P; 5.2 k cycles
// per two tiles of which the tensor pipe needs 2.0 k.  A quarter of the exponentials on the FMA pipe: 5 % slower (registers).
// Every mbarrier wait is bounded; on timeout the CTA raises a status word, frees its tensor memory and returns.
#include <cmath>
#include <type_traits>

#include "cache8.cuh"
#include "cache8_host.h"
#include "sm100.cuh"

namespace fa {

using namespace sm100;

__device__ int g_cache8_pair_status = 0;

namespace {

constexpr int kBM = 128;          // query rows of a tile
constexpr int kRows = 256;        // of the CTA
constexpr int kBN = 128;          // keys per tile
constexpr int kThreads = 384;
constexpr int kMaxStages = 8;
constexpr int kScaleBufs = 8;

template <int D> struct PCfg {
  static constexpr int kUnitBytes = kBN * D * 2;                    // a K or V tile
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kRaw = D == 128 ? 3 : 6;                     // tiles of codes on their way
  static constexpr int kRawBytes = kBN * D;
  static constexpr int kChunks = kRawBytes / 16 / 64;               // 16-byte chunks of a unit per converter thread
  static constexpr int kOCol = 256;                                 // first column of the accumulators
  static constexpr int kQBytes = kBM * D * 2;                       // of a stream
  static constexpr int kRawAt = 2 * kQBytes + kStages * kUnitBytes;
  static constexpr int kShared = kRawAt + kRaw * kRawBytes;
  static constexpr int kSmemBytes = kShared + 1024 /*align slack*/ + 2048 /*PShared*/;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
  // Pieces of the keys, at most: a merge keeps a weight per piece and row over both rings.
  static constexpr int kPieces = (kShared - 2 * kQBytes) / (kRows * (int)sizeof(float));
};

struct PShared {
  uint64_t q_full;
  uint64_t kv_full[kMaxStages];
  uint64_t kv_empty[kMaxStages];
  uint64_t raw_full[kMaxStages];
  uint64_t raw_empty[kMaxStages];  // (one arrival of each converter warp)
  uint64_t s_full[2];      // [stream]: scores computed
  uint64_t p_half[2];      // [stream]: the first 64 keys of P written back (128 arrivals)
  uint64_t p_ready[2];     // [stream]: P written back (128 arrivals)
  uint64_t o_done[2];      // [stream]: its P V finished
  uint64_t sc_full[kScaleBufs];    // scales of tile j in buffer j % kScaleBufs
  uint64_t sc_empty[kScaleBufs];   // read (one arrival of each softmax warp)
  uint32_t tmem_base;
  volatile int abort_flag;
  int last;                // split keys: this CTA merges the pieces
  uint32_t qmost[8];
  alignas(16) float ks[kScaleBufs][kBN / 16];   // scales of each 16 keys
  alignas(16) float vs[kScaleBufs][kBN / 16];
  alignas(16) float lv[kScaleBufs][kBN / 16];   // log2 of the magnitude of those of V
};
static_assert(sizeof(PShared) <= 2048, "PShared must fit its reserve");

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, PShared* sh, int code) {
  return bounded_wait(bar, parity, &sh->abort_flag, &g_cache8_pair_status, code);
}

__device__ __forceinline__ uint2 ld_shared_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// Barrier 1 of the 256 softmax threads: is the predicate set in any of them?
__device__ __forceinline__ bool any_of_256(bool x) {
  int r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.s32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, 1, 256, p;\n"
      "selp.s32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r) : "r"((int)x) : "memory");
  return r != 0;
}

// What a CTA works on.
struct Tile {
  int b, h, hk;            // sequence; first query head of the rows; KV head
  int m0, rows;            // first row of the tile, rows of the problem (tokens * packed heads)
  int pos0;                // position of row r: pos0 + (r >> pack_log2)
  int keys, pad;           // keys the cache holds of the sequence; rows in front of them
  int n_hi, nt;            // key tiles [n_hi - nt, n_hi); tile j of the CTA is n_hi - 1 - j
  int part, parts;         // piece of the keys
};

}  // namespace

// T: type of q and o.
template <typename T, int kCode, int D>
__global__ void __launch_bounds__(kThreads, 1)
cache8_pair_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmO, const fa_decode_args p, const fa_cache8 c8, const int block_shift,
                    const ScoreCfg cfg, const CacheGeo geo, int* const host_status) {
  using C = PCfg<D>;
  using K8 = Code<kCode>;
  constexpr int S = C::kStages;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  PShared* sh = reinterpret_cast<PShared*>(tiles + C::kShared);
  const uint32_t sQ = smem_u32(tiles);
  const uint32_t sKV = sQ + 2 * C::kQBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // behind the append and the checks (a programmatic launch)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (geo.bad && *geo.bad) return;

  // ---- what this CTA works on --------------------------------------------------------------
  Tile w;
  {
    const int heads = p.heads_q >> geo.pack_log2;        // units of heads per sequence
    w.rows = geo.tokens << geo.pack_log2;
    const int mtiles = (w.rows + kRows - 1) / kRows;
    int i = blockIdx.x;
    w.part = i % geo.parts;
    i /= geo.parts;
    const int mt = mtiles - 1 - i % mtiles;
    i /= mtiles;
    const int hu = i % heads, rank = i / heads;
    // long sequences first (their CTAs set the time of the launch)
    w.b = rank;
    if (p.batch > 1 && p.batch <= 32) {
      const int mine = lane < p.batch ? geo.seqlens[lane] : -1;
      int before = 0;
      for (int o = 0; o < p.batch; ++o) {
        const int other = __shfl_sync(0xffffffffu, mine, o);
        before += other > mine || (other == mine && o < lane);
      }
      w.b = __ffs(__ballot_sync(0xffffffffu, lane < p.batch && before == rank)) - 1;
    }
    w.h = hu << geo.pack_log2;
    w.hk = w.h / (p.heads_q / p.heads_kv);
    w.m0 = mt * kRows;
    const int cap = seq_capacity(p, w.b), len = max(0, min(geo.seqlens[w.b], cap)) + geo.n_new;
    w.keys = min(len, cap);
    w.pos0 = len - geo.tokens;
    w.pad = geo.leftpad ? max(0, geo.leftpad[w.b]) : 0;
  }
  const int tq_min = w.pos0 + (w.m0 >> geo.pack_log2);
  const int tq_max = w.pos0 + ((min(w.m0 + kRows, w.rows) - 1) >> geo.pack_log2);
  {
    int klo, khi;
    visible_key_range(cfg, tq_min, tq_max, w.keys, klo, khi);
    const int lo = klo / kBN, hi = (khi + kBN - 1) / kBN;
    const int all = khi > klo ? hi - lo : 0;
    w.parts = chunk_pieces(p, cfg, geo, (p.heads_q >> geo.pack_log2) * ((w.rows + kRows - 1) / kRows), all, lane);
    if (w.part >= w.parts) return;
    const int first = (int)((int64_t)w.part * all / w.parts), last = (int)((int64_t)(w.part + 1) * all / w.parts);
    w.n_hi = lo + last;
    w.nt = last - first;
  }
  const int nt = w.nt;

  if (tid == 0) {
    mbar_init(smem_u32(&sh->q_full), 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh->s_full[i]), 1);
      mbar_init(smem_u32(&sh->o_done[i]), 1);
      mbar_init(smem_u32(&sh->p_half[i]), 128);
      mbar_init(smem_u32(&sh->p_ready[i]), 128);
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(&sh->kv_full[i]), 2);
      mbar_init(smem_u32(&sh->kv_empty[i]), 1);
    }
    for (int i = 0; i < C::kRaw; ++i) {
      mbar_init(smem_u32(&sh->raw_full[i]), 1);
      mbar_init(smem_u32(&sh->raw_empty[i]), 2);
    }
    for (int i = 0; i < kScaleBufs; ++i) {
      mbar_init(smem_u32(&sh->sc_full[i]), 1);
      mbar_init(smem_u32(&sh->sc_empty[i]), 8);
    }
    sh->abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
    prefetch_tmap(&tmO);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(&sh->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const uint32_t raw0 = sQ + C::kRawAt;
  const int total = 2 * nt;                              // units K_0, V_0, K_1, V_1, ...

  if (warp >= 8) {
    reg_dealloc<72>();
    auto page_index = [&](int key) { return divided(key, geo.page_size, geo.page_log2); };
    if (warp >= 10) {
      // ------------------------------- converters -----------------------------------------
      const int ct = tid - 320;
      constexpr int CPR = D / 16;                        // 16-byte chunks of a row
      // This thread's chunk i of a unit: row first + i * kStep, column col.  Lanes of the two 64-column boxes of a row take the halves
      // of a chunk in opposite order: other banks.
      constexpr int kStep = 64 / CPR;
      const int first = ct / CPR, col = (ct % CPR) * 16;
      const uint32_t turn = (uint32_t)(col >> 6) & 1u;
      const uint32_t put = (uint32_t)(col >> 6) * (kBN * 128) + (uint32_t)first * 128;
      const uint32_t put0 = put + (((((uint32_t)col >> 3) & 7u) + turn) ^ (first & 7)) * 16;
      const uint32_t put1 = put + (((((uint32_t)col >> 3) & 7u) + (turn ^ 1u)) ^ (first & 7)) * 16;
      int stage = 0, slot = 0;
      uint32_t phase = 0, sphase = 0;
      bool ok = true;
      for (int n = 0; n < total; ++n) {
        ok = wait_bar(&sh->raw_full[slot], sphase, sh, 13);
        if (!ok) break;
        const uint32_t from = raw0 + slot * C::kRawBytes + ct * 16, dst = sKV + stage * C::kUnitBytes;
        const int left = w.keys - (w.n_hi - 1 - (n >> 1)) * kBN;
#pragma unroll 1
        for (int i0 = 0; i0 < C::kChunks; i0 += 8) {
          uint2 u[8], v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            u[i] = ld_shared_v2(from + (i0 + i) * 1024 + turn * 8);
            v[i] = ld_shared_v2(from + (i0 + i) * 1024 + (turn ^ 1u) * 8);
          }
          if (left < kBN) {                              // rows past the last key hold anything: zeros
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (first + (i0 + i) * kStep >= left) u[i] = v[i] = make_uint2(0u, 0u);
          }
          if (i0 == 0) ok = wait_bar(&sh->kv_empty[stage], phase ^ 1, sh, 11);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint4 a, b;
            K8::integers(u[i].x, a.x, a.y);
            K8::integers(u[i].y, a.z, a.w);
            K8::integers(v[i].x, b.x, b.y);
            K8::integers(v[i].y, b.z, b.w);
            st_shared_v4(dst + put0 + (i0 + i) * (kStep * 128), a);
            st_shared_v4(dst + put1 + (i0 + i) * (kStep * 128), b);
          }
        }
        if (!ok) break;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&sh->raw_empty[slot]));
          mbar_arrive(smem_u32(&sh->kv_full[stage]));
        }
        if (++stage == S) { stage = 0; phase ^= 1; }
        if (++slot == C::kRaw) { slot = 0; sphase ^= 1; }
      }
    } else if (warp == 8 && nt > 0) {
      // ------------------------------- TMA producer, scales -----------------------------------
      // A unit is boxes of geo.box_rows keys that lie inside one page each; lane i brings box i.  Boxes that start past the last key
      // are left out.  The scales: lane i those of keys 16 i to 16 i + 15 of K (i < 8) or of V.  Pages are read one tile ahead of
      // their use, scales too.
      const int box_log2 = 31 - __clz(geo.box_rows);
      auto page_at = [&](int j, int offset) {            // of the key `offset` keys into tile j
        if (geo.table == nullptr) return geo.batch_idx ? geo.batch_idx[w.b] : w.b;
        const int key = (w.n_hi - 1 - j) * kBN + offset;
        return j < nt && offset < kBN && key < w.keys ? geo.table[(int64_t)w.b * geo.table_stride + page_index(key)] : 0;
      };
      const bool of_v = lane >= 8;
      const float* sbase = of_v ? c8.v_scale + (int64_t)w.hk * c8.vs_stride[2] : c8.k_scale + (int64_t)w.hk * c8.ks_stride[2];
      const int64_t s0 = of_v ? c8.vs_stride[0] : c8.ks_stride[0], s1 = of_v ? c8.vs_stride[1] : c8.ks_stride[1];
      auto scale_at = [&](int j, int pg) {
        const int key = (w.n_hi - 1 - j) * kBN + (lane & 7) * 16;
        if (lane >= 16 || j >= nt || key >= w.keys) return 0.f;
        const int row = geo.table ? key - page_index(key) * geo.page_size : key;
        return sbase[pg * s0 + divided(row, c8.block, block_shift) * s1];
      };
      int slot = 0, pg = page_at(0, lane << box_log2), pgs = page_at(0, (lane & 7) * 16);
      float sc = scale_at(0, pgs);
      pgs = page_at(1, (lane & 7) * 16);
      uint32_t sphase = 0;
      bool ok = true;
      int n = 0;
      for (int j = 0; j < nt && ok; ++j) {
        const int k0 = (w.n_hi - 1 - j) * kBN, key = k0 + (lane << box_log2);
        const int row = geo.table ? key - page_index(key) * geo.page_size : key;
        const int boxes = min(kBN >> box_log2, ((w.keys - k0 - 1) >> box_log2) + 1);
        // A scale of V that is no number or infinite goes to the scores instead, which the mask takes out where the key is hidden
        // (0 times either would not be 0).
        const bool odd = !(fabsf(sc) <= 3.4e38f);
        const unsigned spoilt = __ballot_sync(0xffffffffu, odd && of_v) >> 8;
        const float now = of_v ? (odd ? 0.f : sc) : (spoilt >> (lane & 7)) & 1u ? NAN : sc;
        sc = scale_at(j + 1, pgs);
        pgs = page_at(j + 2, (lane & 7) * 16);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t bar = smem_u32(&sh->raw_full[slot]), dst = raw0 + slot * C::kRawBytes;
          if (lane == 0) ok = wait_bar(&sh->raw_empty[slot], sphase ^ 1, sh, 12);
          ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(bar, boxes * (D << box_log2));
          __syncwarp();
          if (lane < boxes) tma_load_4d(dst + (lane << box_log2) * D, kv ? &tmV : &tmK, bar, 0, w.hk, row, pg);
          ++n;
          if (++slot == C::kRaw) { slot = 0; sphase ^= 1; }
          if (kv == 0) {
            const int sb = j % kScaleBufs;
            if (lane == 0) ok = wait_bar(&sh->sc_empty[sb], ((j / kScaleBufs) & 1) ^ 1, sh, 14);
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            if (!ok) break;
            if (lane < 16) (of_v ? sh->vs[sb] : sh->ks[sb])[lane & 7] = now;
            if (of_v && lane < 16) sh->lv[sb][lane & 7] = __log2f(fmaxf(fabsf(now), 0x1p-60f));
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh->sc_full[sb]));
          }
        }
        pg = page_at(j + 1, lane << box_log2);
      }
      // a CTA that gives up still waits for the copies that are on their way to it
      if (!ok)
        for (int m = max(0, n - C::kRaw); m < n; ++m)
          for (int i = 0; i < 1 << 16 && !mbar_try_wait(smem_u32(&sh->raw_full[m % C::kRaw]), (m / C::kRaw) & 1); ++i) {}
    } else if (warp == 9 && nt > 0) {
      // ------------------------------- MMA issuer -------------------------------------------
      // The whole warp runs the control flow in lock step and every lane polls the barriers;
      // the lane chosen once by elect_one issues the MMAs and commits.
      constexpr uint32_t idesc_qk = make_idesc(1, 0, 0, 0, kBM, kBN);
      constexpr uint32_t idesc_pv = make_idesc(1, 0, 0, 1, kBM, D);
      const uint32_t leader = elect_one() ? 1u : 0u;
      bool ok = true;
      auto wwait = [&](uint64_t* bar, uint32_t parity, int code) {
        if (ok) ok = wait_bar(bar, parity, sh, code);
        tc_fence_after();
      };
      auto issue_qk = [&](int x, int stage) {
        const uint64_t dq = make_smem_desc(sQ + x * C::kQBytes, 16, 1024);
        const uint64_t dk = make_smem_desc(sKV + stage * C::kUnitBytes, 16, 1024);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t o = ((kk / 4) * (kBM * 128) + (kk % 4) * 32) >> 4;
          mma_f16_ss_lp(tmem + x * kBN, dq + o, dk + o, idesc_qk, kk > 0 ? 1u : 0u, leader);
        }
        mma_commit_lp(smem_u32(&sh->s_full[x]), leader);
      };
      wwait(&sh->q_full, 0, 21);
      wwait(&sh->kv_full[0], 0, 22);
      if (ok) {
        issue_qk(0, 0);
        issue_qk(1, 0);
        mma_commit_lp(smem_u32(&sh->kv_empty[0]), leader);
      }
      int sv = 1 % S, sk = 2 % S;                          // stages of V_j and K_(j+1)
      uint32_t pv = 1 / S, pk = 2 / S;
      for (int j = 0; j < nt && ok; ++j) {
        wwait(&sh->kv_full[sv], pv & 1, 24);
        if (!ok) break;
        const uint64_t dv = make_smem_desc(sKV + sv * C::kUnitBytes, kBN * 128, 1024);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t a = tmem + x * kBN, d = tmem + C::kOCol + x * D;
          wwait(&sh->p_half[x], j & 1, 25);
          if (!ok) break;
#pragma unroll
          for (int kk = 0; kk < kBN / 32; ++kk)
            mma_f16_ts_lp(d, a + kk * 8, dv + ((kk * 2048) >> 4), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u, leader);
          wwait(&sh->p_ready[x], j & 1, 26);
          if (!ok) break;
#pragma unroll
          for (int kk = kBN / 32; kk < kBN / 16; ++kk)
            mma_f16_ts_lp(d, a + kk * 8, dv + ((kk * 2048) >> 4), idesc_pv, 1u, leader);
          mma_commit_lp(smem_u32(&sh->o_done[x]), leader);
          if (x == 1) mma_commit_lp(smem_u32(&sh->kv_empty[sv]), leader);
          if (j + 1 < nt) {
            if (x == 0) wwait(&sh->kv_full[sk], pk & 1, 22);
            if (!ok) break;
            issue_qk(x, sk);
            if (x == 1) mma_commit_lp(smem_u32(&sh->kv_empty[sk]), leader);
          }
        }
        sv += 2;
        if (sv >= S) { sv -= S; ++pv; }
        sk += 2;
        if (sk >= S) { sk -= S; ++pk; }
      }
    }
  } else {
    // ------------------------------- softmax of a stream ----------------------------------
    reg_alloc<216>();
    const int x = warp >> 2;                         // stream
    // ---- Q: rotated, to fp16 (bf16: times the power of two that brings the largest element of the rows to [2^14, 2^15)), swizzled
    float qinv = 1.f;
    {
      constexpr int QC = D / 8, NQ = kRows * QC / 256, kAtOnce = NQ < 16 ? NQ : 16;
      const T* cos = reinterpret_cast<const T*>(p.rotary_cos);
      const T* sin = reinterpret_cast<const T*>(p.rotary_sin);
      // (rows past the last one read it and are cleared behind the loads: a branch around each load put them one behind the other, 8 us)
      auto load = [&](int k) {
        const int i = k * 256 + tid, r = min(w.m0 + i / QC, w.rows - 1), d = i % QC * 8;
        const int tok = r >> geo.pack_log2, h = w.h + (r & ((1 << geo.pack_log2) - 1));
        const T* row = reinterpret_cast<const T*>(p.q) + w.b * p.q_stride[0] + tok * p.q_stride[1] + (int64_t)h * p.q_stride[2];
        if (cos == nullptr) return *reinterpret_cast<const uint4*>(row + d);
        return rotary_chunk<T, true>(row, d, cos, sin, w.pos0 + tok + w.pad, p.rotary_dim, p.rotary_interleaved, p.rotary_seqlen);
      };
      auto load_all = [&](int k0, uint4* to) {
        if (cos == nullptr) {
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) to[k] = load(k0 + k);
        } else {
#pragma unroll 1
          for (int k = 0; k < kAtOnce; ++k) {
            const uint4 v = load(k0 + k);
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e)
              if (e == k) to[e] = v;
          }
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          if (w.m0 + ((k0 + k) * 256 + tid) / QC >= w.rows) to[k] = make_uint4(0u, 0u, 0u, 0u);
      };
      auto store = [&](int k, uint4 v, float mul) {
        const int i = k * 256 + tid, r = i / QC, c = i % QC;
        if (std::is_same<T, __nv_bfloat16>::value) {
          uint32_t* x = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = Elem<T>::unpack(x[e]);
            x[e] = Elem<__half>::pack(f.x * mul, f.y * mul);
          }
        }
        st_shared_v4(sw128_addr(sQ + (r / kBM) * C::kQBytes + (c >> 3) * (kBM * 128), r % kBM, c & 7), v);
      };
      float qmul = 1.f;
      uint4 held[kAtOnce];
      if (std::is_same<T, __nv_bfloat16>::value) {
        uint32_t most = 0u;
        for (int k0 = NQ - kAtOnce; k0 >= 0; k0 -= kAtOnce) {        // the first ones stay
          load_all(k0, held);
#pragma unroll
          for (int k = 0; k < kAtOnce; ++k) {
            const uint32_t* x = reinterpret_cast<const uint32_t*>(&held[k]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t m = (x[e >> 1] >> (16 * (e & 1))) & 0x7fffu;
              most = max(most, m < 0x7f80u ? m : 0u);                // the largest number
            }
          }
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) sh->qmost[warp] = most;
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, sh->qmost[i]);
        const int e = min(14 - ((int)(most >> 7) - 127), 126);
        if (most != 0u) {
          qmul = __int_as_float((e + 127) << 23);
          qinv = __int_as_float((127 - e) << 23);
        }
      }
      for (int k0 = 0; k0 < NQ; k0 += kAtOnce) {
        if (k0 > 0 || !std::is_same<T, __nv_bfloat16>::value) {
          load_all(k0, held);
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) store(k0 + k, held[k], qmul);
      }
      fence_proxy_async();
      mbar_arrive(smem_u32(&sh->q_full));
    }
    const int row_in_tile = (warp & 3) * 32 + lane;  // TMEM lane
    const int row = w.m0 + x * kBM + row_in_tile;
    const int qpos = w.pos0 + (row >> geo.pack_log2);
    const int sq_min = w.pos0 + ((w.m0 + x * kBM) >> geo.pack_log2), sq_end = w.pos0 + ((w.m0 + x * kBM + kBM - 1) >> geo.pack_log2);
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_addr + C::kOCol + x * D, tS = tmem + lane_addr + x * kBN;
    const float f = cfg.scale_log2 * qinv;
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;

    for (int j = 0; j < nt; ++j) {
      const int k0 = (w.n_hi - 1 - j) * kBN;
      bool masked = (k0 + kBN > w.keys);
      if (cfg.causal) masked |= (k0 + kBN - 1 > sq_min);
      if (cfg.wl >= 0) masked |= (k0 < sq_end - cfg.wl);
      if (cfg.wr >= 0) masked |= (k0 + kBN - 1 > sq_min + cfg.wr);
      const int sb = j % kScaleBufs;
      ok = wait_bar(&sh->sc_full[sb], (j / kScaleBufs) & 1, sh, 29);
      if (!ok) break;
      // mg of each 16 keys turns their scores into the log2 domain.  Masked tiles go there at once, through tensor memory in a rolled loop:
      // with copies of the passes below for them, the code that every tile runs was slower by 14 % (instruction cache).  So do tiles with a
      // negative scale of K, whose largest score has the smallest product (seen before the scores are there, it costs nothing).
      float mg[8];
      {
        const float4 a = *reinterpret_cast<const float4*>(&sh->ks[sb][0]), b = *reinterpret_cast<const float4*>(&sh->ks[sb][4]);
        mg[0] = a.x * f; mg[1] = a.y * f; mg[2] = a.z * f; mg[3] = a.w * f;
        mg[4] = b.x * f; mg[5] = b.y * f; mg[6] = b.z * f; mg[7] = b.w * f;
        masked |= fminf(fminf(fminf(a.x, a.y), fminf(a.z, a.w)), fminf(fminf(b.x, b.y), fminf(b.z, b.w))) < 0.f;
      }
      ok = wait_bar(&sh->s_full[x], j & 1, sh, 31 + x);
      if (!ok) break;
      tc_fence_after();
      if (masked) {
        int vk_lo, vk_hi;
        visible_k_interval(cfg, qpos, w.keys, vk_lo, vk_hi);
#pragma unroll 1
        for (int cc = 0; cc < 4; ++cc) {
          const ColMask cm = make_col_mask(vk_lo - k0 - cc * 32, vk_hi - k0 - cc * 32);
          const float2 k2 = *reinterpret_cast<const float2*>(&sh->ks[sb][cc * 2]);
          uint32_t ra[32];
          tmem_ld32(tS + cc * 32, ra);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float v = __uint_as_float(ra[i]) * (i < 16 ? k2.x : k2.y) * f;
            ra[i] = __float_as_uint(col_visible(cm, i) ? v : -INFINITY);
          }
          tmem_st32(tS + cc * 32, ra);
        }
        tmem_wait_st();
#pragma unroll
        for (int g = 0; g < 8; ++g) mg[g] = 1.f;
      }

      // ---- the 128 scores of this row into registers -------------------------------------
      uint32_t r[4][32];
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) tmem_ld32(tS + cc * 32, r[cc]);
      tmem_wait_ld();

      // ---- row maximum of t + log2 |vs| -----------------------------------------------------------
      float mx = -INFINITY;
      {
        const float4 a = *reinterpret_cast<const float4*>(&sh->lv[sb][0]), b = *reinterpret_cast<const float4*>(&sh->lv[sb][4]);
        const float lv[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const uint32_t* v = &r[g >> 1][(g & 1) * 16];
          float m[5];
#pragma unroll
          for (int i = 0; i < 5; ++i)
            m[i] = fmax3(__uint_as_float(v[3 * i]), __uint_as_float(v[3 * i + 1]), __uint_as_float(v[3 * i + 2]));
          const float most = fmaxf(fmax3(m[0], m[1], m[2]), fmax3(m[3], m[4], __uint_as_float(v[15])));
          mx = fmaxf(mx, fmaf(most, mg[g], lv[g]));
        }
      }
      const bool need = mx > m_run + cfg.rescale_at || j == 0;
      const float alpha = need ? exp2f(m_run - mx) : 1.f;        // from -inf: 0 (-inf - -inf: not used)
      if (j > 0 && __any_sync(0xffffffffu, need)) {
        // (the scores of this tile were computed behind P V of the one before: it is finished)
        ok = wait_bar(&sh->o_done[x], (j - 1) & 1, sh, 35 + x);
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t ro[32];
          tmem_ld32(tO + cc * 32, ro);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ro[i] = __float_as_uint(__uint_as_float(ro[i]) * alpha);
          tmem_st32(tO + cc * 32, ro);
        }
        tmem_wait_st();
        tc_fence_before();
      }
      if (need) {
        m_run = mx;
        l_run = j == 0 ? 0.f : l_run * alpha;
      }
      const float m_safe = m_run == -INFINITY ? 0.f : m_run;

      // ---- p = exp2(t - M), row sum, p vs -> TMEM in place over S ----------------------------
      const float2 nm2 = make_float2(-m_safe, -m_safe);
      float2 acc2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        const float2 v16 = *reinterpret_cast<const float2*>(&sh->vs[sb][cc * 2]);
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float g = mg[cc * 2 + (i >> 4)], v = i < 16 ? v16.x : v16.y;
          const float2 a = f2fma(make_float2(__uint_as_float(r[cc][i]), __uint_as_float(r[cc][i + 1])), make_float2(g, g), nm2);
          const float2 pe = make_float2(ex2(a.x), ex2(a.y));
          acc2[(i >> 1) & 1] = f2add(acc2[(i >> 1) & 1], pe);
          const float2 wt = f2mul(pe, make_float2(v, v));
          pk[i >> 1] = Elem<__half>::pack(wt.x, wt.y);
        }
        tmem_st16(tS + cc * 16, pk);
        if (cc == 1) {
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(smem_u32(&sh->p_half[x]));
        }
      }
      l_run += (acc2[0].x + acc2[0].y) + (acc2[1].x + acc2[1].y);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(smem_u32(&sh->p_ready[x]));
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh->sc_empty[sb]));
    }

    // ---- epilogue ---------------------------------------------------------------------------
    if (ok && nt > 0) ok = wait_bar(&sh->o_done[x], (nt - 1) & 1, sh, 37 + x);
    const bool failed = any_of_256(!ok || sh->abort_flag != 0);
    tc_fence_after();
    if (!failed) {
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
      const float lse = l_run == 0.f ? -INFINITY : m_run + log2f(l_run);
      const bool row_ok = row < w.rows, piece = w.parts > 1;
      const int64_t slot = blockIdx.x;
#pragma unroll
      for (int cc = 0; cc < D / 32; ++cc) {
        uint32_t ra[32];
        if (nt > 0) {
          tmem_ld32(tO + cc * 32, ra);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) ra[i] = 0u;
        }
        if (piece) {
          float* dst = geo.ws + (slot * kRows + x * kBM + row_in_tile) * D + cc * 32;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            if (row_ok)
              *reinterpret_cast<float4*>(dst + i) = make_float4(__uint_as_float(ra[i]) * inv, __uint_as_float(ra[i + 1]) * inv,
                                                                __uint_as_float(ra[i + 2]) * inv, __uint_as_float(ra[i + 3]) * inv);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 v;
            v.x = Elem<T>::pack(__uint_as_float(ra[i]) * inv, __uint_as_float(ra[i + 1]) * inv);
            v.y = Elem<T>::pack(__uint_as_float(ra[i + 2]) * inv, __uint_as_float(ra[i + 3]) * inv);
            v.z = Elem<T>::pack(__uint_as_float(ra[i + 4]) * inv, __uint_as_float(ra[i + 5]) * inv);
            v.w = Elem<T>::pack(__uint_as_float(ra[i + 6]) * inv, __uint_as_float(ra[i + 7]) * inv);
            const int col = cc * 32 + i;
            st_shared_v4(sw128_addr(sQ + x * C::kQBytes + (col / 64) * (kBM * 128), row_in_tile, (col % 64) / 8), v);
          }
        }
      }
      if (!piece) {
        // staged over the Q tile, which no MMA reads any more
        fence_proxy_async();
        asm volatile("bar.sync %0, 128;\n" ::"r"(2 + x) : "memory");
        if (row_in_tile == 0 && row < w.rows) {
#pragma unroll
          for (int bx = 0; bx < D / 64; ++bx)
            tma_store_4d(&tmO, sQ + x * C::kQBytes + bx * (kBM * 128), bx * 64, w.h, (w.m0 + x * kBM) >> geo.pack_log2, w.b);
          tma_store_commit();
          tma_store_wait_read();
        }
      }
      if (piece) {
        // the CTA that finishes last merges; pieces are ordered before the count by the fence of each writer
        float* ws_l = geo.ws + (int64_t)gridDim.x * kRows * D;
        if (row_ok) ws_l[slot * kRows + x * kBM + row_in_tile] = lse;
        __threadfence();
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        if (tid == 0) {
          uint32_t* ctr = geo.counters + blockIdx.x / geo.parts;
          sh->last = atomicAdd(ctr, 1u) == (uint32_t)(w.parts - 1);
          if (sh->last) *ctr = 0u;
        }
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        if (sh->last) {
          __threadfence();
          const int64_t p0 = (int64_t)(blockIdx.x / geo.parts) * geo.parts;
          const int rows = min(kRows, w.rows - w.m0);
          // weights of the pieces per row, over the rings (every K/V tile has been read); w.parts <= geo.parts <= C::kPieces
          float* wt = reinterpret_cast<float*>(tiles + 2 * C::kQBytes);
          if (tid < rows) {
            float m = -INFINITY, sum = 0.f;
            for (int s = 0; s < w.parts; ++s) m = fmaxf(m, ws_l[(p0 + s) * kRows + tid]);
            for (int s = 0; s < w.parts; ++s) {
              const float v = m == -INFINITY ? 0.f : exp2f(ws_l[(p0 + s) * kRows + tid] - m);
              wt[s * kRows + tid] = v;
              sum += v;
            }
            const float g = sum > 0.f ? 1.f / sum : 0.f;
            for (int s = 0; s < w.parts; ++s) wt[s * kRows + tid] *= g;
          }
          asm volatile("bar.sync 1, 256;\n" ::: "memory");
          // four elements of four rows per thread at a time, two pieces in flight each
          constexpr int kStep = 256 / (D / 4);             // rows between a thread's items
          const int d = (tid % (D / 4)) * 4;
          for (int r0 = tid / (D / 4); r0 < rows; r0 += 4 * kStep) {
            float4 acc[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
            for (int s = 0; s < w.parts; ++s) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int r = min(r0 + k * kStep, rows - 1);
                const float4 v = *reinterpret_cast<const float4*>(geo.ws + ((p0 + s) * kRows + r) * D + d);
                const float g = wt[s * kRows + r];
                acc[k].x += g * v.x; acc[k].y += g * v.y; acc[k].z += g * v.z; acc[k].w += g * v.w;
              }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = r0 + k * kStep, gr = w.m0 + r;
              if (r >= rows) break;
              uint2 pk;
              pk.x = Elem<T>::pack(acc[k].x, acc[k].y);
              pk.y = Elem<T>::pack(acc[k].z, acc[k].w);
              *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.o) + (int64_t)w.b * p.o_stride[0] +
                                        (int64_t)(gr >> geo.pack_log2) * p.o_stride[1] +
                                        (int64_t)(w.h + (gr & ((1 << geo.pack_log2) - 1))) * p.o_stride[2] + d) = pk;
            }
          }
        }
      }
    } else if (w.parts > 1 && tid == 0) {
      // A piece whose wait ran out counts too: the counters outlive the call and have to be zero again once the
      // status has been cleared.  (If another CTA is the last, it merges what there is: the call has failed.)
      uint32_t* ctr = geo.counters + blockIdx.x / geo.parts;
      if (atomicAdd(ctr, 1u) == (uint32_t)(w.parts - 1)) *ctr = 0u;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, 512);
  if (tid == 0) report_abort(sh->abort_flag, host_status);
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
template <typename T, int kCode, int D>
static int launch_pair8(const fa_decode_args& d, const fa_cache8& c, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st) {
  if (geo.parts > PCfg<D>::kPieces) {
    set_error("cache8_pair: %d pieces, %d at most", geo.parts, PCfg<D>::kPieces);
    return FA_ERR_LAUNCH;
  }
  const int pack = 1 << geo.pack_log2;
  CUtensorMap tm[3];
  // codes as they lie, no swizzle: their readers are threads
  auto codes = [&](CUtensorMap* m, const void* base, const int64_t* stride) {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)d.heads_kv, (uint64_t)d.page_size, (uint64_t)d.num_pages};
    const uint64_t strides[3] = {(uint64_t)stride[2], (uint64_t)stride[1], (uint64_t)stride[0]};
    const uint32_t box[4] = {(uint32_t)D, 1, (uint32_t)geo.box_rows, 1};
    return encode_tmap(m, base, 1, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
  };
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)d.heads_q, (uint64_t)d.seqlen_q, (uint64_t)d.batch};
  const uint64_t strides[3] = {(uint64_t)d.o_stride[2] * 2, (uint64_t)d.o_stride[1] * 2, (uint64_t)d.o_stride[0] * 2};
  const uint32_t box[4] = {64, (uint32_t)pack, (uint32_t)(kBM / pack), 1};
  if (!codes(&tm[0], d.k_cache, d.kc_stride) || !codes(&tm[1], d.v_cache, d.vc_stride) || !encode_tmap(&tm[2], d.o, 2, 4, dims, strides, box)) {
    set_error("cache8_pair: cuTensorMapEncodeTiled failed");
    return FA_ERR_LAUNCH;
  }
  auto kern = cache8_pair_kernel<T, kCode, D>;
  constexpr int smem = PCfg<D>::kSmemBytes;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_error("cache8_pair: cudaFuncSetAttribute(%d): %s", smem, cudaGetErrorString(e));
    return FA_ERR_LAUNCH;
  }
  const int mtiles = (d.seqlen_q * pack + kRows - 1) / kRows;
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  lc.gridDim = dim3((unsigned)d.batch * (d.heads_q / pack) * mtiles * geo.parts);
  lc.blockDim = dim3(kThreads);
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  // without an append or a check kernel in front of it there is nothing in this call to be behind
  lc.attrs = &attr;
  lc.numAttrs = geo.n_new > 0 || geo.bad != nullptr ? 1 : 0;
  cudaLaunchKernelEx(&lc, kern, tm[0], tm[1], tm[2], d, c, log2_of(c.block), cfg, geo, host_wait_word(d.device));
  return check_launch("cache8_pair");
}

template <typename T>
static int launch_pair8_of(const fa_decode_args& d, const fa_cache8& c, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st) {
  if (c.code == FA_CODE_INT8)
    return d.head_dim == 64 ? launch_pair8<T, FA_CODE_INT8, 64>(d, c, geo, cfg, st) : launch_pair8<T, FA_CODE_INT8, 128>(d, c, geo, cfg, st);
  return d.head_dim == 64 ? launch_pair8<T, FA_CODE_E4M3, 64>(d, c, geo, cfg, st) : launch_pair8<T, FA_CODE_E4M3, 128>(d, c, geo, cfg, st);
}

int cache8_pair(const fa_decode_args& d, const fa_cache8& c, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st) {
  return d.dtype == FA_BF16 ? launch_pair8_of<__nv_bfloat16>(d, c, geo, cfg, st) : launch_pair8_of<__half>(d, c, geo, cfg, st);
}

int cache8_pair_pieces(int head_dim) { return head_dim == 64 ? PCfg<64>::kPieces : PCfg<128>::kPieces; }

int cache8_pair_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_cache8_pair_status, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int cache8_pair_clear_status() {
  const int z = 0;
  return cudaMemcpyToSymbol(g_cache8_pair_status, &z, sizeof(int)) == cudaSuccess ? 0 : -1;
}

}  // namespace fa
