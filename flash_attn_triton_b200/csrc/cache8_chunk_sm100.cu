// Chunks of tokens against the 8-bit KV cache on the 5th-generation tensor cores: one tile of 128 query rows (query heads of a KV head
// packed into its rows) per CTA, two softmax warpgroups that take its key tiles in turn.  The pipeline of fwd_alt_sm100.cu; what differs:
//
//   warps 0-3, 4-7   softmax groups; before their first tile they bring Q (rotated) into shared memory as fp16
//   warp  8          TMA producer: codes of 128 keys x 128 columns (a unit) into a ring
//   warp  9          MMA issuer
//   warp  10         scales of the tiles' keys into shared memory (11 completes the warpgroup)
//   warps 12-15      converters: a unit of codes to fp16, into the swizzled ring that the MMAs read
//
// Mathematics.  As in cache8_decode.cuh: t_j = scale * ks_j * (q . k8_j), weights 2^(t_j - M) * vs_j rounded to fp16, sums of 2^(t_j - M) in
// fp32.  M is the largest t + log2 |vs| of the keys that the row sees, so no weight is above 2^cfg.rescale_at.  The
// codes are fp16 exactly and the scales stay out of the products: ks multiplies the scores, vs the probabilities, in fp32.
// Bound.  Per tile of 128 x 128 scores the tensor pipe has 16 * head_dim / 128 * 64 cycles, the exponentials 1024; a converter thread
// turns 2 x head_dim codes into halves meanwhile.  (With cp.async by the converter threads themselves, asking for a unit took them
// 1050 cycles and the conversion, chunk by chunk, another 1050: 320 us for 4 x 256 tokens behind 1024 to 8192, 32 heads over 8 of 128.)
// Every mbarrier wait is bounded; on timeout the CTA raises a status word, frees its tensor memory and returns.
#include <cmath>
#include <type_traits>

#include "cache8.cuh"
#include "cache8_host.h"
#include "sm100.cuh"

namespace fa {

using namespace sm100;

__device__ int g_cache8_chunk_status = 0;

namespace {

constexpr int kBM = 128;          // query rows of the tile
constexpr int kBN = 128;          // keys per tile
constexpr int kThreads = 512;
constexpr int kMaxStages = 8;
constexpr int kScaleBufs = 4;

template <int D> struct CCfg {
  static constexpr int kUnitCols = D < 128 ? D : 128;
  static constexpr int kUnits = D / kUnitCols;                      // ring units of a K (or V) tile
  static constexpr int kUnitBytes = kBN * kUnitCols * 2;
  static constexpr int kBoxes = kUnitCols / 64;                     // 64-column boxes of a unit
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr int kRaw = D == 256 ? 3 : D == 128 ? 5 : 8;      // units of codes on their way
  static constexpr int kRawBytes = kBN * kUnitCols;
  static constexpr int kChunks = kRawBytes / 16 / 128;              // 16-byte chunks of a unit per converter thread
  static constexpr int kSBuf = D == 256 ? 2 : 3;                    // score buffers
  static constexpr int kOCol = kSBuf * 128;                         // first column of the accumulator
  static constexpr int kQBytes = kBM * D * 2;
  static constexpr int kRawAt = kQBytes + kStages * kUnitBytes;
  static constexpr int kShared = kRawAt + kRaw * kRawBytes;
  static constexpr int kSmemBytes = kShared + 1024 /*align slack*/ + 8192 /*CShared*/;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
  // Pieces of the keys, at most: a merge keeps a weight per piece and row over both rings.
  static constexpr int kPieces = (kShared - kQBytes) / (kBM * (int)sizeof(float));
};

struct CShared {
  uint64_t q_full;
  uint64_t kv_full[kMaxStages];
  uint64_t kv_empty[kMaxStages];
  uint64_t s_full[3];      // [buffer]: scores computed
  uint64_t p_half[3];      // [buffer]: the first 64 keys of P written back (128 arrivals)
  uint64_t p_ready[3];     // [buffer]: P written back (128 arrivals)
  uint64_t o_done[3];      // [buffer]: its P V finished
  uint64_t decided[2];     // [group]: mref settled for the group's tile (128 arrivals)
  uint64_t raw_full[kMaxStages];
  uint64_t raw_empty[kMaxStages];  // (one arrival of each converter warp)
  uint64_t sc_full[kScaleBufs];    // scales of tile j in buffer j % kScaleBufs
  uint64_t sc_empty[kScaleBufs];   // read (128 arrivals of the group)
  uint32_t tmem_base;
  volatile int abort_flag;
  int last;                // split keys: this CTA merges the pieces
  uint32_t qmost[8];
  alignas(16) float mref[kBM];
  float lrun[kBM];         // row sums, up to the tile before the last one each group has settled
  alignas(16) float ks[kScaleBufs][kBN];
  alignas(16) float vs[kScaleBufs][kBN];
  alignas(16) float lv[kScaleBufs][kBN];        // log2 of |vs|, of each key (kFine) or of 16
};
static_assert(sizeof(CShared) <= 8192, "CShared must fit its reserve");

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, CShared* sh, int code) {
  return bounded_wait(bar, parity, &sh->abort_flag, &g_cache8_chunk_status, code);
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

// T: type of q and o.  kAlibi: with slopes.  kFine: a scale for each key of a tile; else every 16 keys have one scale (blocks of a multiple of
// 16 tokens, no left padding), which goes into the exponent's FMA and stays in registers.  With one per key, read from shared memory by every
// thread, a call of 4 x 256 tokens behind 1024 to 8192, 32 heads over 8 of 128, takes 250 us and 195 with one per 16; heads of 256: 404, 356.
template <typename T, int kCode, int D, bool kAlibi, bool kFine>
__global__ void __launch_bounds__(kThreads, 1)
cache8_chunk_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmO, const fa_decode_args p, const fa_cache8 c8, const int block_shift,
                    const ScoreCfg cfg, const CacheGeo geo, int* const host_status) {
  using C = CCfg<D>;
  using K8 = Code<kCode>;
  constexpr int S = C::kStages, NB = C::kSBuf, NU = C::kUnits;
  constexpr bool kPvSplit = !kAlibi;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  CShared* sh = reinterpret_cast<CShared*>(tiles + C::kShared);
  const uint32_t sQ = smem_u32(tiles);
  const uint32_t sKV = sQ + C::kQBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // behind the append and the checks (a programmatic launch)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (geo.bad && *geo.bad) return;

  // ---- what this CTA works on --------------------------------------------------------------
  Tile w;
  {
    const int heads = p.heads_q >> geo.pack_log2;        // units of heads per sequence
    w.rows = geo.tokens << geo.pack_log2;
    const int mtiles = (w.rows + kBM - 1) / kBM;
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
    w.m0 = mt * kBM;
    const int cap = seq_capacity(p, w.b), len = max(0, min(geo.seqlens[w.b], cap)) + geo.n_new;
    w.keys = min(len, cap);
    w.pos0 = len - geo.tokens;
    w.pad = geo.leftpad ? max(0, geo.leftpad[w.b]) : 0;
  }
  const int tq_min = w.pos0 + (w.m0 >> geo.pack_log2);
  const int tq_max = w.pos0 + ((min(w.m0 + kBM, w.rows) - 1) >> geo.pack_log2);
  const int tq_end = w.pos0 + ((w.m0 + kBM - 1) >> geo.pack_log2);     // of the tile's last row, existing or not
  {
    int klo, khi;
    visible_key_range(cfg, tq_min, tq_max, w.keys, klo, khi);
    const int lo = klo / kBN, hi = (khi + kBN - 1) / kBN;
    const int all = khi > klo ? hi - lo : 0;
    w.parts = chunk_pieces(p, cfg, geo, (p.heads_q >> geo.pack_log2) * ((w.rows + kBM - 1) / kBM), all, lane);
    if (w.part >= w.parts) return;
    const int first = (int)((int64_t)w.part * all / w.parts), last = (int)((int64_t)(w.part + 1) * all / w.parts);
    w.n_hi = lo + last;
    w.nt = last - first;
  }
  const int nt = w.nt;

  if (tid == 0) {
    mbar_init(smem_u32(&sh->q_full), 256);
    for (int i = 0; i < NB; ++i) {
      mbar_init(smem_u32(&sh->s_full[i]), 1);
      mbar_init(smem_u32(&sh->o_done[i]), 1);
      mbar_init(smem_u32(&sh->p_half[i]), 128);
      mbar_init(smem_u32(&sh->p_ready[i]), 128);
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(&sh->kv_full[i]), 4);
      mbar_init(smem_u32(&sh->kv_empty[i]), 1);
    }
    for (int i = 0; i < kScaleBufs; ++i) {
      mbar_init(smem_u32(&sh->sc_full[i]), 1);
      mbar_init(smem_u32(&sh->sc_empty[i]), 128);
    }
    for (int i = 0; i < C::kRaw; ++i) {
      mbar_init(smem_u32(&sh->raw_full[i]), 1);
      mbar_init(smem_u32(&sh->raw_empty[i]), 4);
    }
    mbar_init(smem_u32(&sh->decided[0]), 128);
    mbar_init(smem_u32(&sh->decided[1]), 128);
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

  // Order of use of the units: K_0 .. K_(NB-1), then V_j, K_(j+NB).
  struct Unit {
    int tile, un;                                        // of the CTA's tiles
    bool value;
  };
  const int total = 2 * nt * NU, head = (nt < NB ? nt : NB) * NU, mid = head + (nt > NB ? nt - NB : 0) * 2 * NU;
  auto unit_of = [&](int n) {
    Unit x;
    if (n < head) {
      x.value = false;
      x.tile = n / NU;
      x.un = n % NU;
    } else if (n < mid) {
      const int r = (n - head) % (2 * NU), j = (n - head) / (2 * NU);
      x.value = r < NU;
      x.tile = x.value ? j : j + NB;
      x.un = r % NU;
    } else {
      x.value = true;
      x.tile = (mid - head) / (2 * NU) + (n - mid) / NU;
      x.un = (n - mid) % NU;
    }
    return x;
  };
  const uint32_t raw0 = sQ + C::kRawAt;

  if (warp >= 12) {
    // ------------------------------- converters -----------------------------------------
    reg_dealloc<88>();
    const int ct = tid - 384;
    constexpr int CPR = C::kUnitCols / 16;               // 16-byte chunks of a row
    // This thread's chunk i of a unit: row first + i * kStep, column col.  Lanes of the two 64-column boxes of a row take the halves of
    // a chunk in opposite order: other banks.
    constexpr int kStep = 128 / CPR;
    const int first = ct / CPR, col = (ct % CPR) * 16;
    const uint32_t turn = (uint32_t)(col >> 6) & 1u;
    const uint32_t put = (uint32_t)(col >> 6) * (kBN * 128) + (uint32_t)first * 128;
    const uint32_t put0 = put + (((((uint32_t)col >> 3) & 7u) + turn) ^ (first & 7)) * 16;
    const uint32_t put1 = put + (((((uint32_t)col >> 3) & 7u) + (turn ^ 1u)) ^ (first & 7)) * 16;
    int stage = 0, slot = 0;
    uint32_t phase = 0, sphase = 0;
    bool ok = true;
    for (int n = 0; n < total && ok; ++n) {
      ok = wait_bar(&sh->raw_full[slot], sphase, sh, 13);
      if (!ok) break;
      const uint32_t from = raw0 + slot * C::kRawBytes + ct * 16;
      uint2 u[C::kChunks], v[C::kChunks];
#pragma unroll
      for (int i = 0; i < C::kChunks; ++i) {
        u[i] = ld_shared_v2(from + i * 2048 + turn * 8);
        v[i] = ld_shared_v2(from + i * 2048 + (turn ^ 1u) * 8);
      }
      const int left = w.keys - (w.n_hi - 1 - unit_of(n).tile) * kBN;
      if (left < kBN) {                                  // rows past the last key hold anything: zeros
#pragma unroll
        for (int i = 0; i < C::kChunks; ++i)
          if (first + i * kStep >= left) u[i] = v[i] = make_uint2(0u, 0u);
      }
      ok = wait_bar(&sh->kv_empty[stage], phase ^ 1, sh, 11);
      if (!ok) break;
      const uint32_t dst = sKV + stage * C::kUnitBytes;
#pragma unroll
      for (int i = 0; i < C::kChunks; ++i) {
        uint4 a, b;
        K8::integers(u[i].x, a.x, a.y);
        K8::integers(u[i].y, a.z, a.w);
        K8::integers(v[i].x, b.x, b.y);
        K8::integers(v[i].y, b.z, b.w);
        st_shared_v4(dst + put0 + i * (kStep * 128), a);
        st_shared_v4(dst + put1 + i * (kStep * 128), b);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&sh->raw_empty[slot]));
        mbar_arrive(smem_u32(&sh->kv_full[stage]));
      }
      if (++stage == S) { stage = 0; phase ^= 1; }
      if (++slot == C::kRaw) { slot = 0; sphase ^= 1; }
    }
  } else if (warp >= 8) {
    reg_dealloc<56>();
    auto page_index = [&](int key) { return divided(key, geo.page_size, geo.page_log2); };
    if (warp == 8 && nt > 0) {
      // ------------------------------- TMA producer ---------------------------------------
      // A unit is boxes of geo.box_rows keys that lie inside one page each; lane i brings box i.  Boxes that start past the last key
      // are left out.  Pages are read one unit ahead of their use.
      const int box_log2 = 31 - __clz(geo.box_rows);
      auto page_of = [&](int n) {
        int pg = geo.batch_idx ? geo.batch_idx[w.b] : w.b;
        if (geo.table) {
          const int key = n < total ? (w.n_hi - 1 - unit_of(n).tile) * kBN + (lane << box_log2) : w.keys;
          pg = lane < (kBN >> box_log2) && key < w.keys ? geo.table[(int64_t)w.b * geo.table_stride + page_index(key)] : 0;
        }
        return pg;
      };
      int slot = 0, pg = page_of(0);
      uint32_t sphase = 0;
      bool ok = true;
      int n = 0;
      for (; n < total; ++n) {
        const Unit x = unit_of(n);
        const int k0 = (w.n_hi - 1 - x.tile) * kBN, key = k0 + (lane << box_log2);
        const int row = geo.table ? key - page_index(key) * geo.page_size : key + w.pad;
        const int boxes = min(kBN >> box_log2, ((w.keys - k0 - 1) >> box_log2) + 1);
        const uint32_t bar = smem_u32(&sh->raw_full[slot]), dst = raw0 + slot * C::kRawBytes;
        if (lane == 0) ok = wait_bar(&sh->raw_empty[slot], sphase ^ 1, sh, 12);
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(bar, boxes * (C::kUnitCols << box_log2));
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(dst + (lane << box_log2) * C::kUnitCols, x.value ? &tmV : &tmK, bar, x.un * C::kUnitCols, w.hk, row, pg);
        pg = page_of(n + 1);
        if (++slot == C::kRaw) { slot = 0; sphase ^= 1; }
      }
      // a CTA that gives up still waits for the copies that are on their way to it
      if (!ok)
        for (int m = max(0, n - C::kRaw); m < n; ++m)
          for (int i = 0; i < 1 << 16 && !mbar_try_wait(smem_u32(&sh->raw_full[m % C::kRaw]), (m / C::kRaw) & 1); ++i) {}
    } else if (warp == 10 && nt > 0) {
      // ------------------------------- scales -----------------------------------------------
      // Lane i has keys 4 i to 4 i + 3 of a tile (of one page).  Pages are read two tiles ahead, scales one.
      const float* ksbase = c8.k_scale + (int64_t)w.hk * c8.ks_stride[2];
      const float* vsbase = c8.v_scale + (int64_t)w.hk * c8.vs_stride[2];
      auto page_of = [&](int j) {
        const int key = (w.n_hi - 1 - j) * kBN + lane * 4;
        if (geo.table == nullptr) return geo.batch_idx ? geo.batch_idx[w.b] : w.b;
        return j < nt && key < w.keys ? geo.table[(int64_t)w.b * geo.table_stride + page_index(key)] : 0;
      };
      float ks[4], vs[4];
      auto scales_of = [&](int j, int pg) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = (w.n_hi - 1 - j) * kBN + lane * 4 + i;
          ks[i] = vs[i] = 0.f;
          if (j < nt && key < w.keys) {
            const int row = geo.table ? key - page_index(key) * geo.page_size : key + w.pad, blk = divided(row, c8.block, block_shift);
            ks[i] = ksbase[pg * c8.ks_stride[0] + blk * c8.ks_stride[1]];
            vs[i] = vsbase[pg * c8.vs_stride[0] + blk * c8.vs_stride[1]];
          }
        }
      };
      int pg = page_of(0);
      scales_of(0, pg);
      pg = page_of(1);
      for (int j = 0; j < nt; ++j) {
        // A scale of V that is no number or infinite goes to the scores instead, which the mask takes out where the key is hidden
        // (0 times either would not be 0).
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(fabsf(vs[i]) <= 3.4e38f)) {
            ks[i] = NAN;
            vs[i] = 0.f;
          }
        const float4 k4 = make_float4(ks[0], ks[1], ks[2], ks[3]), v4 = make_float4(vs[0], vs[1], vs[2], vs[3]);
        scales_of(j + 1, pg);
        pg = page_of(j + 2);
        const int sb = j % kScaleBufs;
        if (!wait_bar(&sh->sc_empty[sb], ((j / kScaleBufs) & 1) ^ 1, sh, 14)) break;
        if (kFine) {
          *reinterpret_cast<float4*>(&sh->ks[sb][lane * 4]) = k4;
          *reinterpret_cast<float4*>(&sh->vs[sb][lane * 4]) = v4;
          auto log2_of_scale = [](float v) { return __log2f(fmaxf(fabsf(v), 0x1p-60f)); };
          *reinterpret_cast<float4*>(&sh->lv[sb][lane * 4]) =
              make_float4(log2_of_scale(v4.x), log2_of_scale(v4.y), log2_of_scale(v4.z), log2_of_scale(v4.w));
        } else if ((lane & 3) == 0) {
          sh->ks[sb][lane >> 2] = k4.x;
          sh->vs[sb][lane >> 2] = v4.x;
          sh->lv[sb][lane >> 2] = __log2f(fmaxf(fabsf(v4.x), 0x1p-60f));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->sc_full[sb]));
      }
    } else if (warp == 9 && nt > 0) {
      // ------------------------------- MMA issuer -------------------------------------------
      // The whole warp runs the control flow in lock step and every lane polls the barriers;
      // the lane chosen once by elect_one issues the MMAs and commits.
      constexpr uint32_t idesc_qk = make_idesc(1, 0, 0, 0, kBM, kBN);
      constexpr uint32_t idesc_pv = make_idesc(1, 0, 0, 1, kBM, C::kUnitCols);
      const uint32_t leader = elect_one() ? 1u : 0u;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      auto wwait = [&](uint64_t* bar, uint32_t parity, int code) {
        if (ok) ok = wait_bar(bar, parity, sh, code);
        tc_fence_after();
      };
      auto advance = [&]() { if (++stage == S) { stage = 0; phase ^= 1; } };
      auto issue_qk = [&](int buf) {                       // S[buf] = Q K^T with the next K tile of the ring
#pragma unroll
        for (int un = 0; un < NU; ++un) {
          wwait(&sh->kv_full[stage], phase, 22);
          if (!ok) return;
          const uint64_t dq = make_smem_desc(sQ + un * (C::kUnitCols / 64) * (kBM * 128), 16, 1024);
          const uint64_t dk = make_smem_desc(sKV + stage * C::kUnitBytes, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < C::kUnitCols / 16; ++kk) {
            const uint32_t o = ((kk / 4) * (kBM * 128) + (kk % 4) * 32) >> 4;
            mma_f16_ss_lp(tmem + buf * kBN, dq + o, dk + o, idesc_qk, (un > 0 || kk > 0) ? 1u : 0u, leader);
          }
          mma_commit_lp(smem_u32(&sh->kv_empty[stage]), leader);
          advance();
        }
        mma_commit_lp(smem_u32(&sh->s_full[buf]), leader);
      };
      wwait(&sh->q_full, 0, 21);
      for (int i = 0; i < NB && i < nt && ok; ++i) issue_qk(i);
      int buf = 0;
      uint32_t par = 0;                                    // (j / NB) & 1
      for (int j = 0; j < nt && ok; ++j) {
        const uint32_t a = tmem + buf * kBN;
        // the V units of tile j are in the next NU stages
        int st[NU];
#pragma unroll
        for (int un = 0; un < NU; ++un) {
          wwait(&sh->kv_full[stage], phase, 24);
          st[un] = stage;
          advance();
        }
        if (!ok) break;
        if (kPvSplit) {
          wwait(&sh->p_half[buf], par, 25);
          if (!ok) break;
#pragma unroll
          for (int un = 0; un < NU; ++un) {
            const uint64_t dv = make_smem_desc(sKV + st[un] * C::kUnitBytes, kBN * 128, 1024);
#pragma unroll
            for (int kk = 0; kk < kBN / 32; ++kk)
              mma_f16_ts_lp(tmem + C::kOCol + un * C::kUnitCols, a + kk * 8, dv + ((kk * 2048) >> 4), idesc_pv,
                            (j > 0 || kk > 0) ? 1u : 0u, leader);
          }
        }
        wwait(&sh->p_ready[buf], par, 26);
        if (!ok) break;
#pragma unroll
        for (int un = 0; un < NU; ++un) {
          const uint64_t dv = make_smem_desc(sKV + st[un] * C::kUnitBytes, kBN * 128, 1024);
#pragma unroll
          for (int kk = kPvSplit ? kBN / 32 : 0; kk < kBN / 16; ++kk)
            mma_f16_ts_lp(tmem + C::kOCol + un * C::kUnitCols, a + kk * 8, dv + ((kk * 2048) >> 4), idesc_pv,
                          (j > 0 || kk > 0) ? 1u : 0u, leader);
          mma_commit_lp(smem_u32(&sh->kv_empty[st[un]]), leader);
        }
        mma_commit_lp(smem_u32(&sh->o_done[buf]), leader);
        if (j + NB < nt) issue_qk(buf);
        if (++buf == NB) { buf = 0; par ^= 1; }
      }
    }
  } else {
    // ------------------------------- softmax groups -------------------------------------
    reg_alloc<184>();
    // ---- Q: rotated, to fp16 (bf16: times the power of two that brings the largest element of the tile to [2^14, 2^15)), swizzled
    float qinv = 1.f;
    {
      constexpr int QC = D / 8, NQ = kBM * QC / 256, kAtOnce = NQ < 16 ? NQ : 16;
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
        st_shared_v4(sw128_addr(sQ + (c >> 3) * (kBM * 128), r, c & 7), v);
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
    const int x = warp >> 2;                         // group
    const int row_in_tile = (warp & 3) * 32 + lane;  // TMEM lane
    const int row = w.m0 + row_in_tile;
    const int qpos = w.pos0 + (row >> geo.pack_log2);
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_addr + C::kOCol;
    float slope = 0.f;
    if (kAlibi && row < w.rows) slope = p.alibi_slopes[w.b * p.heads_q + w.h + (row & ((1 << geo.pack_log2) - 1))];
    // of this group's latest tile: the factor its maximum asked of what came before, and its row sum
    float alpha = 1.f, sum = 0.f;
    bool ok = true;

    for (int j = x; j < nt && ok; j += 2) {
      const int buf = j % NB;
      const uint32_t par = (j / NB) & 1;
      const uint32_t tS = tmem + lane_addr + buf * kBN;
      const int k0 = (w.n_hi - 1 - j) * kBN;
      bool masked = (k0 + kBN > w.keys);
      if (cfg.causal) masked |= (k0 + kBN - 1 > tq_min);
      if (cfg.wl >= 0) masked |= (k0 < tq_end - cfg.wl);
      if (cfg.wr >= 0) masked |= (k0 + kBN - 1 > tq_min + cfg.wr);

      const int sb = j % kScaleBufs;
      ok = wait_bar(&sh->sc_full[sb], (j / kScaleBufs) & 1, sh, 29);
      if (!kFine) {                                      // a negative scale of K, see below
        const float4 a = *reinterpret_cast<const float4*>(&sh->ks[sb][0]), b = *reinterpret_cast<const float4*>(&sh->ks[sb][4]);
        masked |= fminf(fminf(fminf(a.x, a.y), fminf(a.z, a.w)), fminf(fminf(b.x, b.y), fminf(b.z, b.w))) < 0.f;
      }
      ok = ok && wait_bar(&sh->s_full[buf], par, sh, 31 + x);
      if (!ok) break;
      tc_fence_after();

      // ---- scores times the scales of the keys: mg of each 16 keys turns them into the log2 domain.  Tiles with a mask, with ALiBi or with
      // a scale per key go there at once, through tensor memory in a rolled loop: copies of the passes below for them cost the code that every
      // tile runs 14 % (instruction cache).  With a scale per key the maximum is taken there too, over the keys that the row sees: a key
      // that it does not see, or sees with a low score, may have a scale of V far above theirs.  So do tiles with a negative scale of K, whose
      // largest score has the smallest product.
      const bool masked_or_fine = kAlibi || kFine || masked;
      const float f = cfg.scale_log2 * qinv;
      float mx = -INFINITY;                              // row maximum of t + log2 |vs|
      if (masked_or_fine) {
        int vk_lo, vk_hi;
        visible_k_interval(cfg, qpos, w.keys, vk_lo, vk_hi);
        const float tilt = slope * FA_LOG2E;
#pragma unroll 1
        for (int cc = 0; cc < 4; ++cc) {
          const ColMask cm = make_col_mask(vk_lo - k0 - cc * 32, vk_hi - k0 - cc * 32);
          const float2 k2 = *reinterpret_cast<const float2*>(&sh->ks[sb][kFine ? 0 : cc * 2]);
          const float dist0 = (float)(qpos - k0 - cc * 32);
          uint32_t ra[32];
          tmem_ld32(tS + cc * 32, ra);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float v = __uint_as_float(ra[i]) * (kFine ? sh->ks[sb][cc * 32 + i] : i < 16 ? k2.x : k2.y) * f;
            if (kAlibi) v = fmaf(-tilt, fabsf(dist0 - (float)i), v);
            v = col_visible(cm, i) ? v : -INFINITY;
            ra[i] = __float_as_uint(v);
            if (kFine) mx = fmaxf(mx, v + sh->lv[sb][cc * 32 + i]);
          }
          tmem_st32(tS + cc * 32, ra);
        }
        tmem_wait_st();
      }
      auto factors = [&](int cc) {
        return masked_or_fine ? make_float2(1.f, 1.f) : f2mul(*reinterpret_cast<const float2*>(&sh->ks[sb][cc * 2]), make_float2(f, f));
      };

      // ---- row maximum, vs and mg by 16 keys ------------------------------------------------------
      // The scores are read twice, 32 columns at a time: for the maximum, and for the exponentials (P of columns cc overwrites columns that
      // have been read).  All 128 of a row do not fit beside the rest in what 512 threads have: 512 bytes of them were spilled, and a
      // tile's exponentials took 4200 cycles.
      if (!kFine) {
        uint32_t ra[32], rb[32];
        tmem_ld32(tS, ra);
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t (&cur)[32] = (cc & 1) ? rb : ra;
          uint32_t (&nxt)[32] = (cc & 1) ? ra : rb;
          tmem_wait_ld();
          if (cc < 3) tmem_ld32(tS + (cc + 1) * 32, nxt);
          const float2 mg = factors(cc), lv = *reinterpret_cast<const float2*>(&sh->lv[sb][cc * 2]);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const uint32_t* v = &cur[g * 16];
            float m[5];
#pragma unroll
            for (int i = 0; i < 5; ++i)
              m[i] = fmax3(__uint_as_float(v[3 * i]), __uint_as_float(v[3 * i + 1]), __uint_as_float(v[3 * i + 2]));
            const float most = fmaxf(fmax3(m[0], m[1], m[2]), fmax3(m[3], m[4], __uint_as_float(v[15])));
            mx = fmaxf(mx, fmaf(most, g ? mg.y : mg.x, g ? lv.y : lv.x));
          }
        }
      }

      // ---- the maximum the exponents are relative to, settled in tile order ---------------
      float m_use;
      if (j == 0) {
        m_use = mx;
        sh->mref[row_in_tile] = mx;
        sh->lrun[row_in_tile] = 0.f;
      } else {
        ok = wait_bar(&sh->decided[x ^ 1], ((j - 1) >> 1) & 1, sh, 33 + x);
        if (!ok) break;
        const float m_old = sh->mref[row_in_tile];
        if (j >= 2) sh->lrun[row_in_tile] = __fadd_rn(__fmul_rn(sh->lrun[row_in_tile], alpha), sum);
        const bool need = mx > m_old + cfg.rescale_at;
        m_use = need ? mx : m_old;
        alpha = 1.f;
        if (__any_sync(0xffffffffu, need)) {
          // The accumulator may be touched once P V of the tile before is finished: the one of this
          // tile cannot start before P is written below.
          const int pb = (j - 1) % NB;
          ok = wait_bar(&sh->o_done[pb], ((j - 1) / NB) & 1, sh, 35 + x);
          if (!ok) break;
          tc_fence_after();
          if (need) alpha = exp2f(m_old - mx);
          if (need) sh->mref[row_in_tile] = mx;
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
      }
      mbar_arrive(smem_u32(&sh->decided[x]));
      const float m_safe = (m_use == -INFINITY) ? 0.f : m_use;

      // ---- p = exp2(t - M), row sum, p vs -> TMEM in place over S ----------------------------
      const float2 nm2 = make_float2(-m_safe, -m_safe);
      float2 acc2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      {
        uint32_t ra[32], rb[32];
        tmem_ld32(tS, ra);
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t (&cur)[32] = (cc & 1) ? rb : ra;
          uint32_t (&nxt)[32] = (cc & 1) ? ra : rb;
          tmem_wait_ld();
          if (cc < 3) tmem_ld32(tS + (cc + 1) * 32, nxt);
          const float2 mg = factors(cc);
          float2 v16 = make_float2(0.f, 0.f);            // scales of V of the two 16 keys
          if (!kFine) v16 = *reinterpret_cast<const float2*>(&sh->vs[sb][cc * 2]);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float4 v4;
            if (kFine) v4 = *reinterpret_cast<const float4*>(&sh->vs[sb][cc * 32 + i]);
            else v4.x = v4.y = v4.z = v4.w = i < 16 ? v16.x : v16.y;
            const float2 mul2 = i < 16 ? make_float2(mg.x, mg.x) : make_float2(mg.y, mg.y);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float2 a = f2fma(make_float2(__uint_as_float(cur[i + e]), __uint_as_float(cur[i + e + 1])), mul2, nm2);
              const float2 pe = make_float2(ex2(a.x), ex2(a.y));
              acc2[e >> 1] = f2add(acc2[e >> 1], pe);
              const float2 wt = f2mul(pe, e ? make_float2(v4.z, v4.w) : make_float2(v4.x, v4.y));
              pk[(i + e) >> 1] = Elem<__half>::pack(wt.x, wt.y);
            }
          }
          tmem_st16(tS + cc * 16, pk);
          if (kPvSplit && cc == 1) {
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_u32(&sh->p_half[buf]));
          }
        }
      }
      sum = (acc2[0].x + acc2[0].y) + (acc2[1].x + acc2[1].y);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(smem_u32(&sh->p_ready[buf]));
      mbar_arrive(smem_u32(&sh->sc_empty[sb]));
    }

    // ---- epilogue: both groups, half of the columns each ----------------------------------
    asm volatile("bar.sync 1, 256;\n" ::: "memory");     // every decision is made
    const float m_fin = nt > 0 ? sh->mref[row_in_tile] : -INFINITY;
    // the row sum: the tile before the last, then the last
    const bool last_group = ((nt - 1) & 1) == x;
    if (nt > 0 && !last_group) sh->lrun[row_in_tile] = __fadd_rn(__fmul_rn(sh->lrun[row_in_tile], alpha), sum);
    if (ok && nt > 0) ok = wait_bar(&sh->o_done[(nt - 1) % NB], ((nt - 1) / NB) & 1, sh, 37 + x);
    const bool failed = any_of_256(!ok || sh->abort_flag != 0);
    tc_fence_after();
    float l_all = 0.f;
    if (nt > 0) {
      if (last_group) sh->lrun[row_in_tile] = __fadd_rn(__fmul_rn(sh->lrun[row_in_tile], alpha), sum);
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      l_all = sh->lrun[row_in_tile];
    }
    if (!failed) {
      const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
      const float lse = l_all == 0.f ? -INFINITY : m_fin + log2f(l_all);
      const bool row_ok = row < w.rows;
      const bool piece = w.parts > 1;
      const int64_t slot = blockIdx.x;
#pragma unroll
      for (int c2 = 0; c2 < D / 64; ++c2) {
        const int cc = x * (D / 64) + c2;                // 32 columns
        uint32_t ra[32];
        if (nt > 0) {
          tmem_ld32(tO + cc * 32, ra);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) ra[i] = 0u;
        }
        if (piece) {
          float* dst = geo.ws + (slot * kBM + row_in_tile) * D + cc * 32;
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
            st_shared_v4(sw128_addr(sQ + (col / 64) * (kBM * 128), row_in_tile, (col % 64) / 8), v);
          }
        }
      }
      if (!piece) {
        // staged over the Q tile, which no MMA reads any more
        fence_proxy_async();
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        if (tid == 0) {
#pragma unroll
          for (int bx = 0; bx < D / 64; ++bx)
            tma_store_4d(&tmO, sQ + bx * (kBM * 128), bx * 64, w.h, w.m0 >> geo.pack_log2, w.b);
          tma_store_commit();
          tma_store_wait_read();
        }
      }
      if (piece) {
        // the CTA that finishes last merges; pieces are ordered before the count by the fence of each writer
        float* ws_l = geo.ws + (int64_t)gridDim.x * kBM * D;
        if (x == 0 && row_ok) ws_l[slot * kBM + row_in_tile] = lse;
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
          const int64_t s0 = (int64_t)(blockIdx.x / geo.parts) * geo.parts;
          const int rows = min(kBM, w.rows - w.m0);
          // weights of the pieces per row, over the rings (every K/V tile has been read); w.parts <= geo.parts <= C::kPieces
          float* wt = reinterpret_cast<float*>(tiles + C::kQBytes);
          if (tid < rows) {
            float m = -INFINITY, sum = 0.f;
            for (int s = 0; s < w.parts; ++s) m = fmaxf(m, ws_l[(s0 + s) * kBM + tid]);
            for (int s = 0; s < w.parts; ++s) {
              const float v = m == -INFINITY ? 0.f : exp2f(ws_l[(s0 + s) * kBM + tid] - m);
              wt[s * kBM + tid] = v;
              sum += v;
            }
            const float f = sum > 0.f ? 1.f / sum : 0.f;
            for (int s = 0; s < w.parts; ++s) wt[s * kBM + tid] *= f;
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
                const float4 v = *reinterpret_cast<const float4*>(geo.ws + ((s0 + s) * kBM + r) * D + d);
                const float f = wt[s * kBM + r];
                acc[k].x += f * v.x; acc[k].y += f * v.y; acc[k].z += f * v.z; acc[k].w += f * v.w;
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
template <typename T, int kCode, int D, bool kAlibi, bool kFine>
static int launch_chunk8(const fa_decode_args& d, const fa_cache8& c, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st) {
  if (geo.parts > CCfg<D>::kPieces) {
    set_error("cache8_chunk: %d pieces, %d at most", geo.parts, CCfg<D>::kPieces);
    return FA_ERR_LAUNCH;
  }
  const int pack = 1 << geo.pack_log2;
  CUtensorMap tm[3];
  // codes as they lie, no swizzle: their readers are threads
  auto codes = [&](CUtensorMap* m, const void* base, const int64_t* stride) {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)d.heads_kv, (uint64_t)d.page_size, (uint64_t)d.num_pages};
    const uint64_t strides[3] = {(uint64_t)stride[2], (uint64_t)stride[1], (uint64_t)stride[0]};
    const uint32_t box[4] = {(uint32_t)CCfg<D>::kUnitCols, 1, (uint32_t)geo.box_rows, 1};
    return encode_tmap(m, base, 1, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
  };
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)d.heads_q, (uint64_t)d.seqlen_q, (uint64_t)d.batch};
  const uint64_t strides[3] = {(uint64_t)d.o_stride[2] * 2, (uint64_t)d.o_stride[1] * 2, (uint64_t)d.o_stride[0] * 2};
  const uint32_t box[4] = {64, (uint32_t)pack, (uint32_t)(kBM / pack), 1};
  if (!codes(&tm[0], d.k_cache, d.kc_stride) || !codes(&tm[1], d.v_cache, d.vc_stride) || !encode_tmap(&tm[2], d.o, 2, 4, dims, strides, box)) {
    set_error("cache8_chunk: cuTensorMapEncodeTiled failed");
    return FA_ERR_LAUNCH;
  }
  auto kern = cache8_chunk_kernel<T, kCode, D, kAlibi, kFine>;
  constexpr int smem = CCfg<D>::kSmemBytes;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    set_error("cache8_chunk: cudaFuncSetAttribute(%d): %s", smem, cudaGetErrorString(e));
    return FA_ERR_LAUNCH;
  }
  const int mtiles = (d.seqlen_q * pack + kBM - 1) / kBM;
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
  return check_launch("cache8_chunk");
}

template <typename T, int kCode, int D>
static int launch_chunk8_dim(const fa_decode_args& d, const fa_cache8& c, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st) {
  // (with ALiBi, which is rare, there is the general kernel alone)
  if (cfg.has_alibi) return launch_chunk8<T, kCode, D, true, true>(d, c, geo, cfg, st);
  return c.block % 16 != 0 || geo.leftpad != nullptr ? launch_chunk8<T, kCode, D, false, true>(d, c, geo, cfg, st)
                                                     : launch_chunk8<T, kCode, D, false, false>(d, c, geo, cfg, st);
}
template <typename T, int kCode>
static int launch_chunk8_code(const fa_decode_args& d, const fa_cache8& c, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st) {
  switch (d.head_dim) {
    case 64: return launch_chunk8_dim<T, kCode, 64>(d, c, geo, cfg, st);
    case 128: return launch_chunk8_dim<T, kCode, 128>(d, c, geo, cfg, st);
    case 256: return launch_chunk8_dim<T, kCode, 256>(d, c, geo, cfg, st);
  }
  set_error("cache8_chunk: head_dim %d", d.head_dim);
  return FA_ERR_UNSUPPORTED;
}

int cache8_chunk(const fa_decode_args& d, const fa_cache8& c, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st) {
  if (d.dtype == FA_BF16)
    return c.code == FA_CODE_INT8 ? launch_chunk8_code<__nv_bfloat16, FA_CODE_INT8>(d, c, geo, cfg, st)
                                  : launch_chunk8_code<__nv_bfloat16, FA_CODE_E4M3>(d, c, geo, cfg, st);
  return c.code == FA_CODE_INT8 ? launch_chunk8_code<__half, FA_CODE_INT8>(d, c, geo, cfg, st)
                                : launch_chunk8_code<__half, FA_CODE_E4M3>(d, c, geo, cfg, st);
}

int cache8_chunk_pieces(int head_dim) {
  return head_dim == 64 ? CCfg<64>::kPieces : head_dim == 128 ? CCfg<128>::kPieces : CCfg<256>::kPieces;
}

int cache8_chunk_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_cache8_chunk_status, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int cache8_chunk_clear_status() {
  const int z = 0;
  return cudaMemcpyToSymbol(g_cache8_chunk_status, &z, sizeof(int)) == cudaSuccess ? 0 : -1;
}

}  // namespace fa
