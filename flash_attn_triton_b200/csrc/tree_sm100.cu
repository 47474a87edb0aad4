// Attention of a tree of drafted tokens to a KV cache, on the 5th-generation tensor cores: more than 8 query rows per KV head.
//
//   Work.  A unit is (KV head, tile of 128 query rows) of a sequence; the query heads of a KV head are packed into the rows of a tile (row =
//   node * group + head).  Every unit streams the sequence's keys once, 128 at a time, and at these few rows the memory sets the pace:
//   4 D bytes a key and head against 2 x 2 x 128 x D products.
//   Equal shares.  The sequences' tiles of keys, one sequence after another, are cut into as many equal ranges as there are groups of CTAs; a
//   CTA does one range for one unit of heads, whatever sequences it covers (a segment each), and the CTAs of a group walk the same pages at
//   the same time.  With a CTA per unit and a fixed number of pieces of each sequence, 32 sequences of 1024 to 16384 tokens took as
//   long as the longest, and 96 units kept a third of the SMs idle.  The lengths are on the device, so every warp works out its ranges.
//   One pipeline through all segments: the producer and the MMA issuer run ahead into the next segment (the queries have a buffer per
//   segment where they fit) while the softmax groups finish the one before.
//   Pieces of a sequence that is cut go to the workspace; a small kernel behind this one, launched early, adds them up, always in the same
//   order.  The CTA that finishes last did it at first: 18 pieces of 64 rows took it some 40 us, in 24 round trips to memory.
//
//   warps 0-7   softmax pair 0  : every other tile of keys, warps 0-3 its first 64 keys, warps 4-7 the other 64
//   warps 8-15  softmax pair 1  : the other tiles
//   two warps   TMA producer    : Q of a segment, K/V through a ring of 128-key x 128-column entries
//               MMA issuer      : S[j] = Q K_j^T (SS);  O += P_j V_j (A = P_j from tensor memory)
//   two warps   results of a segment, up to 64 rows and head_dim up to 128 (kApart); else idle (they complete the warpgroup that gives its
//               registers to the softmax warps), and the softmax warps write the results
//
// Tensor memory and the reference of the exponents: as in fwd_alt_sm100.cu.  Here the tiles of all segments are counted through (J), and
// barrier parities follow that count.  kApart has two accumulators (and at head_dim 128 a score buffer less), so that the end of a segment lies under the
// next one's tiles: 16-node trees of 144 sequences of 512 tokens, 32 heads over 8, 82 -> 75 us, at head_dim 64 61 -> 51; 18 of 4096 60 -> 61, 46 -> 41.
// What a tile costs beside its bytes counts twice, for the memory and the SMs together reach the limit of
// the GPU's power, and the clock falls.  18 x 16384 tokens, 64 rows over each of 8 KV heads of 128 (floor 185 us): two groups of four
// softmax warps, a tile each, 254 us, also out of L2; four warps per scheduler 228; P rounded to 16 bits once and not in two parts, as chunks of
// a cache have it, and no work on rows that do not exist 185; 16 rows, softmax for 32 in place of 64, 48 x 500 to 12000 tokens 245 -> 238.  (Errors against float64, relative: fp16 2.1e-4 of two parts, 2.9e-4 of one; bf16 1.6e-3, 2.3e-3.)
#include <type_traits>

#include "cache_geo.cuh"
#include "common.cuh"
#include "sm100.cuh"

namespace fa {

using namespace sm100;

__device__ int g_tree_status = 0;

namespace {

constexpr int kBM = 128;          // query rows of the tile
constexpr int kBN = 128;          // keys per tile
constexpr int kSoftmax = 512;     // threads of the softmax warps
constexpr int kThreads = kSoftmax + 128;
constexpr int kMaxStages = 8;
constexpr int kSharedBytes = 3 * 1024;   // reserve for TShared
constexpr int kMergeAtOnce = 8;   // pieces whose rows are in flight together

// kApart: few rows and head_dim up to 128.  Two warps of their own write the results, from one of two accumulators, so that a segment's end
// lies under the next segment's tiles.
template <int D, bool kApart> struct TCfg {
  static constexpr int kUnitCols = D < 128 ? D : 128;
  static constexpr int kUnits = D / kUnitCols;                      // ring entries of a K (or V) tile
  static constexpr int kUnitBytes = kBN * kUnitCols * 2;
  static constexpr int kBoxes = kUnitCols / 64;                     // TMA boxes of an entry
  static constexpr int kStages = D == 64 ? 8 : 5;
  static constexpr int kQBuf = D == 256 ? 1 : 2;
  static constexpr int kSBuf = D == 256 || (kApart && D == 128) ? 2 : 3;      // score buffers
  static constexpr int kOBuf = kApart ? 2 : 1;                      // accumulators
  static constexpr int kOCol = kSBuf * 128;                         // first column of the accumulator
  static constexpr int kQBytes = kBM * D * 2;
  static constexpr int kRing = kQBuf * kQBytes;                     // where the ring begins
  static constexpr int kSmemTiles = kRing + kStages * kUnitBytes;
  static constexpr int kSmemBytes = kSmemTiles + kSharedBytes;
};

struct TShared {
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[kMaxStages], kv_empty[kMaxStages];
  uint64_t s_full[3];      // [buffer]: scores computed
  // (Barriers that count threads: none may arrive for a phase before the one ahead of it is complete, see fwd_alt_sm100.cu: every tile waits
  // for the decision about the one before, the first of a segment too.)
  uint64_t p_ready[2][3];  // [half][buffer]: P of these warps written back (128 arrivals)
  uint64_t o_done[3];      // [buffer]: its P V finished
  uint64_t decided[2];     // [pair]: mref settled for the pair's tile (256 arrivals)
  uint64_t o_free[2];      // [accumulator]: it has been read, and the sums of its segment (all that read it)
  uint64_t o_last[2];      // [accumulator]: its segment's last P V finished
  uint64_t ended[2];       // [accumulator]: its segment's sums are written (all softmax threads that have rows)
  uint32_t tmem_base;
  volatile int abort_flag;
  alignas(16) float mref[kBM];
  float part[4][kBM];      // [2 pair + half]: row maxima of the two halves of a tile; at the end of a segment row sums
};
static_assert(sizeof(TShared) <= kSharedBytes, "TShared must fit its reserve");

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, TShared* sh, int code) {
  return bounded_wait(bar, parity, &sh->abort_flag, &g_tree_status, code);
}
// The predicate, set in any of the kCount threads that meet at barrier `id`?
template <int kCount> __device__ __forceinline__ bool any_of(bool x, int id) {
  int r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.s32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, %3, %2, p;\n"
      "selp.s32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r) : "r"((int)x), "n"(kCount), "r"(id) : "memory");
  return r != 0;
}
template <int kCount> __device__ __forceinline__ void sync_all() { asm volatile("bar.sync 1, %0;\n" ::"n"(kCount) : "memory"); }
// The two warps that have the halves of the same rows.
__device__ __forceinline__ void sync_halves(int id) { asm volatile("bar.sync %0, 64;\n" ::"r"(id) : "memory"); }

template <typename T> struct TFmt;
template <> struct TFmt<__half> { static constexpr int code = 0; };
template <> struct TFmt<__nv_bfloat16> { static constexpr int code = 1; };

// Nodes [node, node + 32) that a row of the mask sees; those below 0 are the context, which all see.
__device__ __forceinline__ uint32_t seen_of(const uint32_t* bits, int words, int node) {
  const int i = node >> 5;
  auto word = [&](int k) { return k < 0 ? 0xffffffffu : k < words ? bits[k] : 0u; };
  return __funnelshift_r(word(i), word(i + 1), node & 31);
}

// Tiles [first, n_hi) of sequence b; nt of them, walked from the last to the first.
struct Segment {
  int b, k_len, pos0;      // pos0: the root's position
  int first, n_hi, nt, all;
};
// The segments of a range, in order.
struct Walk {
  const int* seqlens;
  int n_new, tokens, capacity;
  int64_t t, end, base;    // next tile, end of the range, first tile of sequence b
  int b;

  __device__ __forceinline__ int len_of(int i) const { return min(max(seqlens[i], 0) + n_new, capacity); }
  __device__ __forceinline__ int tiles_of(int i) const { return max(1, (len_of(i) + kBN - 1) / kBN); }
  __device__ __forceinline__ bool next(Segment& s) {
    if (t >= end) return false;
    s.b = b;
    s.k_len = len_of(b);
    s.pos0 = s.k_len - tokens;
    s.all = max(1, (s.k_len + kBN - 1) / kBN);
    s.first = (int)(t - base);
    s.n_hi = (int)min((int64_t)s.all, end - base);
    s.nt = s.n_hi - s.first;
    t = base + s.n_hi;
    if (s.n_hi == s.all) {
      base += s.all;
      ++b;
    }
    return true;
  }
};

// Ranges that `total` tiles are cut into, `parts` at most: of two tiles at least, and no more than keep a balance between a tile (1.3 us) and
// a piece of a sequence in the merge (0.13 us) -- one sequence of 60000 keys, one unit: 148 ranges 72 us, 117 61.
__device__ __forceinline__ int ranges_of(int64_t total, int batch, int parts) {
  const int64_t most = min((int64_t)parts, min(total / 2, (int64_t)sqrtf(10.f * (float)total * (float)batch)));
  return (int)max((int64_t)1, most);
}

}  // namespace

// geo.parts: ranges that the grid has room for.
// kSplit: 128 / kSplit query rows at most (1, 2 or 4); warps and results of the others are left out.
template <typename T, int D, int kSplit>
__global__ void __launch_bounds__(kThreads, 1)
tree_sm100_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const fa_attn_args p, const float scale_log2, const float rescale_at, const CacheGeo geo, int* const host_status) {
  constexpr bool kApart = kSplit > 1 && D <= 128;
  constexpr int kRows = kBM / kSplit;
  using C = TCfg<D, kApart>;
  constexpr int S = C::kStages, NB = C::kSBuf, NU = C::kUnits, NQ = C::kQBuf, NO = C::kOBuf;
  constexpr int kTmaWarp = kApart ? 18 : 16, kMmaWarp = kTmaWarp + 1;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = smem_raw;                             // (a kernel's dynamic shared memory alone begins at 1024 bytes; checked below)
  TShared* sh = reinterpret_cast<TShared*>(tiles + C::kSmemTiles);
  const uint32_t sQ = smem_u32(tiles), sKV = sQ + C::kRing;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- this CTA's range of tiles and its unit ----------------------------------------------
  const int heads = p.heads_q >> geo.pack_log2;                // units of heads
  const int rows = geo.tokens << geo.pack_log2, mtiles = (rows + kBM - 1) / kBM, U = heads * mtiles;
  const int range = blockIdx.x / U, u = blockIdx.x - range * U;
  const int h = (u / mtiles) << geo.pack_log2, m0 = u % mtiles * kBM;
  const int hk = h / (p.heads_q / p.heads_kv);
  Walk walk;
  int64_t total;
  int ranges;
  {
    walk.seqlens = geo.seqlens;
    walk.n_new = geo.n_new;
    walk.tokens = geo.tokens;
    walk.capacity = geo.capacity;
    // lane i looks after the sequences [i per, (i + 1) per)
    const int per = (p.batch + 31) / 32, b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
    int64_t mine = 0;
    for (int i = b0; i < b1; ++i) mine += walk.tiles_of(i);
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    total = __shfl_sync(0xffffffffu, inc, 31);
    ranges = ranges_of(total, p.batch, geo.parts);
    if (range >= ranges) return;
    walk.t = total * range / ranges;
    walk.end = total * (range + 1) / ranges;
    const unsigned who = __ballot_sync(0xffffffffu, walk.t >= inc - mine && walk.t < inc);
    const int src = __ffs(who) - 1;                            // (walk.t < total: somebody has it)
    walk.base = __shfl_sync(0xffffffffu, inc - mine, src);
    walk.b = __shfl_sync(0xffffffffu, b0, src);
    for (int nt; walk.t >= walk.base + (nt = walk.tiles_of(walk.b)); ++walk.b) walk.base += nt;
  }
  const int count = (int)(walk.end - walk.t);

  if (tid == 0) {
    for (int i = 0; i < NQ; ++i) {
      mbar_init(smem_u32(&sh->q_full[i]), 1);
      mbar_init(smem_u32(&sh->q_empty[i]), 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(smem_u32(&sh->s_full[i]), 1);
      mbar_init(smem_u32(&sh->o_done[i]), 1);
      mbar_init(smem_u32(&sh->p_ready[0][i]), 128 / kSplit);
      mbar_init(smem_u32(&sh->p_ready[1][i]), 128 / kSplit);
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(smem_u32(&sh->kv_full[i]), 1);
      mbar_init(smem_u32(&sh->kv_empty[i]), 1);
    }
    mbar_init(smem_u32(&sh->decided[0]), 256 / kSplit);
    mbar_init(smem_u32(&sh->decided[1]), 256 / kSplit);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh->o_free[i]), kApart ? kRows : kSoftmax / kSplit);
      mbar_init(smem_u32(&sh->o_last[i]), 1);
      mbar_init(smem_u32(&sh->ended[i]), kSoftmax / kSplit);
    }
    sh->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kTmaWarp) {
    tmem_alloc(smem_u32(&sh->tmem_base), 512);
    tmem_relinquish();
  }
  if constexpr (kSplit > 1) {                                  // rows that do not exist: 0, and so are their scores and probabilities
    constexpr int kEmpty = (kBM - kRows) * 8;
    for (int i = tid; i < NQ * (D / 64) * kEmpty; i += kThreads)
      st_shared_v4(sQ + i / kEmpty * (kBM * 128) + kRows * 128 + i % kEmpty * 16, make_uint4(0u, 0u, 0u, 0u));
    fence_proxy_async();
  }
  // the append kernel before this one may still run: it writes the cache, the bits of the mask and the result of the checks
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const bool nothing = (geo.bad != nullptr && *geo.bad != 0u) || (sQ & 1023u) != 0u;
  if ((sQ & 1023u) != 0u && tid == 0) sh->abort_flag = 97;

  // The sums of the segments' rows, (reference, sum) of the four parts of a row: over rows of the first queries' tile that do not exist.
  float2* ends = reinterpret_cast<float2*>(tiles + kRows * 128);
  static_assert(!kApart || 2 * 4 * kRows * 8 <= (kBM - kRows) * 128, "room for the sums");
  // Columns [c0, c1) of a row from the accumulator at tO: to the output, or to a piece of it.
  auto write_rows = [&](const Segment& seg, int row, bool row_ok, float l_all, float m_fin, uint32_t tO, int c0, int c1, float* ws_l) {
    const bool piece = seg.nt < seg.all;
    const float inv = l_all > 0.f ? 1.f / l_all : 0.f;
    // a piece that begins its sequence goes to the CTA's second slot, any other (it then begins the range) to the first
    const int64_t slot = (int64_t)blockIdx.x * 2 + (seg.first == 0);
    const int64_t at = slot * kBM + row - m0;
    T* og = reinterpret_cast<T*>(p.o) + (int64_t)seg.b * p.o_stride[0] + (int64_t)(row >> geo.pack_log2) * p.o_stride[1] +
            (int64_t)(h + (row & ((1 << geo.pack_log2) - 1))) * p.o_stride[2];
#pragma unroll 1
    for (int c = c0; c < c1; c += 16) {
      uint32_t ra[16];
      float o[16];
      tmem_ld16(tO + c, ra);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = __uint_as_float(ra[i]) * inv;
      if (row_ok && piece) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4*>(geo.ws + at * D + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      } else if (row_ok) {
#pragma unroll
        for (int i = 0; i < 16; i += 8)
          *reinterpret_cast<uint4*>(og + c + i) = make_uint4(Elem<T>::pack(o[i], o[i + 1]), Elem<T>::pack(o[i + 2], o[i + 3]),
                                                             Elem<T>::pack(o[i + 4], o[i + 5]), Elem<T>::pack(o[i + 6], o[i + 7]));
      }
      __syncwarp();
    }
    if (piece && c0 == 0 && row_ok) ws_l[at] = l_all > 0.f ? m_fin + log2f(l_all) : -INFINITY;
  };

  if (!kApart && warp >= 18) {
    reg_dealloc<64>();
  } else if (warp == kTmaWarp) {
    // ------------------------------- TMA producer ---------------------------------------
    reg_dealloc<64>();
    const bool many = geo.box_rows < kBN;                      // a tile of keys is several pages
    if (!nothing && (lane == 0 || many)) {
      if (lane == 0) {
        prefetch_tmap(&tmQ);
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
      }
      const int box_log2 = many ? 31 - __clz(geo.box_rows) : 7;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      // What the loads of a tile need: its page (of box `lane`), its first row or how many boxes there are, and whose queries it begins (or -1).
      struct Tile {
        int page, at, fresh;
      };
      Segment seg;
      int j = 0, segs = 0;
      seg.nt = 0;
      auto fetch = [&](Tile& t) {
        t.fresh = -1;
        if (j == seg.nt) {
          walk.next(seg);                                      // (no more than `count` tiles are asked for)
          j = 0;
          t.fresh = seg.b;
        }
        const int tile = seg.n_hi - 1 - j++, key = tile * kBN + (many ? lane << box_log2 : 0);
        t.page = geo.batch_idx ? geo.batch_idx[seg.b] : seg.b;
        t.at = tile * kBN + (geo.leftpad ? geo.leftpad[seg.b] : 0);
        if (geo.table) {
          t.page = lane < (kBN >> box_log2) && key < seg.k_len
                       ? geo.table[(int64_t)seg.b * geo.table_stride + (geo.page_log2 >= 0 ? key >> geo.page_log2 : key / geo.page_size)]
                       : 0;
          t.at = geo.page_log2 >= 0 ? (tile * kBN) & (geo.page_size - 1) : (tile * kBN) % geo.page_size;
          if (many) t.at = max(0, min(kBN >> box_log2, ((seg.k_len - tile * kBN - 1) >> box_log2) + 1));
        }
      };
      auto load = [&](const CUtensorMap* tm, const Tile& t) {
#pragma unroll
        for (int un = 0; un < NU; ++un) {
          const uint32_t bar = smem_u32(&sh->kv_full[stage]), dst = sKV + stage * C::kUnitBytes;
          if (lane == 0) ok = ok && wait_bar(&sh->kv_empty[stage], phase ^ 1, sh, 11);
          if (many) {
            // boxes that start past the last key are not loaded (their rows are masked, and zeroed in V)
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            if (!ok) return;
            if (lane == 0) mbar_expect_tx(bar, t.at * (C::kUnitCols * 2 << box_log2));
            __syncwarp();
            if (lane < t.at) {
              for (int bx = 0; bx < C::kBoxes; ++bx)
                tma_load_4d(dst + bx * (kBN * 128) + (lane << box_log2) * 128, tm, bar, un * C::kUnitCols + bx * 64, hk, 0, t.page);
            }
          } else {
            if (!ok) return;
            mbar_expect_tx(bar, C::kUnitBytes);
            for (int bx = 0; bx < C::kBoxes; ++bx)
              tma_load_4d(dst + bx * (kBN * 128), tm, bar, un * C::kUnitCols + bx * 64, hk, t.at, t.page);
          }
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      };
      // order of use: K_0 .. K_(NB-1), then V_J, K_(J+NB); a page is read one tile ahead of its use
      Tile held[NB], next;
      fetch(next);
      for (int i = 0; i < count + NB && ok; ++i) {
        if (i >= NB) load(&tmV, held[0]);
#pragma unroll
        for (int k = 0; k + 1 < NB; ++k) held[k] = held[k + 1];
        if (i < count) {
          const Tile now = next;
          held[NB - 1] = now;
          if (now.fresh >= 0) {
            if (lane == 0) {
              const int qb = segs % NQ;
              if (segs >= NQ) ok = ok && wait_bar(&sh->q_empty[qb], (segs / NQ - 1) & 1, sh, 15);
              if (ok) {
                const uint32_t bar = smem_u32(&sh->q_full[qb]);
                mbar_expect_tx(bar, C::kQBytes / kSplit);
                for (int bx = 0; bx < D / 64; ++bx)
                  tma_load_4d(sQ + qb * C::kQBytes + bx * (kBM * 128), &tmQ, bar, bx * 64, h, m0 >> geo.pack_log2, now.fresh);
              }
            }
            if (many) ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            ++segs;
          }
          if (i + 1 < count) fetch(next);
          if (ok) load(&tmK, now);
        }
      }
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------- MMA issuer -----------------------------------------
    // The whole warp runs the control flow in lock step and every lane polls the barriers;
    // the lane chosen once by elect_one issues the MMAs and commits.
    reg_dealloc<64>();
    if (!nothing) {
      constexpr uint32_t idesc_qk = make_idesc(1, TFmt<T>::code, 0, 0, kBM, kBN);
      constexpr uint32_t idesc_pv = make_idesc(1, TFmt<T>::code, 0, 1, kBM, C::kUnitCols);
      const uint32_t leader = elect_one() ? 1u : 0u;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      auto wwait = [&](uint64_t* bar, uint32_t parity, int code) {
        if (ok) ok = wait_bar(bar, parity, sh, code);
        ok = __all_sync(0xffffffffu, ok);                      // (the lanes leave together)
        tc_fence_after();
      };
      auto advance = [&]() { if (++stage == S) { stage = 0; phase ^= 1; } };
      Walk vwalk = walk;
      Segment qs, vs;                                          // of the tiles of Q K^T and of P V
      int qj = 0, vj = 0, qsegs = 0, vsegs = 0;
      qs.nt = vs.nt = 0;
      int qbuf = 0, vbuf = 0;
      uint32_t par = 0;                                        // (J / NB) & 1 of P V
      for (int i = 0; i < count + NB && ok; ++i) {
        if (i >= NB) {                                         // O += P V of tile i - NB
          if (vj == vs.nt) {
            vwalk.next(vs);
            vj = 0;
            ++vsegs;
          }
          const uint32_t a = tmem + vbuf * kBN;
          uint32_t v[NU];
          int st[NU];
#pragma unroll
          for (int un = 0; un < NU; ++un) {
            wwait(&sh->kv_full[stage], phase, 24);
            st[un] = stage;
            v[un] = sKV + stage * C::kUnitBytes;
            advance();
          }
          if (!ok) break;
          // Keys that no row sees -- past the end of the sequence, nodes that it does not use -- may hold anything, and 0 times
          // a NaN is one: their values become 0.  Here, because this warp knows that the ring entry is loaded.
          const int k0 = (vs.n_hi - 1 - vj) * kBN;
          if (k0 + kBN > vs.pos0) {
            constexpr int kChunks = NU * C::kBoxes * 8, kRowsAtOnce = 32 / kChunks > 0 ? 32 / kChunks : 1;
            const uint32_t* any = geo.tree_bits + ((int64_t)vs.b * (geo.tokens + 1) + geo.tokens) * geo.tree_words;
            bool zeroed = false;
            for (int c0 = 0; c0 < kBN; c0 += 32) {
              const uint32_t dead = ~seen_of(any, geo.tree_words, k0 + c0 - vs.pos0);
              if (dead == 0u) continue;
              zeroed = true;
              for (int r0 = 0; r0 < 32; r0 += kRowsAtOnce) {
#pragma unroll
                for (int c = lane; c < kRowsAtOnce * kChunks; c += 32) {
                  const int r = r0 + c / kChunks, chunk = c % kChunks, un = chunk / (C::kBoxes * 8), in = chunk % (C::kBoxes * 8);
                  if (dead >> r & 1u)
                    st_shared_v4((NU > 1 && un ? v[NU - 1] : v[0]) + (in / 8) * (kBN * 128) + (c0 + r) * 128 + in % 8 * 16,
                                 make_uint4(0u, 0u, 0u, 0u));
                }
              }
            }
            if (zeroed) {
              fence_proxy_async();
              __syncwarp();
            }
          }
          const uint32_t fresh = vj > 0 ? 1u : 0u;             // (accumulate)
          const int ob = (vsegs - 1) % NO;                     // accumulator
          if (vj == 0 && vsegs > NO) wwait(&sh->o_free[ob], ((vsegs - 1) / NO - 1) & 1, 27);
          wwait(&sh->p_ready[0][vbuf], par, 25);
          if (!ok) break;
#pragma unroll
          for (int un = 0; un < NU; ++un) {
            const uint64_t dv = make_smem_desc(v[un], kBN * 128, 1024);
#pragma unroll
            for (int kk = 0; kk < kBN / 32; ++kk) {
              mma_f16_ts_lp(tmem + C::kOCol + ob * D + un * C::kUnitCols, a + (kk / 2) * 32 + (kk % 2) * 8, dv + ((kk * 2048) >> 4), idesc_pv, kk > 0 ? 1u : fresh, leader);
            }
          }
          wwait(&sh->p_ready[1][vbuf], par, 26);
          if (!ok) break;
#pragma unroll
          for (int un = 0; un < NU; ++un) {
            const uint64_t dv = make_smem_desc(v[un], kBN * 128, 1024);
#pragma unroll
            for (int kk = kBN / 32; kk < kBN / 16; ++kk) {
              mma_f16_ts_lp(tmem + C::kOCol + ob * D + un * C::kUnitCols, a + (kk / 2) * 32 + (kk % 2) * 8, dv + ((kk * 2048) >> 4), idesc_pv, 1u, leader);
            }
            mma_commit_lp(smem_u32(&sh->kv_empty[st[un]]), leader);
          }
          mma_commit_lp(smem_u32(&sh->o_done[vbuf]), leader);
          if (++vj == vs.nt && kApart) mma_commit_lp(smem_u32(&sh->o_last[ob]), leader);
          if (++vbuf == NB) { vbuf = 0; par ^= 1; }
        }
        if (i < count) {                                       // S[qbuf] = Q K^T of tile i
          if (qj == qs.nt) {
            walk.next(qs);
            qj = 0;
            ++qsegs;
            wwait(&sh->q_full[(qsegs - 1) % NQ], ((qsegs - 1) / NQ) & 1, 21);
          }
          const int qb = (qsegs - 1) % NQ;
#pragma unroll
          for (int un = 0; un < NU; ++un) {
            wwait(&sh->kv_full[stage], phase, 22);
            if (!ok) break;
            const uint64_t dq = make_smem_desc(sQ + qb * C::kQBytes + un * (C::kUnitCols / 64) * (kBM * 128), 16, 1024);
            const uint64_t dk = make_smem_desc(sKV + stage * C::kUnitBytes, 16, 1024);
#pragma unroll
            for (int kk = 0; kk < C::kUnitCols / 16; ++kk) {
              const uint32_t o = ((kk / 4) * (kBM * 128) + (kk % 4) * 32) >> 4;
              mma_f16_ss_lp(tmem + qbuf * kBN, dq + o, dk + o, idesc_qk, (un > 0 || kk > 0) ? 1u : 0u, leader);
            }
            mma_commit_lp(smem_u32(&sh->kv_empty[stage]), leader);
            advance();
          }
          if (!ok) break;
          if (++qj == qs.nt) mma_commit_lp(smem_u32(&sh->q_empty[qb]), leader);
          mma_commit_lp(smem_u32(&sh->s_full[qbuf]), leader);
          if (++qbuf == NB) qbuf = 0;
        }
      }
    }
  } else if (kApart && warp >= 16 + kRows / 32) {
    reg_dealloc<64>();
  } else if (kApart && warp >= 16) {
    // ------------------------------- results --------------------------------------------
    reg_dealloc<64>();
    const int row = (warp & 1) * 32 + lane;          // also the TMEM lane
    const bool row_ok = row < rows;
    const uint32_t lane_addr = (uint32_t)((warp & 1) * 32) << 16;
    float* ws_l = geo.ws + (int64_t)gridDim.x * 2 * kBM * D;
    Segment seg;
    for (int segs = 0; !nothing && walk.next(seg); ++segs) {
      const int ob = segs & 1;
      const uint32_t par = (segs >> 1) & 1;
      if (!__all_sync(0xffffffffu, wait_bar(&sh->ended[ob], par, sh, 36) && wait_bar(&sh->o_last[ob], par, sh, 37))) break;
      tc_fence_after();
      float2 e[4];
      float m_fin = -INFINITY, l_all = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = ends[(ob * 4 + i) * kRows + row];
        m_fin = fmaxf(m_fin, e[i].x);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) l_all += e[i].x == m_fin ? e[i].y : e[i].y * exp2f(e[i].x - m_fin);
      write_rows(seg, row, row_ok, l_all, m_fin, tmem + lane_addr + C::kOCol + ob * D, 0, D, ws_l);
      tc_fence_before();
      mbar_arrive(smem_u32(&sh->o_free[ob]));
    }
  } else if ((warp & 3) >= kRows / 32) {
    reg_alloc<104>();                                // (rows that do not exist)
  } else {
    // ------------------------------- softmax groups -------------------------------------
    reg_alloc<104>();
    const int x = warp >> 3, half = (warp >> 2) & 1;
    const int row_in_tile = (warp & 3) * 32 + lane;  // TMEM lane
    const int row = m0 + row_in_tile, node_of = min(row >> geo.pack_log2, geo.tokens - 1);
    const int together = 2 + x * 4 + (warp & 3);     // barrier with the warp of the other half
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const bool row_ok = row < rows;
    float* ws_l = geo.ws + (int64_t)gridDim.x * 2 * kBM * D;
    bool ok = true;
    int J0 = 0;
    Segment seg;
    for (int segs = 0; !nothing && ok && walk.next(seg); ++segs, J0 += seg.nt) {
      const int nt = seg.nt;
      const uint32_t tO = tmem + lane_addr + C::kOCol + segs % NO * D;
      float m_own = -INFINITY, sum = 0.f;            // of this thread's keys: their sum relative to m_own
      for (int j = (J0 & 1) ^ x; j < nt; j += 2) {
        const int J = J0 + j, buf = J % NB;
        const uint32_t par = (J / NB) & 1;
        const uint32_t tS = tmem + lane_addr + buf * kBN + half * 64;
        const int k0 = (seg.n_hi - 1 - j) * kBN + half * 64;       // of this half
        const bool masked = k0 + 64 > seg.pos0;
        // 32 scores, scaled, and what this row does not see at -inf
        auto mask_chunk = [&](uint32_t (&r)[32], int cc) {
          const uint32_t* bits = geo.tree_bits + ((int64_t)seg.b * (geo.tokens + 1) + node_of) * geo.tree_words;
          const uint32_t seen = seen_of(bits, geo.tree_words, k0 + 32 * cc - seg.pos0);
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = seen >> i & 1u ? __float_as_uint(__uint_as_float(r[i]) * scale_log2) : __float_as_uint(-INFINITY);
        };

        // (After a wait that ran out a warp goes on without waiting, to the end of the segment: the warp of the other half meets it twice a
        // tile in any case.  What is computed is thrown away.)
        if (ok) ok = __all_sync(0xffffffffu, wait_bar(&sh->s_full[buf], par, sh, 31 + x));
        tc_fence_after();
        // ---- row maximum.  The scores are read twice, 32 at a time, which keeps these loops short: with a row's scores in
        // registers and everything unrolled, the softmax warps waited for instructions more than for anything else -----------------
        float mx = -INFINITY;
#pragma unroll 1
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t r[32];
          tmem_ld32(tS + cc * 32, r);
          tmem_wait_ld();
          if (masked) mask_chunk(r, cc);
          float mt[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mt[i] = fmax3(__uint_as_float(r[i]), __uint_as_float(r[4 + i]), __uint_as_float(r[8 + i]));
#pragma unroll
          for (int i = 0; i < 4; ++i) mt[i] = fmax3(mt[i], __uint_as_float(r[12 + i]), __uint_as_float(r[16 + i]));
#pragma unroll
          for (int i = 0; i < 4; ++i) mt[i] = fmax3(mt[i], __uint_as_float(r[20 + i]), __uint_as_float(r[24 + i]));
#pragma unroll
          for (int i = 0; i < 4; ++i) mt[i] = fmaxf(mt[i], __uint_as_float(r[28 + i]));
          mx = fmaxf(fmax3(mx, mt[0], mt[1]), fmaxf(mt[2], mt[3]));
        }
        const float mul = masked ? 1.f : scale_log2;
        mx *= mul;
        sh->part[2 * x + half][row_in_tile] = mx;

        // ---- the maximum the exponents are relative to, settled in tile order -------------
        // (the halves of a tile come to the same: the reference before it and the larger of their maxima)
        // (also for the first tile of a segment: its reference takes the place of the last segment's)
        if (J > 0 && ok) ok = __all_sync(0xffffffffu, wait_bar(&sh->decided[x ^ 1], ((J - 1) >> 1) & 1, sh, 33 + x));
        const float m_old = j > 0 ? sh->mref[row_in_tile] : -INFINITY;
        sync_halves(together);
        mx = fmaxf(mx, sh->part[2 * x + (half ^ 1)][row_in_tile]);
        const bool need = j == 0 || mx > m_old + rescale_at;
        const float m_use = need ? mx : m_old;
        if (need && half == 0) sh->mref[row_in_tile] = mx;
        if (j > 0 && __any_sync(0xffffffffu, need)) {
          // The accumulator may be touched once P V of the tile before is finished: the one of this
          // tile cannot start before P is written below.  A half of the columns each.
          if (ok) ok = __all_sync(0xffffffffu, wait_bar(&sh->o_done[(J - 1) % NB], ((J - 1) / NB) & 1, sh, 35 + x));
          tc_fence_after();
          const float alpha = need ? exp2f(m_old - mx) : 1.f;      // from -inf: 0
#pragma unroll 1
          for (int cc = half * (D / 64); cc < (half + 1) * (D / 64); ++cc) {
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
        sync_halves(together);                                     // (P V of either half's keys goes to all columns)
        mbar_arrive(smem_u32(&sh->decided[x]));
        const float m_safe = (m_use == -INFINITY) ? 0.f : m_use;
        if (m_use != m_own) {
          sum *= exp2f(m_own - m_use);                             // from -inf: 0
          m_own = m_use;
        }

        // ---- P = exp2(s - m), row sum, P -> TMEM over the scores: those of 32 keys over the first 16 columns of theirs ---------------
        const float2 mul2 = make_float2(mul, mul), nm2 = make_float2(-m_safe, -m_safe);
        float2 acc2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t r[32];
          tmem_ld32(tS + cc * 32, r);
          tmem_wait_ld();
          if (masked) mask_chunk(r, cc);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 a = f2fma(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), mul2, nm2);
            const float2 pe = make_float2(ex2(a.x), ex2(a.y));
            acc2[(i >> 1) & 1] = f2add(acc2[(i >> 1) & 1], pe);
            pk[i >> 1] = Elem<T>::pack(pe.x, pe.y);
          }
          tmem_st16(tS + cc * 32, pk);
        }
        sum += (acc2[0].x + acc2[0].y) + (acc2[1].x + acc2[1].y);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&sh->p_ready[half][buf]));
      }

      // ---- end of the segment --------------------------------------------------------------
      if constexpr (kApart) {
        if (ok && segs >= 2) ok = wait_bar(&sh->o_free[segs & 1], ((segs >> 1) - 1) & 1, sh, 38);      // (the sums there have been read)
        ends[((segs & 1) * 4 + 2 * x + half) * kRows + row_in_tile] = make_float2(m_own, sum);
        mbar_arrive(smem_u32(&sh->ended[segs & 1]));
        ok = !any_of<64>(!ok, together);                   // (the warps of both halves leave together)
        continue;
      }
      // a quarter of the columns each
      sync_all<kSoftmax / kSplit>();                       // every decision is made
      const int last = J0 + nt - 1;
      const float m_fin = sh->mref[row_in_tile];
      sh->part[2 * x + half][row_in_tile] = m_own == m_fin ? sum : sum * exp2f(m_own - m_fin);
      sync_all<kSoftmax / kSplit>();
      const float l_all = (sh->part[0][row_in_tile] + sh->part[1][row_in_tile]) + (sh->part[2][row_in_tile] + sh->part[3][row_in_tile]);
      if (ok) ok = wait_bar(&sh->o_done[last % NB], (last / NB) & 1, sh, 37 + x);
      if (any_of<kSoftmax / kSplit>(!ok || sh->abort_flag != 0, 1)) break;
      tc_fence_after();
      const int c0 = (2 * x + half) * (D / 4);
      write_rows(seg, row, row_ok, l_all, m_fin, tO, c0, c0 + D / 4, ws_l);
      tc_fence_before();
      mbar_arrive(smem_u32(&sh->o_free[0]));
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kTmaWarp) tmem_dealloc(tmem, 512);
  if (tid == 0) report_abort(sh->abort_flag, host_status);
}

// Adds up the pieces of the sequences that are cut, 256 / (D / 4) rows of a unit per CTA: grid (row groups x units, sequences or, where there are
// fewer of them, ends of ranges: one that is the first inside a sequence stands for it).
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(const fa_attn_args p, const CacheGeo geo) {
  constexpr int kRows = 256 / (D / 4);
  const int heads = p.heads_q >> geo.pack_log2, rows = geo.tokens << geo.pack_log2, mtiles = (rows + kBM - 1) / kBM, U = heads * mtiles;
  const int u = blockIdx.x / (kBM / kRows), m0 = u % mtiles * kBM, r = blockIdx.x % (kBM / kRows) * kRows + threadIdx.x / (D / 4);
  const int h = (u / mtiles) << geo.pack_log2, d = threadIdx.x % (D / 4) * 4, lane = threadIdx.x & 31;
  Walk walk;
  walk.seqlens = geo.seqlens;
  walk.n_new = geo.n_new;
  walk.capacity = geo.capacity;
  const int per = (p.batch + 31) / 32, b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
  int64_t mine = 0;
  for (int i = b0; i < b1; ++i) mine += walk.tiles_of(i);
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  const int64_t total = __shfl_sync(0xffffffffu, inc, 31), ranges = ranges_of(total, p.batch, geo.parts);
  // the sequence and its first tile, `before`
  const bool by_sequence = p.batch < geo.parts;
  const int64_t cut = total * (blockIdx.y + 1) / ranges;       // end of range blockIdx.y
  const bool owner = by_sequence ? (int)blockIdx.y >= b0 && (int)blockIdx.y < b1 : cut >= inc - mine && cut < inc;
  const unsigned who = __ballot_sync(0xffffffffu, owner);
  asm volatile("griddepcontrol.wait;" ::: "memory");           // (what has been read so far is no other kernel's work)
  if (who == 0u || (!by_sequence && (int64_t)blockIdx.y + 1 >= ranges)) return;
  int b = __shfl_sync(0xffffffffu, b0, __ffs(who) - 1), nt = 0;
  int64_t before = __shfl_sync(0xffffffffu, inc - mine, __ffs(who) - 1);
  for (; nt = walk.tiles_of(b), by_sequence ? b < (int)blockIdx.y : before + nt <= cut; ++b) before += nt;
  // the range of a tile: the last one that begins at it or before
  const int first = (int)(((before + 1) * ranges - 1) / total), last = (int)(((before + nt) * ranges - 1) / total);
  if (first == last || (!by_sequence && first != (int)blockIdx.y) || m0 + r >= rows || (geo.bad != nullptr && *geo.bad != 0u)) return;
  const float* ws_l = geo.ws + (int64_t)geo.parts * U * 2 * kBM * D;
  const int parts = last - first + 1;
  // the piece that begins the sequence is in its CTA's second slot
  auto slot_of = [&](int i) { return ((int64_t)(first + i) * U + u) * 2 + (i == 0); };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float wsum = 0.f, m = -INFINITY;
  for (int i0 = 0; i0 < parts; i0 += kMergeAtOnce) {
    float l[kMergeAtOnce];
    float4 v[kMergeAtOnce];
#pragma unroll
    for (int k = 0; k < kMergeAtOnce; ++k) {
      const int64_t at = slot_of(min(i0 + k, parts - 1)) * kBM + r;
      l[k] = i0 + k < parts ? ws_l[at] : -INFINITY;
      v[k] = *reinterpret_cast<const float4*>(geo.ws + at * D + d);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < kMergeAtOnce; ++k) mn = fmaxf(mn, l[k]);
    const float mf = mn == -INFINITY ? 0.f : mn, sc = exp2f(m - mf);
    acc.x *= sc; acc.y *= sc; acc.z *= sc; acc.w *= sc;
    wsum *= sc;
    m = mn;
#pragma unroll
    for (int k = 0; k < kMergeAtOnce; ++k) {
      if (i0 + k >= parts) break;
      const float w = exp2f(l[k] - mf);              // pieces without a finite score weigh 0, which a NaN in them survives
      wsum += w;
      acc.x += w * v[k].x; acc.y += w * v[k].y; acc.z += w * v[k].z; acc.w += w * v[k].w;
    }
  }
  const float f = wsum > 0.f ? 1.f / wsum : 0.f;
  const int gr = m0 + r;
  uint2 pk;
  pk.x = Elem<T>::pack(acc.x * f, acc.y * f);
  pk.y = Elem<T>::pack(acc.z * f, acc.w * f);
  *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.o) + (int64_t)b * p.o_stride[0] + (int64_t)(gr >> geo.pack_log2) * p.o_stride[1] +
                            (int64_t)(h + (gr & ((1 << geo.pack_log2) - 1))) * p.o_stride[2] + d) = pk;
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
static int units_of(const fa_decode_args& d, int pack_log2) {
  return (d.heads_q >> pack_log2) * (int)((((int64_t)d.seqlen_q << pack_log2) + kBM - 1) / kBM);
}

// Ranges for U units: as many as there are SMs for, and beyond that the number of ranges (up to 8) whose last wave is the fullest, less a fiftieth
// for each wave.  Measured with 0, 0.02, 0.1 in its place (us, head_dim 64): 100 units, 4 x 1000 tokens 69, 52, 51; 16 x 4000 376, 368, 368;
// 128 units, 8 x 4000 383, 385, 391 to 403; head_dim 128, 90 units, 16 x 4000 492, 466, 465; 110 units 576, 584, 575.
int tree_sm100_ranges(const fa_decode_args& d, int pack_log2) {
  const int U = units_of(d, pack_log2), sms = sm_count(d.device);
  if (2 * U <= sms) return sms / U;
  int best = 1;
  double cost = 1e30;
  for (int n = 1; n <= 8; ++n) {
    const int64_t waves = ((int64_t)U * n + sms - 1) / sms;
    const double c = (double)waves / n + 0.02 * waves;
    if (c < cost) {
      cost = c;
      best = n;
    }
  }
  return best;
}
// Two pieces of every CTA, with their LSEs.
size_t tree_sm100_piece_bytes(const fa_decode_args& d, int pack_log2) {
  const int ranges = tree_sm100_ranges(d, pack_log2);
  return ranges == 1 ? 0 : (size_t)units_of(d, pack_log2) * ranges * 2 * kBM * (d.head_dim + 1) * sizeof(float);
}

static bool encode_rows(CUtensorMap* m, const void* base, int D, int heads, int64_t rows, int64_t batch, const int64_t* stride, int box_heads,
                        int box_rows) {
  // dims (innermost first): head_dim, heads, rows, batch (or page)
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)heads, (uint64_t)rows, (uint64_t)batch};
  const uint64_t strides[3] = {(uint64_t)stride[2] * 2, (uint64_t)stride[1] * 2, (uint64_t)stride[0] * 2};
  const uint32_t box[4] = {64, (uint32_t)box_heads, (uint32_t)box_rows, 1};
  return encode_tmap(m, base, 2, 4, dims, strides, box);
}

template <typename T, int D, int kSplit>
static int launch_tree(const fa_decode_args& d, const CacheGeo& geo, float scale_log2, float rescale_at, cudaStream_t st) {
  fa_attn_args a = {};
  a.dtype = d.dtype;
  a.device = d.device;
  a.batch = d.batch;
  a.seqlen_q = d.seqlen_q;
  a.heads_q = d.heads_q;
  a.heads_kv = d.heads_kv;
  a.head_dim = D;
  a.o = d.o;
  for (int i = 0; i < 3; ++i) a.o_stride[i] = d.o_stride[i];
  const int pack = 1 << geo.pack_log2;
  CUtensorMap tm[3];
  if (!encode_rows(&tm[0], d.q, D, d.heads_q, d.seqlen_q, d.batch, d.q_stride, pack, kBM / kSplit / pack) ||
      !encode_rows(&tm[1], d.k_cache, D, d.heads_kv, d.page_size, d.num_pages, d.kc_stride, 1, geo.box_rows) ||
      !encode_rows(&tm[2], d.v_cache, D, d.heads_kv, d.page_size, d.num_pages, d.vc_stride, 1, geo.box_rows)) {
    set_error("tree_sm100: cuTensorMapEncodeTiled failed");
    return FA_ERR_LAUNCH;
  }
  using C = TCfg<D, (kSplit > 1 && D <= 128)>;
  static_assert(C::kSmemBytes <= 227 * 1024, "shared memory budget");
  auto kern = tree_sm100_kernel<T, D, kSplit>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
  if (e != cudaSuccess) {
    set_error("tree_sm100: cudaFuncSetAttribute(%d): %s", C::kSmemBytes, cudaGetErrorString(e));
    return FA_ERR_LAUNCH;
  }
  cudaLaunchConfig_t lc = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  lc.gridDim = dim3((unsigned)units_of(d, geo.pack_log2) * geo.parts);
  lc.blockDim = dim3(kThreads);
  lc.dynamicSmemBytes = C::kSmemBytes;
  lc.stream = st;
  lc.attrs = &attr;
  lc.numAttrs = 1;
  cudaLaunchKernelEx(&lc, kern, tm[0], tm[1], tm[2], a, scale_log2, rescale_at, geo, host_wait_word(d.device));
  if (int r = check_launch("tree_sm100")) return r;
  if (geo.parts == 1) return FA_OK;
  lc.gridDim = dim3((unsigned)units_of(d, geo.pack_log2) * (kBM * D / 4 / 256), (unsigned)(d.batch < geo.parts ? d.batch : geo.parts - 1));
  lc.blockDim = dim3(256);
  lc.dynamicSmemBytes = 0;
  cudaLaunchKernelEx(&lc, tree_merge_kernel<T, D>, a, geo);
  return check_launch("tree_merge");
}

template <typename T>
static int launch_rows(const fa_decode_args& d, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st) {
  const int64_t rows = (int64_t)d.seqlen_q << geo.pack_log2;
  auto launch = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    const float s = cfg.scale_log2, r = cfg.rescale_at;
    return rows <= 32 ? launch_tree<T, D, 4>(d, geo, s, r, st) : rows <= 64 ? launch_tree<T, D, 2>(d, geo, s, r, st) : launch_tree<T, D, 1>(d, geo, s, r, st);
  };
  switch (d.head_dim) {
    case 64: return launch(std::integral_constant<int, 64>{});
    case 128: return launch(std::integral_constant<int, 128>{});
    case 256: return launch(std::integral_constant<int, 256>{});
  }
  set_error("tree_sm100: head_dim %d", d.head_dim);
  return FA_ERR_UNSUPPORTED;
}

int tree_sm100(const fa_decode_args& d, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st) {
  return d.dtype == FA_BF16 ? launch_rows<__nv_bfloat16>(d, geo, cfg, st) : launch_rows<__half>(d, geo, cfg, st);
}

int tree_sm100_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_tree_status, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int tree_sm100_clear_status() {
  const int z = 0;
  return cudaMemcpyToSymbol(g_tree_status, &z, sizeof(int)) == cudaSuccess ? 0 : -1;
}

}  // namespace fa
