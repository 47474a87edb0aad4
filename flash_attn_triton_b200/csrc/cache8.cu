// Calls on the 8-bit KV cache: value checks, append, attention.  A decode step is one launch where nothing is appended and the tables are
// small, else the append (which then makes the checks) and the attention behind it.
#include "cache8_host.h"
#include "cache_dev.cuh"
#include "cache_geo.cuh"
#include "check_words.h"

namespace fa {

int decode8_int8(const fa_decode_args&, const fa_cache8&, const ScoreCfg&, int, const Geom8&, const DecodeCheck&, bool, cudaStream_t);
int decode8_e4m3(const fa_decode_args&, const fa_cache8&, const ScoreCfg&, int, const Geom8&, const DecodeCheck&, bool, cudaStream_t);
Geom8 decode8_geometry(const fa_decode_args& a, const fa_cache8& c, int unit_rows, int row_groups);
int cache8_chunk(const fa_decode_args& d, const fa_cache8& c, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st);
int cache8_pair(const fa_decode_args& d, const fa_cache8& c, const CacheGeo& geo, const ScoreCfg& cfg, cudaStream_t st);
int cache8_chunk_pieces(int head_dim);
int cache8_pair_pieces(int head_dim);
int launch_decode_check(const fa_decode_args& a, uint32_t* host, uint32_t* dev, cudaStream_t st);

namespace {

constexpr size_t kAlign = 16;
size_t aligned(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

int unit_rows_of(const fa_decode_args& a) { return a.seqlen_q * (a.heads_q / a.heads_kv) <= 8 ? 8 : 16; }

// How a call is run.  Workspace: pieces, counters if the caller brings none, the word with the result of the checks.
struct Plan {
  bool chunk, pair;                    // pair: 256 query rows per CTA
  int unit_rows;                       // decode
  Geom8 geo;
  int pack_log2, parts, capacity;      // chunk
  size_t piece_bytes, counter_bytes;
  int counters;
  bool append, inside;                 // the first kernel makes the checks, in every CTA
  size_t word_at() const { return aligned(piece_bytes) + aligned(counter_bytes); }
  size_t bytes() const { return word_at() + kAlign; }
};

// A chunk: more than 16 query rows per KV head.  The decode kernel would read the cache once per 16 rows; the tcgen05 kernel takes 128 at a
// time (4 x 256 tokens behind 1024 to 8192, 32 heads over 8 of 128: 669 us, 199).  Near the border, without an append, 4 sequences of those lengths,
// heads of 64 / 128, tcgen05 against decode units: 24 rows 43 / 47 us against 35 / 42, 48 rows 44 / 50 against 41 / 51, 64 rows 44 / 51 against
// 48 / 59; 32 sequences: 171 / 194 against 146 / 200, 171 / 194 against 195 / 269, 172 / 195 against 242 / 336.  So decode units would gain up to
// a fifth at 17 to 32 rows.  They would gain more where the group is no power of two, whose heads do not share a tile: 28 heads over 4, 3 tokens
// (21 rows) 100 / 113 against 26 / 36, 8 tokens (56 rows) 101 / 114 against 35 / 41.
bool plan_chunk(const fa_decode_args& a, const fa_cache8& c, Plan& p) {
  const int G = a.heads_q / a.heads_kv;
  if (a.num_splits != 0 || (int64_t)a.seqlen_q * G <= 16 || a.softmax_scale < 0.f) return false;
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return false;
  if (a.block_table && a.page_size % 16 != 0) return false;          // 16 keys are looked up at a time
  p.pack_log2 = 0;
  if ((G & (G - 1)) == 0 && G <= 64)
    while ((1 << p.pack_log2) < G) ++p.pack_log2;
  const int64_t cap = a.block_table ? (int64_t)a.block_table_stride * a.page_size : a.page_size;
  const int64_t rows = (int64_t)a.seqlen_q << p.pack_log2;
  p.pair = a.head_dim <= 128 && rows > 128 && a.alibi_slopes == nullptr && a.cache_leftpad == nullptr && c.block % 16 == 0;
  const int per_cta = p.pair ? 256 : 128;
  const int64_t mtiles = (rows + per_cta - 1) / per_cta;
  const int64_t units = (int64_t)a.batch * (a.heads_q >> p.pack_log2) * mtiles;
  if (units > (1 << 28) || cap > (1 << 30)) return false;
  p.capacity = (int)cap;
  // pieces of at least four key tiles, only while the units do not fill the SMs twice (chunk_pieces() has how many there are), and no more
  // than a merge has room for the weights of (pairs: 144; one unit alone would have a piece per SM)
  const int64_t sms = sm_count(a.device), fill = units >= 2 * sms ? 1 : sms / units > 4 ? sms / units : 4, most = (cap + 511) / 512;
  const int64_t room = p.pair ? cache8_pair_pieces(a.head_dim) : cache8_chunk_pieces(a.head_dim);
  p.parts = (int)(fill < most ? fill : most);
  if (p.parts > room) p.parts = (int)room;
  if (p.parts < 1) p.parts = 1;
  p.counters = p.parts > 1 ? (int)units : 0;
  p.piece_bytes = p.parts > 1 ? (size_t)units * p.parts * per_cta * (a.head_dim + 1) * sizeof(float) : 0;
  return true;
}

Plan plan_of(const fa_decode_args& a, const fa_cache8& c) {
  Plan p = {};
  p.chunk = plan_chunk(a, c, p);
  if (!p.chunk) {
    p.unit_rows = unit_rows_of(a);
    const int64_t rows = (int64_t)a.seqlen_q * (a.heads_q / a.heads_kv);
    const int groups = (int)((rows + p.unit_rows - 1) / p.unit_rows);
    p.geo = decode8_geometry(a, c, p.unit_rows, groups);
    p.piece_bytes = p.geo.splits == 1 ? 0 : (size_t)p.geo.rows * a.seqlen_q * a.heads_q * (a.head_dim + 1) * sizeof(float);
    p.counters = p.piece_bytes ? a.batch * a.heads_kv * groups : 0;
  }
  p.counter_bytes = a.counters ? 0 : (size_t)p.counters * sizeof(uint32_t);
  p.append = a.k_new != nullptr;
  // (an append has few CTAs: 16 x 84 entries, checked by a kernel of its own in front, cost a step of 45 us 5 of them)
  p.inside = (int64_t)a.batch * (a.block_table ? a.block_table_stride : 1) <= (p.append ? 4 * kInlineCheck : kInlineCheck) &&
             (p.append || !p.chunk);
  return p;
}

bool empty(const fa_decode_args& a) { return a.batch <= 0 || a.seqlen_q <= 0 || a.heads_q <= 0 || a.heads_kv <= 0; }

// host: word for the checks or null; *queued is set once a kernel that writes it is on the stream.
int run(const fa_decode_args& args, const fa_cache8& c, const Plan& plan, uint32_t* host, bool* queued, cudaStream_t st) {
  fa_decode_args a = args;
  char* ws = static_cast<char*>(a.workspace);
  uint32_t* word = reinterpret_cast<uint32_t*>(ws + plan.word_at());
  if (plan.counters && a.counters == nullptr) {
    a.counters = reinterpret_cast<uint32_t*>(ws + aligned(plan.piece_bytes));
    const cudaError_t e = cudaMemsetAsync(a.counters, 0, plan.counter_bytes, st);
    if (e != cudaSuccess) {
      set_error("decode8: cudaMemsetAsync: %s", cudaGetErrorString(e));
      return FA_ERR_LAUNCH;
    }
  }
  const bool check = host != nullptr, first = check && !plan.inside;
  if (first) {
    if (int r = launch_decode_check(a, host, word, st)) return r;
    *queued = true;
  }
  if (plan.append) {
    const bool here = check && plan.inside;
    if (int r = append8_launch(append_of(a, c), &a, a.dtype, c.code, a.device, here ? host : nullptr, check ? word : nullptr, here, st)) return r;
    if (here) *queued = true;
  }
  const bool behind = plan.append || first;
  ScoreCfg cfg = make_score_cfg(a.softmax_scale, 0.f, a.causal, a.window_left, a.window_right, a.alibi_slopes != nullptr);
  // Chunks raise a row's maximum late only where the type of the outputs hides it.  Weights are one fp16 each: the largest of a row is exactly
  // 1 relative to its own maximum and rounded like the others relative to an older one (error against float64, 2 x 1537 tokens behind 5000 to
  // 11000: fp16 9.5e-4 at most and 1.34e-5 rms raised at once, 1.47e-3 and 1.56e-5 late, 853 and 787 us; bf16, 4 x 256 behind 1024 to 8192:
  // 1.641e-4 and 1.647e-4 rms, 220 and 200 us).
  if (a.dtype == FA_F16) cfg.rescale_at = 0.f;
  if (plan.chunk) {
    CacheGeo geo = {};
    geo.seqlens = a.cache_seqlens;
    geo.table = a.block_table;
    geo.table_stride = a.block_table_stride;
    geo.batch_idx = a.cache_batch_idx;
    geo.leftpad = a.cache_leftpad;
    geo.page_size = a.page_size;
    geo.page_log2 = page_shift_of(a);
    geo.box_rows = 128;                // keys that one copy brings: they lie inside one page
    while (a.block_table && a.page_size % geo.box_rows != 0) geo.box_rows /= 2;
    geo.n_new = plan.append ? a.seqlen_new : 0;
    geo.tokens = a.seqlen_q;
    geo.pack_log2 = plan.pack_log2;
    geo.parts = plan.parts;
    geo.sms = sm_count(a.device);
    geo.capacity = plan.capacity;
    geo.ws = reinterpret_cast<float*>(ws);
    geo.counters = a.counters;
    geo.bad = check ? word : nullptr;
    return plan.pair ? cache8_pair(a, c, geo, cfg, st) : cache8_chunk(a, c, geo, cfg, st);
  }
  const DecodeCheck chk = {check && plan.inside && !plan.append ? host : nullptr, check && behind ? word : nullptr};
  const int r = c.code == FA_CODE_INT8 ? decode8_int8(a, c, cfg, plan.unit_rows, plan.geo, chk, behind, st)
                                       : decode8_e4m3(a, c, cfg, plan.unit_rows, plan.geo, chk, behind, st);
  if (check && r == FA_OK) *queued = true;
  return r;
}

int refused(const fa_decode_args& a, const Plan& plan) {
  if (plan.chunk)
    if (const int code = host_wait_status(a.device)) {
      set_error("fa_decode_paged8: a bounded device-side wait ran out earlier on device %d (code %d); the tcgen05 kernels "
                "stay off until fa_device_wait_clear()", a.device, code);
      return FA_ERR_DEVICE_WAIT;
    }
  if (a.workspace == nullptr || a.workspace_bytes < plan.bytes()) {
    set_error("decode8 workspace too small: need %zu bytes, got %zu", plan.bytes(), a.workspace_bytes);
    return FA_ERR_WORKSPACE;
  }
  FA_REQUIRE(a.counters == nullptr || a.num_counters >= plan.counters, "decode8: too few counters");
  return FA_OK;
}

}  // namespace

size_t decode8_workspace_bytes(const fa_decode_args& a, const fa_cache8& c) { return empty(a) ? 0 : plan_of(a, c).bytes(); }
int decode8_counters(const fa_decode_args& a, const fa_cache8& c) { return empty(a) ? 0 : plan_of(a, c).counters; }

int decode8_paged(const fa_decode_args& a, const fa_cache8& c, cudaStream_t st) {
  if (empty(a)) return FA_OK;
  const Plan plan = plan_of(a, c);
  if (int r = refused(a, plan)) return r;
  return run(a, c, plan, nullptr, nullptr, st);
}

int decode8_paged_checked(const fa_decode_args& a, const fa_cache8& c, uint32_t* failed, cudaStream_t st) {
  *failed = 0;
  if (empty(a)) return FA_OK;
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone) {
    cudaGetLastError();
    set_error("value checks cannot run while the stream is being captured; turn them off with set_validation(False)");
    return FA_ERR_LAUNCH;
  }
  const Plan plan = plan_of(a, c);
  if (int r = refused(a, plan)) return r;
  uint32_t* host = nullptr;
  const int slot = take_check_word(false, a.device, &host);
  if (slot < 0) return FA_ERR_LAUNCH;
  bool queued = false;
  int r = run(a, c, plan, host, &queued, st);
  if (queued) {
    const int w = await_check_word(slot, failed, st);
    if (r == FA_OK) r = w;
  }
  give_check_word(slot, queued);
  return r;
}

}  // namespace fa
