// Decode over the 8-bit KV cache: the kernels for codes of type int8.
#include "cache8_decode.cuh"

namespace fa {

int decode8_int8(const fa_decode_args& a, const fa_cache8& c, const ScoreCfg& cfg, int unit_rows, const Geom8& g, const DecodeCheck& chk,
                 bool behind, cudaStream_t st) {
  return a.dtype == FA_BF16 ? launch_decode8<__nv_bfloat16, FA_CODE_INT8>(a, c, cfg, unit_rows, g, chk, behind, st)
                            : launch_decode8<__half, FA_CODE_INT8>(a, c, cfg, unit_rows, g, chk, behind, st);
}

Geom8 decode8_geometry(const fa_decode_args& a, const fa_cache8& c, int unit_rows, int row_groups) {
  auto of = [&](auto d) {
    constexpr int D = decltype(d)::value;
    using S8 = Decode8<D, 8>;
    using S16 = Decode8<D, 16>;
    static_assert(S8::kTile8 == S16::kTile8, "");
    Geom8 g;
    g.row_groups = row_groups;
    g.resident = sm_count(a.device) * (unit_rows == 8 ? S8::kResident : S16::kResident);
    const int64_t cap = a.block_table ? (int64_t)a.block_table_stride * a.page_size : a.page_size;
    const int64_t nt = cap > 0 ? (cap + S8::kTile8 - 1) / S8::kTile8 : 1;
    g.max_tiles = (int)nt;
    g.page = div_by(a.page_size);
    g.block = div_by(c.block);
    g.k_page = (uint32_t)(a.kc_stride[0] / 16);
    g.k_row = (uint32_t)(a.kc_stride[1] / 16);
    g.v_page = (uint32_t)(a.vc_stride[0] / 16);
    g.v_row = (uint32_t)(a.vc_stride[1] / 16);
    g.splits = 0;
    if (a.num_splits > 0 || a.batch > kMaxBalanced || a.batch * nt > (1 << 30)) {
      g.splits = a.num_splits > 0 ? (int)(a.num_splits < nt ? a.num_splits : nt) : 1;
      g.ranges = g.rows = a.batch * g.splits;
    } else {
      // the most that any lengths ask for
      const int U = a.heads_kv * row_groups, once = g.resident / U;
      const int64_t most = a.batch * nt, n = once == 0 || most > (int64_t)kLongest8 * once ? (int64_t)kWaves8 * g.resident / U : once;
      g.ranges = (int)(n < 1 ? 1 : n < most ? n : most);
      g.rows = g.ranges + a.batch;
    }
    return g;
  };
  switch (a.head_dim) {
    case 16: return of(std::integral_constant<int, 16>{});
    case 32: return of(std::integral_constant<int, 32>{});
    case 64: return of(std::integral_constant<int, 64>{});
    case 128: return of(std::integral_constant<int, 128>{});
    default: return of(std::integral_constant<int, 256>{});
  }
}

}  // namespace fa
