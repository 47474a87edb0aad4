// Decode over the 8-bit KV cache: the kernels for codes of type int8.
#include "cache8_decode.cuh"

namespace fa {

int decode8_int8(const fa_decode_args& a, const fa_cache8& c, const ScoreCfg& cfg, int unit_rows, const DecodeGeom& g, const DecodeCheck& chk,
                 bool behind, cudaStream_t st) {
  return a.dtype == FA_BF16 ? launch_decode8<__nv_bfloat16, FA_CODE_INT8>(a, c, cfg, unit_rows, g, chk, behind, st)
                            : launch_decode8<__half, FA_CODE_INT8>(a, c, cfg, unit_rows, g, chk, behind, st);
}

DecodeGeom decode8_geometry(const fa_decode_args& a, int unit_rows, int row_groups) {
  auto of = [&](auto d) {
    constexpr int D = decltype(d)::value;
    using S8 = Decode8<D, 8>;
    using S16 = Decode8<D, 16>;
    static_assert(S8::kTile8 == S16::kTile8, "");
    return decode_geometry(a, row_groups, unit_rows == 8 ? S8::kResident : S16::kResident, S8::kTile8, kLongest8);
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
