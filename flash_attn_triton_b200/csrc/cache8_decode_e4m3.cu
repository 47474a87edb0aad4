// Decode over the 8-bit KV cache: the kernels for codes of type e4m3.
#include "cache8_decode.cuh"

namespace fa {

int decode8_e4m3(const fa_decode_args& a, const fa_cache8& c, const ScoreCfg& cfg, int unit_rows, const Geom8& g, const DecodeCheck& chk,
                 bool behind, cudaStream_t st) {
  return a.dtype == FA_BF16 ? launch_decode8<__nv_bfloat16, FA_CODE_E4M3>(a, c, cfg, unit_rows, g, chk, behind, st)
                            : launch_decode8<__half, FA_CODE_E4M3>(a, c, cfg, unit_rows, g, chk, behind, st);
}

}  // namespace fa
