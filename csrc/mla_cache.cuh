// The 8-bit MLA latent cache: format and argument blocks shared by its kernels.
//
// A cache of B sequences and Tmax slots holds e4m3 codes [B, Tmax, L] and one fp32 scale per token
// [B, Tmax]; value = code * scale.  The scale is the least power of two 2^k, k >= -126, under which
// the row's largest magnitude fits e4m3 (448 * 2^k).  A power of two costs no accuracy (e4m3 is a
// floating-point format: its relative step does not depend on where in a binade the row's maximum
// falls), makes the division exact, and a value then has four significant bits, so it is exact in
// bf16.  A row holding a NaN or an infinity gets scale NaN and codes 0: codes are always finite, so
// a stale or masked row can never turn 0 * code into NaN inside a matrix product.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"

namespace kimi {
namespace mlac {

constexpr float kLog2e = 1.4426950408889634f;

KIMI_D int64_t get(const MlaCacheInts& v, int b) {
  return v.is64 ? static_cast<const int64_t*>(v.p)[b] : (int64_t) static_cast<const int32_t*>(v.p)[b];
}

// Length of sequence b as given, and the position of its first query token.  Both are cut to +-2^40, far past any slot:
// a position of INT64_MAX sees every key, and adding to it does not wrap.
KIMI_D int64_t cut(int64_t v) {
  constexpr int64_t far = (int64_t)1 << 40;
  return v < -far ? -far : v > far ? far : v;
}
KIMI_D int64_t first_position(const MlaCacheAttnArgs& a, int b, int64_t* len) {
  *len = cut(get(a.lengths, b));
  return a.start.p ? cut(get(a.start, b)) : *len - a.queries;
}

// Two e4m3 codes (low half of `w`) to floats.
KIMI_D float2 codes2(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xFFFFu), __NV_E4M3);
  return __half22float2(__half2(h));
}
KIMI_D float code1(uint8_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(__half(h));
}
KIMI_D uint32_t to_codes2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

}  // namespace mlac
}  // namespace kimi
