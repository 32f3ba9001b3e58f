// Writing the 8-bit MLA latent cache and reading it back (format: mla_cache.cuh).
//
//   write   x [B, T, L] (fp32 / bf16 / fp16, any batch and token stride) -> codes and scale of slot
//           offsets[b] + j for j < counts[b]; slots outside [0, Tmax) are dropped.
//   read    codes, scales -> out [B, T, L] in fp32 / bf16 / fp16; rows at or past lengths[b] are zeros.
//
// Both move bytes: L * (sizeof(T) + 1) + 4 per token against a handful of integer operations per
// element.  One warp owns one token row.  The writer holds its row in registers between the maximum
// and the rounding, so x crosses HBM once; the maximum runs on the magnitudes' bit patterns, which
// order like the values and put infinities and NaN on top, two 16-bit elements per instruction.
//
// The copy rate bounds both: 64 x 4,096 rows of 1,536 in bf16 (1.21 GB) are written in 175 us (6.9 TB/s) and
// read in 185 us (6.5 TB/s; a measured plain copy: 6.55).  One decode step's 64 rows are 4.5 us of a caller's
// time, 1.5 to 2.2 on the GPU: the launch.  Splitting a row's number by a 32-bit division saved the small calls
// nothing and cost the large write 8 % (189 us).
#include <type_traits>

#include "mla_cache.cuh"

namespace kimi {
namespace {

using namespace mlac;

constexpr int kRowWarps = 4;  // rows (warps) per CTA

// Exponent k of the row's scale from the fp32 bits of its largest magnitude (finite).
KIMI_D int scale_exponent(uint32_t top) {
  // top = 1.M * 2^(E - 127) <= 1.75 * 2^(8 + k)  <=>  k >= E - 135, one more when 1.M > 1.75
  const int k = (int)(top >> 23) - 135 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return k < -126 ? -126 : k;
}
KIMI_D float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

// Eight consecutive elements as loaded, with the running maximum of their magnitudes' bits.
template <typename T>
struct Oct {
  uint32_t w[4];  // pairs of 16-bit elements
  KIMI_D void load(const T* p) { *reinterpret_cast<int4*>(w) = __ldg(reinterpret_cast<const int4*>(p)); }
  KIMI_D void clear() { w[0] = w[1] = w[2] = w[3] = 0; }
  KIMI_D uint32_t top(uint32_t t) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __vmaxu2(t, w[i] & 0x7FFF7FFFu);
    return t;
  }
  KIMI_D float2 pair(int i) const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    else
      return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
  static KIMI_D uint32_t fold(uint32_t t) { return max(t & 0xFFFFu, t >> 16); }
  // fp32 bits of the magnitude whose 16-bit pattern is t; non-finite patterns stay non-finite
  static KIMI_D uint32_t bits(uint32_t t) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return t << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)t)));
  }
};
template <>
struct Oct<float> {
  float f[8];
  KIMI_D void load(const float* p) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  KIMI_D void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
  }
  KIMI_D uint32_t top(uint32_t t) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) t = max(t, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    return t;
  }
  KIMI_D float2 pair(int i) const { return make_float2(f[2 * i], f[2 * i + 1]); }
  static KIMI_D uint32_t fold(uint32_t t) { return t; }
  static KIMI_D uint32_t bits(uint32_t t) { return t; }
};

// Slot of token j of sequence b, or -1.
KIMI_D int64_t write_slot(const MlaCacheWriteArgs& a, int b, int64_t j) {
  if (a.counts.p && j >= get(a.counts, b)) return -1;
  const int64_t s = cut(get(a.offsets, b)) + j;
  return s >= 0 && s < a.cache.slots ? s : -1;
}

// Rows of up to OCTS * 256 elements, L % 8 == 0, 16-byte aligned rows of x and 8-byte aligned rows of codes.
template <typename T, int OCTS>
__global__ void __launch_bounds__(kRowWarps * 32) write_kernel(const __grid_constant__ MlaCacheWriteArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (row >= (int64_t)a.batch * a.tokens) return;
  const int b = (int)(row / a.tokens);
  const int64_t j = row - (int64_t)b * a.tokens;
  const int64_t slot = write_slot(a, b, j);
  if (slot < 0) return;
  const T* x = static_cast<const T*>(a.x) + b * a.x_b + j * a.x_t;
  const int octs = a.cache.width >> 3;
  Oct<T> v[OCTS];
#pragma unroll
  for (int i = 0; i < OCTS; ++i) {
    const int o = lane + 32 * i;
    if (o < octs) v[i].load(x + o * 8);
    else v[i].clear();
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < OCTS; ++i) top = v[i].top(top);
  top = Oct<T>::bits(__reduce_max_sync(0xffffffffu, Oct<T>::fold(top)));
  const bool bad = top >= 0x7F800000u;
  const int k = bad ? 0 : scale_exponent(top);
  const float inv = pow2(-k);
  uint8_t* c = a.cache.codes + b * a.cache.code_b + slot * a.cache.code_t;
#pragma unroll
  for (int i = 0; i < OCTS; ++i) {
    const int o = lane + 32 * i;
    uint32_t r[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 p = v[i].pair(2 * h), q = v[i].pair(2 * h + 1);
      r[h] = bad ? 0u : to_codes2(p.x * inv, p.y * inv) | (to_codes2(q.x * inv, q.y * inv) << 16);
    }
    if (o < octs) *reinterpret_cast<uint2*>(c + o * 8) = make_uint2(r[0], r[1]);
  }
  if (lane == 0)
    a.cache.scales[b * a.cache.scale_b + slot * a.cache.scale_t] = bad ? __uint_as_float(0x7FC00000u) : pow2(k);
}

// Any width and alignment: two passes over the row, one element at a time.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) write_any_kernel(const __grid_constant__ MlaCacheWriteArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (row >= (int64_t)a.batch * a.tokens) return;
  const int b = (int)(row / a.tokens);
  const int64_t j = row - (int64_t)b * a.tokens;
  const int64_t slot = write_slot(a, b, j);
  if (slot < 0) return;
  const T* x = static_cast<const T*>(a.x) + b * a.x_b + j * a.x_t;
  uint32_t top = 0;
  for (int l = lane; l < a.cache.width; l += 32) top = max(top, __float_as_uint(to_f<T>(x[l])) & 0x7FFFFFFFu);
  top = __reduce_max_sync(0xffffffffu, top);
  const bool bad = top >= 0x7F800000u;
  const int k = bad ? 0 : scale_exponent(top);
  const float inv = pow2(-k);
  uint8_t* c = a.cache.codes + b * a.cache.code_b + slot * a.cache.code_t;
  for (int l = lane; l < a.cache.width; l += 32) c[l] = bad ? 0 : (uint8_t)to_codes2(to_f<T>(x[l]) * inv, 0.f);
  if (lane == 0)
    a.cache.scales[b * a.cache.scale_b + slot * a.cache.scale_t] = bad ? __uint_as_float(0x7FC00000u) : pow2(k);
}

template <typename T, bool OCT>
__global__ void __launch_bounds__(kRowWarps * 32) read_kernel(const __grid_constant__ MlaCacheReadArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (row >= (int64_t)a.batch * a.tokens) return;
  const int b = (int)(row / a.tokens);
  const int64_t j = row - (int64_t)b * a.tokens;
  const bool live = !a.lengths.p || j < get(a.lengths, b);
  const uint8_t* c = a.cache.codes + b * a.cache.code_b + j * a.cache.code_t;
  const float s = live ? a.cache.scales[b * a.cache.scale_b + j * a.cache.scale_t] : 0.f;
  T* y = static_cast<T*>(a.out) + row * a.cache.width;
  if constexpr (OCT) {
    const int octs = a.cache.width >> 3;
#pragma unroll 4
    for (int o = lane; o < octs; o += 32) {
      float f[8];
      uint2 w = make_uint2(0u, 0u);
      if (live) w = __ldg(reinterpret_cast<const uint2*>(c) + o);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = codes2((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
        f[2 * i] = p.x * s;
        f[2 * i + 1] = p.y * s;
      }
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(y + o * 8) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(y + o * 8 + 4) = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        Vec<T> v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v.set(i, f[i]);
        v.store(y + o * 8);
      }
    }
  } else {
    for (int l = lane; l < a.cache.width; l += 32) y[l] = from_f<T>(live ? code1(c[l]) * s : 0.f);
  }
}

bool aligned(const void* p, int64_t to) { return (reinterpret_cast<uintptr_t>(p) % to) == 0; }

template <typename T>
cudaError_t launch_write(const MlaCacheWriteArgs& a, cudaStream_t s) {
  const int64_t rows = (int64_t)a.batch * a.tokens, grid = (rows + kRowWarps - 1) / kRowWarps;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const int64_t eb = a.x_b * (int64_t)sizeof(T), et = a.x_t * (int64_t)sizeof(T);
  const bool oct = a.cache.width % 8 == 0 && aligned(a.x, 16) && eb % 16 == 0 && et % 16 == 0 &&
                   aligned(a.cache.codes, 8) && a.cache.code_b % 8 == 0 && a.cache.code_t % 8 == 0;
  const int octs = (a.cache.width / 8 + 31) / 32;
#define KIMI_MLAC_W(N) write_kernel<T, N><<<(unsigned)grid, kRowWarps * 32, 0, s>>>(a)
  if (oct && octs <= 8) {
    if (octs <= 1) KIMI_MLAC_W(1);
    else if (octs <= 2) KIMI_MLAC_W(2);
    else if (octs <= 3) KIMI_MLAC_W(3);
    else if (octs <= 4) KIMI_MLAC_W(4);
    else if (octs <= 6) KIMI_MLAC_W(6);
    else KIMI_MLAC_W(8);
  } else {
    write_any_kernel<T><<<(unsigned)grid, kRowWarps * 32, 0, s>>>(a);
  }
#undef KIMI_MLAC_W
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_read(const MlaCacheReadArgs& a, cudaStream_t s) {
  const int64_t rows = (int64_t)a.batch * a.tokens, grid = (rows + kRowWarps - 1) / kRowWarps;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const bool oct = a.cache.width % 8 == 0 && aligned(a.cache.codes, 8) && a.cache.code_b % 8 == 0 &&
                   a.cache.code_t % 8 == 0 && aligned(a.out, 16);
  if (oct) read_kernel<T, true><<<(unsigned)grid, kRowWarps * 32, 0, s>>>(a);
  else read_kernel<T, false><<<(unsigned)grid, kRowWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t mla_cache_write(int dtype, const MlaCacheWriteArgs& a, cudaStream_t s) {
  if (a.batch <= 0 || a.tokens <= 0) return cudaSuccess;
  switch (dtype) {
    case 0: return launch_write<float>(a, s);
    case 1: return launch_write<__nv_bfloat16>(a, s);
    case 2: return launch_write<__half>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t mla_cache_read(int dtype, const MlaCacheReadArgs& a, cudaStream_t s) {
  if (a.batch <= 0 || a.tokens <= 0) return cudaSuccess;
  switch (dtype) {
    case 0: return launch_read<float>(a, s);
    case 1: return launch_read<__nv_bfloat16>(a, s);
    case 2: return launch_read<__half>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace kimi
