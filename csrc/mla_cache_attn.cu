// Attention of one or a few query tokens per sequence over the 8-bit MLA latent cache.
//
//   s_iht = scale * scale_t * sum_l q_ihl code_tl      for t < lengths[b], t <= start[b] + i
//   o_ihl = sum_t softmax_t(s)_iht * scale_t * code_tl  (a row that sees no key: zeros)
//
// q is absorbed into the latent space (W_uk^T q), one latent row serves as key and value of every
// head, so the rows (i, h) of one sequence share each cache byte read.  start[b] is the position of
// the first query token (lengths[b] - queries when not given).
//
// The long axis is split over CTAs; each keeps a running maximum and sum per row (base 2) and an
// unnormalised context, and a second kernel joins the splits.
#include "device_info.h"
#include "mla_cache.cuh"
#include "mla_cache_attn.h"

namespace kimi {
namespace {

using namespace mlac;

constexpr int kThreads = 256;
constexpr int kRows = 8;   // query rows of a CTA
constexpr int kChunk = 32;  // tokens of a chunk, one lane each in the softmax

int generic_splits(const MlaCacheAttnArgs& a) {
  const int tiles = (a.queries * a.heads + kRows - 1) / kRows;
  const int64_t want = (2 * (int64_t)device_sms() + (int64_t)a.batch * tiles - 1) / ((int64_t)a.batch * tiles);
  const int64_t most = (a.cache.slots + 2 * kChunk - 1) / (2 * kChunk);
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n);
}

size_t generic_smem(int width) {
  const size_t wp = (width + 3) / 4 * 4;
  return kRows * wp * sizeof(float) + kChunk * (wp + 4) + kChunk * kRows * sizeof(float) + kChunk * sizeof(float) +
         4 * kRows * sizeof(float);
}

// Compensated addition (Kahan): `lost` carries what rounding took off the sum so far.
KIMI_D void add_kept(float& sum, float& lost, float x) {
  const float y = x - lost, t = sum + y;
  lost = (t - sum) - y;
  sum = t;
}

// fp32 arithmetic on any width and alignment: the form for fp32 queries and for what TMA cannot address (widths, strides
// or a base that are no multiples of 16 bytes; widths under 64).  A warp scores 4 tokens x 8 rows
// per pass over the latent axis (a lane holds four adjacent columns: 128 FMAs per 12 shared-memory
// loads); in the context phase a thread owns four adjacent columns of up to CP groups of 1,024.  A chunk's products
// are added up on their own and its total with the rounding kept: equal weights along a cache round the same way at
// every step, so 131,072 plain additions end up to 3e-3 off, these within a few roundings of a chunk.  The FMA
// pipes bound it: 16 x 2,048 tokens, 12 heads take 302 us at width 1,544, where TMA cannot address the rows,
// and 32 us on the tensor cores at width 1,552.  fp32 queries: 4 x up to 1,000 tokens, 10 heads, width 640 33.6 us.
template <typename T, int CP>
__global__ void __launch_bounds__(kThreads) attn_any_kernel(const __grid_constant__ MlaCacheAttnArgs a) {
  extern __shared__ __align__(16) unsigned char any_smem[];
  const int width = a.cache.width, wp = (width + 3) / 4 * 4, pitch = wp + 4;
  float* sq = reinterpret_cast<float*>(any_smem);                       // [kRows][wp]
  uint8_t* sx = reinterpret_cast<uint8_t*>(sq + kRows * wp);            // [kChunk][pitch]
  float* sp = reinterpret_cast<float*>(sx + kChunk * pitch);            // [kChunk][kRows]
  float* ssc = sp + kChunk * kRows;                                     // [kChunk] token scales
  float* sstat = ssc + kChunk;  // max, sum, rescale, what the sum's last addition lost: [kRows] each
  const int split = blockIdx.x, tile = blockIdx.y, b = blockIdx.z, splits = gridDim.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = a.queries * a.heads, row0 = tile * kRows, nrow = min(kRows, rows - row0);
  int64_t len;
  const int64_t start = first_position(a, b, &len);
  len = len < 0 ? 0 : len > a.cache.slots ? a.cache.slots : len;
  // keys that the last row of the tile sees, and this split's share of them in whole chunks
  const int64_t seen = start + (row0 + nrow - 1) / a.heads + 1;
  const int64_t lim = seen < len ? (seen < 0 ? 0 : seen) : len;
  const int64_t share = ((lim + splits - 1) / splits + kChunk - 1) / kChunk * kChunk;
  const int64_t t0 = (int64_t)split * share, t1 = t0 + share < lim ? t0 + share : lim;
  for (int i = tid; i < kRows * wp; i += kThreads) {
    const int r = i / wp, l = i - r * wp;
    float v = 0.f;
    if (r < nrow && l < width) {
      const int qi = (row0 + r) / a.heads, h = (row0 + r) - qi * a.heads;
      v = to_f<T>(static_cast<const T*>(a.q)[b * a.q_b + qi * a.q_i + h * a.q_h + l]);
    }
    sq[i] = v;
  }
  for (int i = tid; i < kChunk * pitch; i += kThreads) sx[i] = 0;
  if (tid < kRows) {
    sstat[tid] = -INFINITY;
    sstat[kRows + tid] = sstat[3 * kRows + tid] = 0.f;
  }
  float acc[CP][4][kRows], low[CP][4][kRows];  // context, and what its last addition lost
#pragma unroll
  for (int c = 0; c < CP; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int r = 0; r < kRows; ++r) acc[c][e][r] = low[c][e][r] = 0.f;
  const uint8_t* xb = a.cache.codes + b * a.cache.code_b;
  const float* cb = a.cache.scales + b * a.cache.scale_b;
  const bool words = width % 4 == 0 && a.cache.code_t % 4 == 0 && (reinterpret_cast<uintptr_t>(xb) & 3) == 0;
  const float to2 = a.scale * kLog2e;
  for (int64_t c0 = t0; c0 < t1; c0 += kChunk) {
    const int nt = (int)(t1 - c0 < kChunk ? t1 - c0 : kChunk);
    __syncthreads();  // the previous chunk is consumed
    if (words) {
      const int wn = width / 4;
#pragma unroll 4
      for (int i = tid; i < nt * wn; i += kThreads) {
        const int t = i / wn, l = i - t * wn;
        *reinterpret_cast<uint32_t*>(sx + t * pitch + l * 4) =
            __ldg(reinterpret_cast<const uint32_t*>(xb + (c0 + t) * a.cache.code_t) + l);
      }
    } else {
      for (int i = tid; i < nt * width; i += kThreads) {
        const int t = i / width, l = i - t * width;
        sx[t * pitch + l] = xb[(c0 + t) * a.cache.code_t + l];
      }
    }
    if (tid < kChunk) ssc[tid] = tid < nt ? cb[(c0 + tid) * a.cache.scale_t] : 0.f;
    __syncthreads();
    {
      constexpr int TW = kChunk / (kThreads / 32);  // tokens of a warp
      float dot[TW][kRows];
#pragma unroll
      for (int t = 0; t < TW; ++t)
#pragma unroll
        for (int r = 0; r < kRows; ++r) dot[t][r] = 0.f;
      for (int l = 4 * lane; l < wp; l += 128) {
        float x[TW][4];
#pragma unroll
        for (int t = 0; t < TW; ++t) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(sx + (warp * TW + t) * pitch + l);
          const float2 p = codes2(w), q = codes2(w >> 16);
          x[t][0] = p.x; x[t][1] = p.y; x[t][2] = q.x; x[t][3] = q.y;
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float4 q = *reinterpret_cast<const float4*>(sq + r * wp + l);
#pragma unroll
          for (int t = 0; t < TW; ++t) dot[t][r] += q.x * x[t][0] + q.y * x[t][1] + q.z * x[t][2] + q.w * x[t][3];
        }
      }
#pragma unroll
      for (int t = 0; t < TW; ++t)
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float d = warp_sum(dot[t][r]);
          if (lane == 0) sp[(warp * TW + t) * kRows + r] = d;
        }
    }
    __syncthreads();
    if (warp < nrow) {  // one warp per row, one lane per token
      const int64_t t = c0 + lane;
      const bool sees = lane < nt && t <= start + (row0 + warp) / a.heads;
      const float s = sp[lane * kRows + warp] * ssc[lane] * to2;
      const float m0 = sstat[warp], m = fmaxf(m0, warp_max(sees ? s : -INFINITY));
      const float base = m == -INFINITY ? 0.f : m;  // no key so far, or only -inf scores: weights of 0
      const float p = sees ? exp2f(s - base) : 0.f;
      const float sum = warp_sum(p);
      sp[lane * kRows + warp] = p * (sees ? ssc[lane] : 0.f);
      if (lane == 0) {
        const float f = exp2f(m0 - base);
        sstat[warp] = m;
        float total = sstat[kRows + warp] * f, lost = sstat[3 * kRows + warp] * f;
        add_kept(total, lost, sum);
        sstat[kRows + warp] = total;
        sstat[2 * kRows + warp] = f;
        sstat[3 * kRows + warp] = lost;
      }
    } else if (warp < kRows) {
      sp[lane * kRows + warp] = 0.f;
      if (lane == 0) sstat[2 * kRows + warp] = 1.f;
    }
    __syncthreads();
    float f[kRows];
    bool moved = false;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      f[r] = sstat[2 * kRows + r];
      moved |= f[r] != 1.f;
    }
#pragma unroll
    for (int c = 0; c < CP; ++c) {
      const int l = 4 * tid + c * 4 * kThreads;
      if (l >= wp) continue;
      float part[4][kRows];  // of this chunk
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < kRows; ++r) part[e][r] = 0.f;
      for (int t = 0; t < nt; ++t) {
        const float4 w0 = *reinterpret_cast<const float4*>(sp + t * kRows);
        const float4 w1 = *reinterpret_cast<const float4*>(sp + t * kRows + 4);
        const float w[kRows] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
        const uint32_t u = *reinterpret_cast<const uint32_t*>(sx + t * pitch + l);
        const float2 p = codes2(u), q = codes2(u >> 16);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          part[0][r] += w[r] * p.x;
          part[1][r] += w[r] * p.y;
          part[2][r] += w[r] * q.x;
          part[3][r] += w[r] * q.y;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          if (moved) {
            acc[c][e][r] *= f[r];
            low[c][e][r] *= f[r];
          }
          add_kept(acc[c][e][r], low[c][e][r], part[e][r]);
        }
    }
  }
  __syncthreads();
  const bool whole = splits == 1;
  float* ml = a.part_acc + (int64_t)a.batch * splits * rows * width;
  const int64_t slot = (int64_t)b * splits + split;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (r >= nrow) break;
    const float sum = sstat[kRows + r];
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int c = 0; c < CP; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int l = 4 * tid + c * 4 * kThreads + e;
        if (l >= width) continue;
        if (whole) static_cast<T*>(a.out)[((int64_t)b * rows + row0 + r) * width + l] = from_f<T>(acc[c][e][r] * inv);
        else if (sum != 0.f) a.part_acc[(slot * rows + row0 + r) * width + l] = acc[c][e][r];
      }
    if (!whole && tid == 0) {
      ml[(slot * rows + row0 + r) * 2] = sstat[r];
      ml[(slot * rows + row0 + r) * 2 + 1] = sum;
    }
  }
}

// Joins the splits of one row: weights 2^(m_s - max) against the split's own maximum.  A split without
// a key has sum 0 and its context is neither written nor read; a NaN sum is kept.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ MlaCacheAttnArgs a, int splits) {
  const int rows = a.queries * a.heads, width = a.cache.width;
  const int r = blockIdx.x % rows, b = blockIdx.x / rows;
  const float* ml = a.part_acc + (int64_t)a.batch * splits * rows * width;
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) {
    const float* p = ml + (((int64_t)b * splits + s) * rows + r) * 2;
    if (p[1] != 0.f) m = fmaxf(m, p[0]);
  }
  const float base = m == -INFINITY ? 0.f : m;
  const int l = blockIdx.y * 256 + threadIdx.x;
  if (l >= width) return;
  float acc = 0.f, sum = 0.f;
  for (int s = 0; s < splits; ++s) {
    const int64_t i = ((int64_t)b * splits + s) * rows + r;
    if (ml[i * 2 + 1] != 0.f) {
      const float f = exp2f(ml[i * 2] - base);
      sum += f * ml[i * 2 + 1];
      acc += f * a.part_acc[i * width + l];
    }
  }
  static_cast<T*>(a.out)[((int64_t)b * rows + r) * width + l] = from_f<T>(sum != 0.f ? acc / sum : 0.f);
}

template <typename T>
cudaError_t launch_any(const MlaCacheAttnArgs& a, cudaStream_t s) {
  const int rows = a.queries * a.heads, splits = generic_splits(a), width = a.cache.width;
  const int64_t tiles = (rows + kRows - 1) / kRows;
  if (tiles > 65535 || a.batch > 65535) return cudaErrorInvalidValue;
  const size_t smem = generic_smem(width);
  const dim3 grid(splits, (unsigned)tiles, a.batch);
  cudaError_t e;
#define KIMI_MLAC_ANY(CP)                                                             \
  do {                                                                                \
    e = ensure_dynamic_smem(attn_any_kernel<T, CP>, (int)smem);                       \
    if (e != cudaSuccess) return e;                                                   \
    attn_any_kernel<T, CP><<<grid, kThreads, smem, s>>>(a);                           \
  } while (0)
  if (width <= 1024) KIMI_MLAC_ANY(1);
  else KIMI_MLAC_ANY(2);
  
#undef KIMI_MLAC_ANY
  e = cudaGetLastError();
  if (e != cudaSuccess || splits == 1) return e;
  attn_join_kernel<T><<<dim3((unsigned)(a.batch * rows), (width + 255) / 256), 256, 0, s>>>(a, splits);
  return cudaGetLastError();
}

}  // namespace

// 8 rows of fp32 query and a 32-token chunk have to fit shared memory.
bool mla_cache_attn_supported(int width) { return width > 0 && width <= 2048; }

int mla_cache_attn_form(int dtype, int width) {
  if (!mla_cache_attn_supported(width)) return 0;
  MlaCacheAttnArgs a;  // one row over a contiguous cache
  a.cache.width = width;
  a.cache.code_t = width;
  a.cache.slots = 64;
  a.cache.code_b = a.cache.slots * width;
  a.batch = a.queries = a.heads = 1;
  return mla_attn_tc_supported(dtype, a) ? 2 : 1;
}

int64_t mla_cache_attn_workspace(int dtype, const MlaCacheAttnArgs& a) {
  if (mla_attn_tc_supported(dtype, a)) return mla_attn_tc_workspace(dtype, a);
  const int splits = generic_splits(a);
  return splits == 1 ? 0 : (int64_t)a.batch * splits * a.queries * a.heads * (a.cache.width + 2);
}

cudaError_t mla_cache_attn(int dtype, const MlaCacheAttnArgs& a, cudaStream_t s) {
  if (a.batch <= 0 || a.queries <= 0 || a.heads <= 0) return cudaSuccess;
  if (!mla_cache_attn_supported(a.cache.width)) return cudaErrorInvalidValue;
  if (mla_attn_tc_supported(dtype, a)) return mla_attn_tc(dtype, a, s);
  switch (dtype) {
    case 0: return launch_any<float>(a, s);
    case 1: return launch_any<__nv_bfloat16>(a, s);
    case 2: return launch_any<__half>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace kimi
