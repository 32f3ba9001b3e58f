// Attention over the 8-bit MLA latent cache on tcgen05 (sm_100a), bf16 and fp16 queries.
//
//   s_rt = coef_r * scale_t * sum_l q_rl code_tl        rows r = (query token, head) of one sequence
//   o_rl = sum_t softmax_t(s)_rt * scale_t * code_tl     (a row that sees no key: zeros)
//
// The codes are the tensor cores' operand as they lie in memory.  Both products run as kind::f8f6f4
// MMAs with the cache tile as the A operand and the few query rows on N, so the padding of M = 128
// costs nothing for 3 heads and nothing is converted on the way:
//
//   S^T [64 tokens x rows]    = C [64 x L]    * Q^T [L x rows]        A K-major
//   O^T [128 latents x rows] += C^T [128 x 64] * P^T [64 x rows]      A MN-major, the same shared-memory tile
//
// One tile is 64 tokens, in boxes of 64 tokens x 128 latents (8 KB, TMA with the 128-byte swizzle): a
// box row of 128 bytes serves as a K-major row of the first product and as an MN-major row of the
// second.  O^T stays in TMEM for a whole sequence segment (L / 128 accumulators of `rows` columns).
//
// Splitting into 8-bit parts keeps 16-bit accuracy.  A query row is scaled by a power of two to
// [128, 256) and written as q = q0 + q1 / 32 + q2 / 1024 in e4m3, each part the rounding of what the
// one before left (5 bits a part): two parts hold every bf16, three every fp16 within 2^-17 of the
// row's maximum.  The parts sit side by side on N (A is read once) and are added in fp32.  The weights
// v = 2^(s + log2(scale_t) - ref) <= 2^15 are split into e5m2 parts (3 + 4 + 4 + .. bits) along K, all
// accumulating into the same columns: three for bf16 outputs (11 bits), four for fp16 (14 bits).  e5m2
// because of its range: the parts of a weight 2^-18 below the row's reference are still whole, where
// e4m3's step of 2^-9 would cut what many small weights add up to.
//
// The softmax reference of a row is a power of two that only moves when some weight would pass 2^15
// (then the row's accumulator columns are rescaled in TMEM, exactly); the sums use the scores alone
// with a reference of their own, so token scales far apart cost neither range nor accuracy.
//
// Work split: the tiles of all (sequence, row tile) pairs form one list, cut into equal contiguous
// ranges, one per CTA, from the lengths on the device: ragged batches stay balanced and a launch (or
// a captured graph) needs no lengths on the host.  A CTA that has a whole pair writes its output; the
// others leave a normalised context and its log-sum, joined by a second kernel in a fixed order.
//
// Roles of a CTA (10 warps): warp 0 loads, warp 1 issues the MMAs, warps 2-9 are two groups of four
// that share the rows: scores -> weights, rescaling, query preparation and the epilogue.
// Every mbarrier wait is bounded and reports through the status word.
#include <cudaTypedefs.h>

#include <mutex>

#include "device_info.h"
#include "mla_cache.cuh"
#include "mla_cache_attn.h"
#include "tc_common.cuh"

namespace kimi {
namespace {

using namespace mlac;

constexpr int kTile = 64;                  // tokens of a tile
constexpr int kBox = kTile * 128;          // bytes of a box
constexpr int kThreads = 320;
constexpr int kMaxSlots = 32;              // ring slots
constexpr int kSmemMax = 227 * 1024;
constexpr float kTop = 15.f;               // a weight may reach 2^kTop
constexpr float kRoom = 4.f;               // a new reference leaves this many bits
constexpr float kSumRoom = 40.f;           // the sums' reference may lag by this many bits

struct Plan {
  int rh = 0;          // rows of one compute group (template)
  int rows_tile = 0;   // rows of a pair (<= 2 * rh)
  int row_tiles = 0;
  int boxes = 0;       // boxes of a tile: ceil(L / 128)
  int slots = 0;       // ring slots
  int s_bufs = 0;
  int ahead = 0;       // boxes of the next tile's scores issued before this tile's context product
  uint32_t tmem = 0;
  size_t smem = 0;
  bool direct = false;  // one CTA per pair, nothing to join
  int grid = 0;
};

struct TcParams {
  CUtensorMap map;
  MlaCacheAttnArgs a;
  int rows, rows_tile, row_tiles, boxes, slots, s_bufs, ahead, direct, min_tiles, t_first;
  uint32_t tmem;
  int64_t z_mul;       // 0 when every sequence reads the same cache rows
  float* part_o;       // [grid + pairs][rows_tile][L]
  float* part_lse;     // [grid + pairs][rows_tile]
  int* prefix;         // [pairs + 2]: first tile of each pair, total, tiles per CTA
  int* status;
};

constexpr int pad16(int n) { return (n + 15) / 16 * 16; }
// QP parts of a query row; QP + 1 parts of a weight.
template <int RH, int QP>
struct Shape {
  static constexpr int WP = QP + 1;
  static constexpr int R = 2 * RH;             // rows, padded
  static constexpr int NS = pad16(QP * R);     // N of the score product
  static constexpr int NP = pad16(R);          // N of the context product
  static constexpr int P_BYTES = NP * 128 * ((WP + 1) / 2);  // one weight buffer
};

KIMI_D void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// kind::f8f6f4 instruction descriptor: fp32 accumulator, A e4m3 (0), B e4m3 (0) or e5m2 (1).
constexpr uint32_t idesc_f8(int m, int n, bool a_mn, bool b_e5m2) {
  return (1u << 4) | ((b_e5m2 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
KIMI_D void tmem_ld4(uint32_t addr, float* v) {
  uint32_t r[4];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
}
KIMI_D float tmem_ld1(uint32_t addr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n" : "=r"(r) : "r"(addr));
  return __uint_as_float(r);
}
KIMI_D void tmem_st1(uint32_t addr, float v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};\n" ::"r"(addr), "r"(__float_as_uint(v)) : "memory");
}
KIMI_D void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
KIMI_D void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
KIMI_D void group_sync(int id) { asm volatile("bar.sync %0, 128;\n" ::"r"(id) : "memory"); }
KIMI_D bool group_any(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n bar.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(id), "r"(v ? 1u : 0u)
      : "memory");
  return r != 0;
}
KIMI_D float pow2i(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }
// v * 2^e for any integer-valued e, exact while the result is a normal number.
KIMI_D float scale2(float v, float e) {
  const int n = (int)fminf(fmaxf(e, -250.f), 250.f), h = n / 2;
  return v * pow2i(h) * pow2i(n - h);
}
// The e5m2 parts of two fp16 values: takes the rounding off `h`, exactly.
KIMI_D uint32_t take_e5m2x2(__half2& h) {
  const __nv_fp8x2_storage_t c = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(h), __NV_SATFINITE, __NV_E5M2);
  h = __hsub2(h, __half2(__nv_cvt_fp8x2_to_halfraw2(c, __NV_E5M2)));
  return c;
}

// Tiles of pair v: the keys its last row sees.
KIMI_D int pair_tiles(const TcParams& p, int v, int64_t* len_out, int64_t* start_out) {
  const int b = v / p.row_tiles, rt = v - b * p.row_tiles;
  int64_t len = get(p.a.lengths, b);
  const int64_t start = p.a.start.p ? get(p.a.start, b) : len - p.a.queries;
  len = len < 0 ? 0 : len > p.a.cache.slots ? p.a.cache.slots : len;
  const int last = min(p.rows, (rt + 1) * p.rows_tile) - 1;
  const int64_t seen = start + last / p.a.heads + 1;
  const int64_t lim = seen < 0 ? 0 : seen < len ? seen : len;
  *len_out = len;
  *start_out = start;
  return (int)((lim + kTile - 1) / kTile);
}

// This CTA's share of the tile list, walked pair by pair (every role walks it on its own).
struct Walk {
  int v, skip, left;  // pair, tiles of it that belong to CTAs before, tiles of this CTA still to come
  int t0, t1, tiles;  // the segment: tiles [t0, t1) of the pair's `tiles`
  int64_t len, start;
  KIMI_D bool next(const TcParams& p, int pairs) {
    while (left > 0 && v < pairs) {
      tiles = pair_tiles(p, v, &len, &start);
      if (skip < tiles) {
        t0 = skip;
        t1 = min(tiles, skip + left);
        left -= t1 - t0;
        skip = 0;
        return true;
      }
      skip -= tiles;
      ++v;
    }
    return false;
  }
};

template <typename T, int RH, int QP>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ TcParams p) {
  using S = Shape<RH, QP>;
  constexpr int R = S::R;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);  // [slots][kBox]
  uint8_t* sq = ring + (size_t)p.slots * kBox;                // [boxes][NS][128] query parts
  uint8_t* sp = sq + (size_t)p.boxes * S::NS * 128;           // [2][P_BYTES] weight parts
  float* sref = reinterpret_cast<float*>(sp + 2 * S::P_BYTES);  // [R] weight references
  float* sreft = sref + R;                                    // [R] sum references
  float* scoef = sreft + R;                                   // [R] score factors
  float* sred = scoef + R;                                    // [2 kinds][4 warps][R]
  int* slim = reinterpret_cast<int*>(sred + 8 * R);           // [R] keys that a row sees
  uint64_t* bars = reinterpret_cast<uint64_t*>(slim + R);
  uint64_t* full = bars;
  uint64_t* empty = full + kMaxSlots;
  uint64_t* s_full = empty + kMaxSlots;
  uint64_t* s_empty = s_full + 2;
  uint64_t* p_full = s_empty + 2;
  uint64_t* pv_done = p_full + 2;
  uint64_t* q_full = pv_done + 2;
  uint64_t* drain = q_full + 1;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
  int* swalk = reinterpret_cast<int*>(tslot + 1);             // [3] first pair, skip, tiles

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pairs = p.a.batch * p.row_tiles;
  const int width = p.a.cache.width;

  // ---- set-up: barriers, TMEM, this CTA's share of the tiles
  if (tid == 0) {
    for (int i = 0; i < p.slots; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&s_empty[i], 8);
      tc::mbar_init(&p_full[i], 8);
      tc::mbar_init(&pv_done[i], 1);
    }
    tc::mbar_init(q_full, 8);
    tc::mbar_init(drain, 1);
    tc::fence_barrier_init();
    tc::tma_prefetch(&p.map);
  }
  if (warp == 1) tc::tmem_alloc(tslot, p.tmem);
  if (warp == 0) {
    int64_t len, start;
    if (p.direct) {
      const int n = pair_tiles(p, blockIdx.x, &len, &start);
      if (lane == 0) {
        swalk[0] = blockIdx.x;
        swalk[1] = 0;
        swalk[2] = n;
      }
    } else {
      int total = 0;
      for (int v0 = 0; v0 < pairs; v0 += 32) total += __reduce_add_sync(0xffffffffu, v0 + lane < pairs ? pair_tiles(p, v0 + lane, &len, &start) : 0);
      const int per = max(p.min_tiles, (total + (int)gridDim.x - 1) / (int)gridDim.x);
      const int mine = blockIdx.x * per;  // < 2^31: total tiles are bounded by the host
      int before = 0, first = pairs, skip = 0;
      for (int v0 = 0; v0 < pairs; v0 += 32) {
        const int n = v0 + lane < pairs ? pair_tiles(p, v0 + lane, &len, &start) : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        const int at = before + incl - n;
        if (blockIdx.x == 0 && v0 + lane < pairs) p.prefix[v0 + lane] = at;
        const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && mine >= at && mine < at + n);
        if (hit && first == pairs) {
          first = v0 + __ffs(hit) - 1;
          skip = mine - __shfl_sync(0xffffffffu, at, __ffs(hit) - 1);
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) {
        swalk[0] = first;
        swalk[1] = skip;
        swalk[2] = max(0, min(per, total - mine));
        if (blockIdx.x == 0) {
          p.prefix[pairs] = total;
          p.prefix[pairs + 1] = per;
        }
      }
    }
  }
  // rows of the weight buffers past R stay zero
  for (int i = tid; i < 2 * S::P_BYTES / 16; i += kThreads) reinterpret_cast<int4*>(sp)[i] = make_int4(0, 0, 0, 0);
  for (int i = tid; i < p.boxes * S::NS * 8; i += kThreads) reinterpret_cast<int4*>(sq)[i] = make_int4(0, 0, 0, 0);
  tc::fence_proxy_async();
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tslot;
  const uint32_t tm_s = tmem + (uint32_t)(p.boxes * S::NP);  // score buffers behind the accumulators
  Walk w;
  w.v = swalk[0];
  w.skip = swalk[1];
  w.left = swalk[2];

  if (warp == 0) {
    // ---- loads
    if (lane == 0) {
      bool ok = true;
      uint32_t n = 0;  // boxes loaded so far
      while (ok && w.next(p, pairs)) {
        const int b = w.v / p.row_tiles;
        for (int t = w.t0; ok && t < w.t1; ++t)
          for (int k = 0; k < p.boxes; ++k, ++n) {
            const uint32_t slot = n % p.slots, use = n / p.slots;
            if (use > 0 && !tc::mbar_wait(&empty[slot], (use - 1) & 1, p.status, tc::kTimeoutEmpty)) {
              ok = false;
              break;
            }
            tc::mbar_arrive_expect_tx(&full[slot], kBox);
            const int y = p.t_first ? t * kTile : (int)(b * p.z_mul), z = p.t_first ? (int)(b * p.z_mul) : t * kTile;
            tc::tma_load_3d(ring + (size_t)slot * kBox, &p.map, &full[slot], k * 128, y, z);
          }
        ++w.v;
      }
      // copies in flight land before the CTA ends
      for (uint32_t i = n > (uint32_t)p.slots ? n - p.slots : 0; i < n; ++i)
        tc::mbar_wait_local(&full[i % p.slots], (i / p.slots) & 1, p.status, tc::kTimeoutDrain, tc::kDrainNs);
    }
  } else if (warp == 1) {
    // ---- MMAs
    if (lane == 0) {
      bool ok = true;
      uint32_t n_tile = 0, seg = 0;  // tiles and segments so far
      constexpr uint32_t id_s = idesc_f8(64, S::NS, false, false);
      const uint32_t ring0 = tc::smem_u32(ring), q0 = tc::smem_u32(sq), p0 = tc::smem_u32(sp);
      auto scores = [&](uint32_t g, int k0, int k1) {  // boxes [k0, k1) of tile g's score product
        const uint32_t buf = g % p.s_bufs, use = g / p.s_bufs;
        if (k0 == 0) {
          if (use > 0 && !tc::mbar_wait(&s_empty[buf], (use - 1) & 1, p.status, tc::kTimeoutTmemEmpty)) return false;
          tc::tc_fence_after();
        }
        for (int k = k0; k < k1; ++k) {
          const uint32_t n = g * p.boxes + k, slot = n % p.slots;
          if (!tc::mbar_wait(&full[slot], (n / p.slots) & 1, p.status, tc::kTimeoutFull)) return false;
          tc::tc_fence_after();
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_f8(tm_s + buf * S::NS, tc::smem_desc_sw128(ring0 + slot * kBox + j * 32, 16, 1024),
                   tc::smem_desc_sw128(q0 + k * S::NS * 128 + j * 32, 16, 1024), id_s, (k | j) != 0);
        }
        if (k1 == p.boxes && k0 < k1) tc::mma_commit(&s_full[buf]);
        return true;
      };
      while (ok && w.next(p, pairs)) {
        if (!tc::mbar_wait(q_full, seg & 1, p.status, tc::kTimeoutTmemEmpty)) break;
        tc::tc_fence_after();
        ok = scores(n_tile, 0, p.boxes);
        for (int t = w.t0; ok && t < w.t1; ++t, ++n_tile) {
          const bool more = t + 1 < w.t1;
          if (more && p.ahead > 0 && !(ok = scores(n_tile + 1, 0, p.ahead))) break;
          const uint32_t pb = n_tile & 1;
          if (!(ok = tc::mbar_wait(&p_full[pb], (n_tile >> 1) & 1, p.status, tc::kTimeoutTmemFull))) break;
          tc::tc_fence_after();
          for (int k = 0; k < p.boxes; ++k) {
            const uint32_t slot = (n_tile * p.boxes + k) % p.slots;
#pragma unroll
            for (int part = 0; part < S::WP; ++part)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                mma_f8(tmem + (uint32_t)(k * S::NP), tc::smem_desc_sw128(ring0 + slot * kBox + j * 4096, 8192, 1024),
                       tc::smem_desc_sw128(p0 + pb * S::P_BYTES + (part >> 1) * S::NP * 128 + (part & 1) * 64 + j * 32, 16, 1024),
                       idesc_f8(128, S::NP, true, true), (t > w.t0 || part > 0 || j > 0) ? 1u : 0u);
            tc::mma_commit(&empty[slot]);
          }
          tc::mma_commit(&pv_done[pb]);
          if (more && p.ahead < p.boxes) ok = scores(n_tile + 1, p.ahead, p.boxes);
        }
        ++seg;
        ++w.v;
      }
      tc::mma_commit(drain);
      tc::mbar_wait_local(drain, 0, p.status, tc::kTimeoutDrain, tc::kDrainNs);
    }
  } else {
    // ---- compute groups: rows [grp * RH, grp * RH + RH) of the pair
    const int grp = (warp - 2) >> 2, quad = warp & 3, bar_id = 1 + grp, cw = warp - 2;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int tok = quad * 16 + (lane & 15);  // score lanes 0-15 of each quadrant hold the 64 tokens
    const bool active = lane < 16;
    const int r0 = grp * RH;
    float* red = sred + quad * R;  // [2][4][R]
    // A wait that fails only makes this warp skip its later waits: every warp walks all tiles, so the
    // groups' named barriers always meet and the kernel ends (its results are void, as the status says).
    bool ok = true;
    uint32_t n_tile = 0;
    auto wait = [&](uint64_t* bar, uint32_t use, int code) {  // the warp is converged again behind it
      ok = ok && tc::mbar_wait(bar, use & 1, p.status, code);
      __syncwarp();
      tc::tc_fence_after();
    };
    while (w.next(p, pairs)) {
      const int b = w.v / p.row_tiles, row0 = (w.v - b * p.row_tiles) * p.rows_tile;
      const int nrow = min(p.rows_tile, p.rows - row0);
      // -- query rows into parts; one warp per row
      for (int r = cw; r < nrow; r += 8) {
        const int qi = (row0 + r) / p.a.heads, h = (row0 + r) - qi * p.a.heads;
        const T* q = static_cast<const T*>(p.a.q) + b * p.a.q_b + qi * p.a.q_i + h * p.a.q_h;
        uint32_t top = 0;
        for (int l = lane; l < width; l += 32) top = max(top, __float_as_uint(to_f<T>(q[l])) & 0x7FFFFFFFu);
        top = __reduce_max_sync(0xffffffffu, top);
        const bool bad = top >= 0x7F800000u;
        const int k = bad ? 0 : min(126, 134 - (int)(top >> 23));  // the maximum to [128, 256)
        const float f = bad ? 0.f : pow2i(k);
        for (int l = lane; l < p.boxes * 128; l += 32) {
          float x = l < width && !bad ? to_f<T>(q[l]) * f : 0.f;
#pragma unroll
          for (int part = 0; part < QP; ++part) {
            const int n = part * R + r;
            const uint8_t c = (uint8_t)to_codes2(x, 0.f);
            sq[(size_t)(l >> 7) * S::NS * 128 + (n >> 3) * 1024 + (n & 7) * 128 + ((((l >> 4) & 7) ^ (n & 7)) << 4) + (l & 15)] = c;
            x = (x - code1(c)) * 32.f;
          }
        }
        if (lane == 0) scoef[r] = bad ? __uint_as_float(0x7FC00000u) : p.a.scale * kLog2e * pow2i(-k);
      }
      if (cw == 0)
        for (int r = lane; r < R; r += 32) {
          const int64_t seen = w.start + (row0 + r) / p.a.heads + 1;
          slim[r] = r >= nrow || seen < 0 ? 0 : (int)(seen < w.len ? seen : w.len);
          sref[r] = -INFINITY;
          sreft[r] = -INFINITY;
          if (r >= nrow) scoef[r] = 0.f;
        }
      tc::fence_proxy_async();
      tc::tc_fence_before();
      __syncwarp();
      asm volatile("bar.sync 3, 256;\n" ::: "memory");
      if (lane == 0) tc::mbar_arrive(q_full);
      float sum[RH];
#pragma unroll
      for (int r = 0; r < RH; ++r) sum[r] = 0.f;
      const float* scales = p.a.cache.scales + b * p.a.cache.scale_b;
      for (int t = w.t0; t < w.t1; ++t, ++n_tile) {
        const int at = t * kTile + tok;
        const float st = active && at < w.len ? scales[at * p.a.cache.scale_t] : 0.f;
        const float lg = log2f(st);
        const uint32_t buf = n_tile % p.s_bufs, pb = n_tile & 1;
        wait(&s_full[buf], n_tile / p.s_bufs, tc::kTimeoutTmemFull);
        float s[RH];
        {
          float v[QP][RH];
#pragma unroll
          for (int part = 0; part < QP; ++part)
#pragma unroll
            for (int r = 0; r < RH; r += 4) tmem_ld4(tm_s + lanes + buf * S::NS + part * R + r0 + r, v[part] + r);
          tmem_wait_ld();
#pragma unroll
          for (int r = 0; r < RH; ++r) {
            float x = v[QP - 1][r];
#pragma unroll
            for (int part = QP - 2; part >= 0; --part) x = fmaf(x, 0.03125f, v[part][r]);
            s[r] = x;
          }
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&s_empty[buf]);
        // slots past the length hold anything: their rows of the tile become zeros
        if ((int64_t)(t + 1) * kTile > w.len) {
          const int from = (int)(w.len - (int64_t)t * kTile), n = (kTile - from) * 8;
          for (int k = 0; k < p.boxes; ++k) {
            uint8_t* box = ring + (size_t)((n_tile * p.boxes + k) % p.slots) * kBox + from * 128;
            for (int i = tid - 64; i < n; i += 256) reinterpret_cast<int4*>(box)[i] = make_int4(0, 0, 0, 0);
          }
        }
        bool raise = false;
        uint32_t see = 0;
#pragma unroll
        for (int r = 0; r < RH; ++r) {
          s[r] *= scoef[r0 + r] * st;
          const bool on = active && at < slim[r0 + r];
          see |= (on ? 1u : 0u) << r;
          raise |= on && (s[r] + lg > sref[r0 + r] + kTop || s[r] > sreft[r0 + r] + kSumRoom);
        }
        __syncwarp();
        if (group_any(bar_id, raise)) {
          // some row outgrew its reference: new ones from the tile's maxima
#pragma unroll
          for (int r = 0; r < RH; ++r) {
            float ma = (see >> r) & 1 ? s[r] + lg : -INFINITY, ms = (see >> r) & 1 ? s[r] : -INFINITY;
            ma = warp_max(ma);
            ms = warp_max(ms);
            if (lane == 0) {
              red[r0 + r] = ma;
              red[4 * R + r0 + r] = ms;
            }
          }
          group_sync(bar_id);
          bool waited = false;
#pragma unroll
          for (int r = 0; r < RH; ++r) {
            float ma = -INFINITY, ms = -INFINITY;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              ma = fmaxf(ma, sred[q * R + r0 + r]);
              ms = fmaxf(ms, sred[(4 + q) * R + r0 + r]);
            }
            if (ms > sreft[r0 + r] + kSumRoom) sum[r] *= exp2f(sreft[r0 + r] - ceilf(ms));
            if (t > w.t0 && ma > sref[r0 + r] + kTop) {  // uniform over the group
              if (!waited) {
                wait(&pv_done[pb ^ 1], (n_tile - 1) >> 1, tc::kTimeoutTmemEmpty);
                waited = true;
              }
              const float d = sref[r0 + r] - (ceilf(ma) - (kTop - kRoom));
              for (int k = 0; k < p.boxes; ++k) {
                const uint32_t c = tmem + lanes + (uint32_t)(k * S::NP + r0 + r);
                float v = tmem_ld1(c);
                tmem_wait_ld();
                tmem_st1(c, d == -INFINITY ? 0.f : scale2(v, d));
              }
            }
          }
          if (waited) tmem_wait_st();
          group_sync(bar_id);
          if (quad == 0 && lane < RH) {
            float ma = -INFINITY, ms = -INFINITY;
            for (int q = 0; q < 4; ++q) {
              ma = fmaxf(ma, sred[q * R + r0 + lane]);
              ms = fmaxf(ms, sred[(4 + q) * R + r0 + lane]);
            }
            if (ma > sref[r0 + lane] + kTop) sref[r0 + lane] = ceilf(ma) - (kTop - kRoom);
            if (ms > sreft[r0 + lane] + kSumRoom) sreft[r0 + lane] = ceilf(ms);
          }
          group_sync(bar_id);
        }
        // weights into parts; the buffer was last read by the context product of two tiles ago
        if (n_tile >= 2) wait(&pv_done[pb], (n_tile >> 1) - 1, tc::kTimeoutTmemEmpty);
        uint8_t* wp = sp + pb * S::P_BYTES + (tok & 15);
#pragma unroll
        for (int r = 0; r < RH; r += 2) {
          float v[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = s[r + e], ax = x + lg;
            const bool on = (see >> (r + e)) & 1;
            // a score of -inf weighs nothing, also against a reference of -inf
            sum[r + e] += on && x != -INFINITY ? exp2f(x - sreft[r0 + r + e]) : 0.f;
            v[e] = on && ax != -INFINITY ? exp2f(ax - sref[r0 + r + e]) : 0.f;
          }
          if (active) {
            // fp16 holds three parts; with four, the first comes off in fp32
            __half2 h;
            if constexpr (S::WP == 3) h = __floats2half2_rn(v[0], v[1]);
#pragma unroll
            for (int part = 0; part < S::WP; ++part) {
              uint32_t c;
              if (S::WP > 3 && part == 0) {
                c = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E5M2);
                const float2 d = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c, __NV_E5M2)));
                h = __floats2half2_rn(v[0] - d.x, v[1] - d.y);
              } else {
                c = take_e5m2x2(h);
              }
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int n = r0 + r + e;
                wp[(part >> 1) * S::NP * 128 + (n >> 3) * 1024 + (n & 7) * 128 + ((((part & 1) * 4 + quad) ^ (n & 7)) << 4)] =
                    (uint8_t)(c >> (8 * e));
              }
            }
          }
        }
        tc::fence_proxy_async();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&p_full[pb]);
      }
      // -- epilogue: normalise, write the output or this CTA's part of it
      const uint32_t last = n_tile - 1;
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        const float x = warp_sum(sum[r]);  // idle lanes hold 0
        if (lane == 0) red[r0 + r] = x;
      }
      group_sync(bar_id);
      const bool whole = w.t0 == 0 && w.t1 == w.tiles;
      const int64_t slot = (int64_t)blockIdx.x + w.v;
      float inv[RH];
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        const float x = sred[r0 + r] + sred[R + r0 + r] + sred[2 * R + r0 + r] + sred[3 * R + r0 + r];
        inv[r] = x != 0.f ? 1.f / x : 0.f;
        if (!whole && quad == 0 && lane == 0 && r0 + r < nrow)
          p.part_lse[slot * p.rows_tile + r0 + r] = x != 0.f ? sreft[r0 + r] + log2f(x) : -INFINITY;
      }
      wait(&pv_done[last & 1], last >> 1, tc::kTimeoutTmemEmpty);
      for (int k = 0; k < p.boxes; ++k) {
        float v[RH];
#pragma unroll
        for (int r = 0; r < RH; r += 4) tmem_ld4(tmem + lanes + (uint32_t)(k * S::NP + r0 + r), v + r);
        tmem_wait_ld();
        const int l = k * 128 + quad * 32 + lane;
        if (l < width) {
#pragma unroll
          for (int r = 0; r < RH; ++r) {
            if (r0 + r >= nrow) continue;
            // inv == 0: no key (the accumulator may hold a stale column); references are finite otherwise
            const float o = inv[r] == 0.f ? 0.f : scale2(v[r], sref[r0 + r] - sreft[r0 + r]) * inv[r];
            if (whole)
              static_cast<T*>(p.a.out)[((int64_t)b * p.rows + row0 + r0 + r) * width + l] = from_f<T>(o);
            else
              p.part_o[(slot * p.rows_tile + r0 + r) * width + l] = o;
          }
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      asm volatile("bar.sync 3, 256;\n" ::: "memory");  // references and query rows are rewritten next
      ++w.v;
    }
    if (p.direct && swalk[2] == 0) {  // a pair without a key
      const int b = blockIdx.x / p.row_tiles, row0 = (blockIdx.x - b * p.row_tiles) * p.rows_tile;
      const int64_t n = (int64_t)min(p.rows_tile, p.rows - row0) * width;
      T* out = static_cast<T*>(p.a.out) + ((int64_t)b * p.rows + row0) * width;
      for (int64_t i = tid - 64; i < n; i += 256) out[i] = from_f<T>(0.f);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_relinquish();
    tc::tmem_dealloc(tmem, p.tmem);
  }
}

// Joins the CTAs of a pair: weights 2^(lse_c - max).  A pair inside one CTA is already written.
template <typename T>
__global__ void __launch_bounds__(256) attn_tc_join_kernel(const __grid_constant__ TcParams p) {
  const int v = blockIdx.x / p.rows_tile, r = blockIdx.x - v * p.rows_tile;
  const int b = v / p.row_tiles, row0 = (v - b * p.row_tiles) * p.rows_tile, width = p.a.cache.width;
  if (row0 + r >= p.rows) return;
  const int pairs = p.a.batch * p.row_tiles, per = p.prefix[pairs + 1];
  const int at = p.prefix[v], n = p.prefix[v + 1] - at;
  const int c0 = n > 0 ? at / per : 0, c1 = n > 0 ? (at + n - 1) / per : -1;
  if (n > 0 && c0 == c1) return;
  float m = -INFINITY;
  for (int c = c0; c <= c1; ++c) m = fmaxf(m, p.part_lse[((int64_t)c + v) * p.rows_tile + r]);
  const float base = m == -INFINITY ? 0.f : m;
  for (int l = blockIdx.y * 256 + threadIdx.x; l < width; l += gridDim.y * 256) {
    float acc = 0.f, sum = 0.f;
    for (int c = c0; c <= c1; ++c) {
      const int64_t i = ((int64_t)c + v) * p.rows_tile + r;
      const float f = exp2f(p.part_lse[i] - base);
      sum += f;
      acc += f * p.part_o[i * width + l];
    }
    static_cast<T*>(p.a.out)[((int64_t)b * p.rows + row0 + r) * width + l] = from_f<T>(sum != 0.f ? acc / sum : 0.f);
  }
}

template <int RH, int QP>
bool fit(int boxes, Plan* pl) {
  using S = Shape<RH, QP>;
  const int o_cols = boxes * S::NP;
  const int bufs = o_cols + 2 * S::NS <= 512 ? 2 : o_cols + S::NS <= 512 ? 1 : 0;
  const size_t fixed = (size_t)boxes * S::NS * 128 + 2 * S::P_BYTES + (3 + 8 + 1) * S::R * 4 + (2 * kMaxSlots + 10) * 8 + 64 + 1024;
  if (!bufs || fixed >= kSmemMax) return false;
  int slots = (int)((kSmemMax - fixed) / kBox);
  slots = slots < kMaxSlots ? slots : kMaxSlots;
  if (slots < boxes + 2) return false;  // a tile and something to load meanwhile
  pl->rh = RH;
  pl->boxes = boxes;
  pl->slots = slots;
  pl->s_bufs = bufs;
  pl->ahead = slots - boxes < boxes ? slots - boxes : boxes;
  uint32_t cols = 32;
  while (cols < (uint32_t)(o_cols + bufs * S::NS)) cols *= 2;
  pl->tmem = cols;
  pl->smem = fixed + (size_t)slots * kBox;
  return true;
}

// Rows of a CTA: the fewest padded rows that hold them all, else as many as fit TMEM and shared memory
// (the cache is then read once per row tile, mostly from L2).
template <int QP>
bool make_plan(const MlaCacheAttnArgs& a, Plan* pl) {
  const int boxes = (a.cache.width + 127) / 128, rows = a.queries * a.heads;
  Plan best;
#define KIMI_MLAC_FIT(RH)                                   \
  if (best.rh == 0 || 2 * best.rh < rows) {                  \
    Plan c;                                                  \
    if (fit<RH, QP>(boxes, &c)) best = c;                    \
  }
  KIMI_MLAC_FIT(4)
  KIMI_MLAC_FIT(8)
  KIMI_MLAC_FIT(12)
  KIMI_MLAC_FIT(16)
  KIMI_MLAC_FIT(24)
#undef KIMI_MLAC_FIT
  if (best.rh == 0) return false;
  *pl = best;
  pl->row_tiles = (rows + 2 * best.rh - 1) / (2 * best.rh);
  pl->rows_tile = (rows + pl->row_tiles - 1) / pl->row_tiles;
  const int64_t pairs = (int64_t)a.batch * pl->row_tiles, tiles = (a.cache.slots + kTile - 1) / kTile;
  if (pairs > (1 << 20) || pairs * tiles > (1 << 30)) return false;
  const int sms = device_sms();
  pl->direct = tiles == 1;
  pl->grid = pl->direct ? (int)pairs : (int)(pairs * tiles < sms ? pairs * tiles : sms);
  return true;
}

bool plan_for(int dtype, const MlaCacheAttnArgs& a, Plan* pl) {
  return dtype == 1 ? make_plan<2>(a, pl) : make_plan<3>(a, pl);
}

bool make_map(CUtensorMap* m, const MlaCacheAttnArgs& a, bool t_first, bool one) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  if (!fn) return false;
  const cuuint64_t nb = one ? 1 : a.batch, sb = one ? (cuuint64_t)a.cache.code_t * a.cache.slots : a.cache.code_b;
  cuuint64_t dims[3] = {(cuuint64_t)a.cache.width, t_first ? (cuuint64_t)a.cache.slots : nb,
                        t_first ? nb : (cuuint64_t)a.cache.slots};
  cuuint64_t strides[2] = {t_first ? (cuuint64_t)a.cache.code_t : sb, t_first ? sb : (cuuint64_t)a.cache.code_t};
  cuuint32_t box[3] = {128, t_first ? (cuuint32_t)kTile : 1u, t_first ? 1u : (cuuint32_t)kTile};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, a.cache.codes, dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

__device__ int g_mla_cache_status = 0;
std::mutex g_status_mutex;
int* g_status_addr[64] = {};  // device address of g_mla_cache_status, per device

int* status_ptr() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  std::lock_guard<std::mutex> lock(g_status_mutex);
  if (!g_status_addr[dev]) {
    void* q = nullptr;
    if (cudaGetSymbolAddress(&q, g_mla_cache_status) != cudaSuccess) return nullptr;
    g_status_addr[dev] = static_cast<int*>(q);
  }
  return g_status_addr[dev];
}

template <typename T, int RH, int QP>
cudaError_t launch(const TcParams& p, const Plan& pl, cudaStream_t s) {
  auto kern = attn_tc_kernel<T, RH, QP>;
  cudaError_t e = ensure_dynamic_smem(kern, (int)pl.smem);
  if (e != cudaSuccess) return e;
  kern<<<pl.grid, kThreads, pl.smem, s>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess || pl.direct) return e;
  const int pairs = p.a.batch * p.row_tiles;
  attn_tc_join_kernel<T><<<dim3((unsigned)(pairs * p.rows_tile), (p.a.cache.width + 255) / 256), 256, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int QP>
cudaError_t launch_rh(const TcParams& p, const Plan& pl, cudaStream_t s) {
  switch (pl.rh) {
    case 4: return launch<T, 4, QP>(p, pl, s);
    case 8: return launch<T, 8, QP>(p, pl, s);
    case 12: return launch<T, 12, QP>(p, pl, s);
    case 16: return launch<T, 16, QP>(p, pl, s);
    case 24: return launch<T, 24, QP>(p, pl, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

// 16-bit queries, and code rows that TMA can address: 16-byte base and strides.
bool mla_attn_tc_supported(int dtype, const MlaCacheAttnArgs& a) {
  if (dtype != 1 && dtype != 2) return false;
  if (a.cache.width % 16 || a.cache.width < 64 || a.cache.slots > (1 << 30)) return false;
  if ((reinterpret_cast<uintptr_t>(a.cache.codes) & 15) || (a.batch > 1 && a.cache.code_b % 16)) return false;
  if (a.cache.slots > 1 && (a.cache.code_t % 16 || a.cache.code_t < a.cache.width)) return false;
  Plan pl;
  return plan_for(dtype, a, &pl);
}

int64_t mla_attn_tc_workspace(int dtype, const MlaCacheAttnArgs& a) {
  Plan pl;
  if (!plan_for(dtype, a, &pl) || pl.direct) return 0;
  const int64_t pairs = (int64_t)a.batch * pl.row_tiles;
  return (pl.grid + pairs) * pl.rows_tile * (a.cache.width + 1) + pairs + 2;
}

cudaError_t mla_attn_tc(int dtype, const MlaCacheAttnArgs& a, cudaStream_t s) {
  Plan pl;
  if (!plan_for(dtype, a, &pl)) return cudaErrorInvalidValue;
  TcParams p{};
  p.a = a;
  if (a.cache.slots == 1) p.a.cache.code_t = a.cache.width;  // the stride of a lone slot says nothing
  p.rows = a.queries * a.heads;
  p.rows_tile = pl.rows_tile;
  p.row_tiles = pl.row_tiles;
  p.boxes = pl.boxes;
  p.slots = pl.slots;
  p.s_bufs = pl.s_bufs;
  p.ahead = pl.ahead;
  p.direct = pl.direct ? 1 : 0;
  p.min_tiles = 1;
  p.tmem = pl.tmem;
  const bool one = a.batch == 1 || a.cache.code_b == 0;  // every sequence reads the same rows
  p.z_mul = one ? 0 : 1;
  p.t_first = one || p.a.cache.code_t <= a.cache.code_b ? 1 : 0;
  // the encoder needs the device's context on this host thread
  static thread_local bool bound = false;
  if (!bound) {
    (void)cudaFree(nullptr);
    bound = true;
  }
  if (!make_map(&p.map, p.a, p.t_first, one)) return cudaErrorInvalidValue;
  const int64_t pairs = (int64_t)a.batch * pl.row_tiles, units = pl.direct ? 0 : (pl.grid + pairs) * pl.rows_tile;
  p.part_o = a.part_acc;
  p.part_lse = a.part_acc + units * a.cache.width;
  p.prefix = reinterpret_cast<int*>(p.part_lse + units);
  p.status = status_ptr();
  if (!p.status) return cudaErrorInvalidValue;
  return dtype == 1 ? launch_rh<__nv_bfloat16, 2>(p, pl, s) : launch_rh<__half, 3>(p, pl, s);
}

int* mla_cache_default_status() { return status_ptr(); }

int mla_cache_status(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_mla_cache_status, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_mla_cache_status, &zero, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

}  // namespace kimi
