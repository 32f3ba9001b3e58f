// Attention over the 8-bit MLA latent cache on tcgen05 (sm_100a).
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
// Splitting into 8-bit parts keeps the query type's accuracy.  A query row is scaled by a power of two to
// [128, 256) and written as q = q0 + q1 / 32 + q2 / 1024 + .. in e4m3, each part the rounding of what the
// one before left (5 bits a part): two parts hold every bf16 and three every fp16 but for what lies more than
// 2^-18, 2^-27 below the row's maximum.  The parts sit side by side on N (A is
// read once) and are added in fp32.  The weights v = 2^(s + log2(scale_t) - ref) <= 2^15 are split into
// e5m2 parts (3 + 4 + 4 + .. bits), all added up in fp32: three for bf16 outputs (11 bits), four for fp16
// (14).  e5m2 because of its range: it ends at 2^-16, so all 11 bits of a weight are there
// down to 2^-20 of the largest possible, where e4m3's step of 2^-9 would cut what many small weights add up to.
//
// fp32 queries do not come here.  With more parts (five of the query, six of a weight) the operands hold fp32, but the
// tensor cores' own sums do not: 160 sequences of up to 200 tokens, 6 heads, width 1488, random queries and cache ended
// at 1.03 x 2^-16 of what was added up, where the fp32 FMAs of the other form end at 0.07 x 2^-16.
//
// The softmax reference of a row is a power of two that only moves when some weight would pass 2^15
// (then the row's accumulator columns are rescaled in TMEM, exactly); the sums use the scores alone
// with a reference of their own, so token scales far apart cost neither range nor accuracy.
//
// Work split: the tiles of all (sequence, row tile) pairs form one list, cut into equal contiguous
// ranges, one per CTA (more where they would be longer than a stretch, see kStretch), from the lengths on the device:
// ragged batches stay balanced and a launch (or
// a captured graph) needs no lengths on the host.  A range that has a whole pair writes its output; the
// others leave a normalised context and its log-sum, joined by a second kernel in a fixed order.
//
// Three launches, each started while the one before still runs (programmatic dependent launch): the
// query parts; the attention, each CTA of which finds its own range of the list; the join.  The query parts are written as
// the image of their shared-memory tile, so that a CTA brings in the next sequence's queries with one
// bulk copy while it still works on the last tile of this one.
//
// What bounds it.  One product reads its tile from shared memory once per run of weight parts, at 128 bytes a clock:
// with 24 rows of width 1536 a tile of 96 KB is written once, read once (with 72 KB of query parts) for the scores and
// three times (with 24 KB of weights each) for the context: by that count 4,980 clocks of 6,260 measured between moves of
// the accumulators (the counters show 56 % of the shared-memory and L1 throughput over the whole kernel, start, epilogue,
// moves and waits included); the rest is scores -> weights -> context one behind the other, since 72 KB of query parts
// leave a ring of one and a half tiles.  With 12 rows the count is 3,770 of 4,730.  64 x 4,608 tokens of width 1536 (453 MB)
// take 168 us for 24 heads, and 97 - 98 for 3 (4.7 TB/s, 71 % of the measured copy; this kernel alone 92.6 at 76 %): memory,
// through a ring of two tiles.  Under this load the GPU runs at its power limit.
// Short calls are three launches and one tile's latency: 13.3 - 13.8 us for one sequence of 257 tokens.
//
// Roles of an attention CTA (10 warps): warp 0 loads, warp 1 issues the MMAs, warps 2-9 are two groups
// of four that share the rows: scores -> weights, rescaling and the epilogue.
// Every mbarrier wait is bounded and reports through the status word.  What a CTA had in hand when one gave up is written as
// NaN, and so is everything while the word stays set.
#include <cudaTypedefs.h>

#include <algorithm>
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
constexpr int kMaxStages = 32;             // of the ring
// Tiles ahead that are brought into L2 (the ring holds one and a half at width 1536).  0 / 1, back to back, 64 x 4,608,
// width 1536: 24 heads 150.7 / 142.7 us, 12 heads 122.3 / 108.8, 3 heads 87.3 / 83.6.
constexpr int kFetch = 1;
// Boxes of a ring stage, at most: a wide stage reads long pieces of each cached row together.  3 / 4 / 8 boxes: 64 x 6,144,
// 16 heads, width 1024 103.0 / 92.9 / 86.1 us; 64 x 4,096, 10 heads, width 640 (five boxes) 56.8 / 56.8 / 49.5.
constexpr int kMaxGroup = 8;
constexpr int kSmemMax = 227 * 1024;
constexpr int kMaxGrid = 256;              // CTAs of the attention kernel
template <int SL>
constexpr int kJoinThreads = SL == 1 ? 128 : 256;
constexpr int kPrepThreads = 256;          // 8 elements of a query row each: widths up to 2,048
constexpr int kMisaligned = 9;             // status: shared memory off a 1,024-byte boundary
constexpr float kTop = 15.f;               // a weight may reach 2^kTop
// A new reference leaves the row's largest weight at 2^(kTop - kRoom), or down to half of that: each bit of room saves
// moves of the accumulators (a stall of the CTA) and raises the floor of the weights.  e5m2 ends in steps of 2^-16, so
// a weight is held to within 2^(kRoom - 31) of the largest, and what many small weights add up to may be lost from the
// context while the sum in the denominator has it.  kStretch bounds how many: each stretch of the cache this long
// starts with references of its own.  A stretch then loses 2^(kRoom - 31) * kStretch of its weights' sum at most:
// 2^-12 for bf16 with six bits, 2^-14 for fp16 with four, a sixteenth and an eighth of one unit of the type.
// bf16 with six bits / nine: 64 x 4,608, width 1536, 24 heads 168 / 156 us, 12 heads of ragged lengths 85.5 / 78.3;
// 8 x up to 2,048, 4 tokens of 12 heads, width 768 25.2 / 22.6.  fp16 with four / six: one sequence of 131,072, 16 heads,
// width 1024 57.7 / 55.7.
template <int QP>
constexpr float kRoom = QP == 2 ? 6.f : 4.f;
constexpr int kStretch = 8192 / kTile;     // tiles
constexpr float kNoRef = -3e38f;            // finite: a score of -inf weighs nothing against it
constexpr float kSumRoom = 40.f;           // the sums' reference may lag by this many bits

struct Plan {
  int rh = 0;          // rows of one compute group (template)
  int rows_tile = 0;   // rows of a pair (<= 2 * rh)
  int row_tiles = 0;
  int boxes = 0;       // boxes of a tile: ceil(L / 128)
  int group = 0;       // boxes of a ring stage: one wait, one release
  int tile_stages = 0;  // stages of a tile
  int stages = 0;      // of the ring
  int s_bufs = 0;
  int stack = 0;       // weight parts side by side on N
  int runs = 0;        // context products of a box: ceil(parts / stack)
  int ns = 0, np = 0;  // N of the score and of the context product
  int p_bytes = 0;     // one weight buffer
  int p_bufs = 2;
  uint32_t tmem = 0;
  size_t smem = 0;
  bool direct = false;  // one CTA per pair, nothing to join
  int grid = 0;
  int stretch = 0;      // places of a range at most
  int64_t ranges = 0;   // of the tile list, at most (see Walk)
};

struct TcParams {
  CUtensorMap map;
  MlaCacheAttnArgs a;
  int rows, rows_tile, row_tiles, boxes, group, tile_stages, stages, s_bufs, direct, t_first, q_vec;
  int wide;            // one copy per stage (L a multiple of 128), else one per box
  int fetch;           // tiles ahead that are brought into L2
  int r_pad, stack, runs, ns, np, p_bytes, p_bufs, q_bytes, grid;
  int part_c;          // numbers of parts that a range takes up (see part_of)
  int start;           // places of a pair in front of its tiles (see kStart)
  int stretch;         // places of a range at most (see kStretch)
  uint32_t tmem;
  int64_t z_mul;       // 0 when every sequence reads the same cache rows
  uint8_t* q_parts;    // [pairs][q_bytes]: the shared-memory image of a pair's query parts
  float* coef;         // [pairs][R] score factors
  float* part_o;       // [ranges + min(ranges, pairs)][rows_tile][L]
  float* part_lse;     // [ranges + min(ranges, pairs)][rows_tile]
  int* prefix;         // [pairs + 2]: first place of each pair, total, places of a range
  int* status;
};

constexpr int pad16(int n) { return (n + 15) / 16 * 16; }
// QP parts of a query row; QP + 1 parts of a weight.
template <int RH, int QP>
struct Shape {
  static constexpr int R = 2 * RH;          // rows, padded
  static constexpr int NS = pad16(QP * R);  // N of the score product
  static constexpr int WP = QP + 1;
  static constexpr int MAX_STACK = RH <= 8 ? WP : RH <= 12 ? 3 : 2;  // registers of the epilogue
};

KIMI_D bool elect_one() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e != 0;
}
// Descriptors as (low, high) words: a step along a tile only moves the low word's address field.
KIMI_D void mma_f8(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                   uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n mov.b64 a, {%1, %2};\n mov.b64 b, {%3, %4};\n setp.ne.b32 p, %6, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %5, p;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
KIMI_D void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                   tc::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
               : "memory");
}
// All boxes of a stage in one copy: tokens y.., 128-latent chunks c.. of sequence b; and the same into L2 only.
KIMI_D void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int y, int c, int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];\n" ::"r"(tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(y), "r"(c), "r"(b), "r"(tc::smem_u32(bar))
      : "memory");
}
KIMI_D void tma_prefetch_4d(const CUtensorMap* map, int y, int c, int b) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];\n" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(0), "r"(y), "r"(c), "r"(b)
               : "memory");
}
// Whether the phase of this parity is over; does not block.
KIMI_D bool mbar_over(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(tc::smem_u32(bar)), "r"(parity & 1)
      : "memory");
  return done != 0;
}
// Programmatic dependent launch: let the next kernel of the stream start / wait for the one before.
KIMI_D void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
KIMI_D void pdl_wait() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
// kind::f8f6f4 instruction descriptor: fp32 accumulator, A e4m3 (0), B e4m3 (0) or e5m2 (1).
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n, bool a_mn, bool b_e5m2) {
  return (1u << 4) | ((b_e5m2 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
// N consecutive columns (a multiple of 4) of this warp's 32 lanes; complete after tmem_wait_ld.
template <int N>
KIMI_D void tmem_ldn(uint32_t addr, float* v) {
  if constexpr (N >= 8) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
    if constexpr (N > 8) tmem_ldn<N - 8>(addr + 8, v + 8);
  } else {
    uint32_t r[4];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
  }
}
// N columns of lanes 0-15 for each half of the warp: threads 16-31 get the columns SPLIT further on.
template <int N, int SPLIT>
KIMI_D void tmem_ld_halves(uint32_t addr, float* v) {
  if constexpr (N == 2) {
    uint32_t r[2];
    asm volatile("tcgen05.ld.sync.aligned.16x32bx2.x2.b32 {%0,%1}, [%2], %3;\n"
                 : "=r"(r[0]), "=r"(r[1])
                 : "r"(addr), "n"(SPLIT));
    v[0] = __uint_as_float(r[0]);
    v[1] = __uint_as_float(r[1]);
  } else if constexpr (N == 4) {
    uint32_t r[4];
    asm volatile("tcgen05.ld.sync.aligned.16x32bx2.x4.b32 {%0,%1,%2,%3}, [%4], %5;\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(SPLIT));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
  } else {
    constexpr int H = N % 4 ? N - 2 : N - 4;
    tmem_ld_halves<H, SPLIT>(addr, v);
    tmem_ld_halves<N - H, SPLIT>(addr + H, v + H);
  }
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
// The .aligned instructions of the compute groups want whole converged warps: each is behind a __syncwarp
// where a lane-dependent branch comes before it.
KIMI_D void group_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, 128;\n" ::"r"(id) : "memory");
}
KIMI_D bool group_any(int id, bool v) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n bar.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(id), "r"(v ? 1u : 0u)
      : "memory");
  return r != 0;
}
KIMI_D float pow2i(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }
// 2^e as two factors, for any integer-valued e: their product is applied one at a time.
KIMI_D float2 pow2_pair(float e) {
  const int n = (int)fminf(fmaxf(e, -250.f), 250.f), h = n / 2;
  return make_float2(pow2i(h), pow2i(n - h));
}
KIMI_D float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
KIMI_D float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// Maximum over the 16 lanes of this half of the warp.
KIMI_D float half_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
KIMI_D float half_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
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
  int64_t len;
  const int64_t start = first_position(p.a, b, &len);
  len = len < 0 ? 0 : len > p.a.cache.slots ? p.a.cache.slots : len;
  const int last = min(p.rows, (rt + 1) * p.rows_tile) - 1;
  const int64_t seen = start + last / p.a.heads + 1;
  const int64_t lim = seen < 0 ? 0 : seen < len ? seen : len;
  *len_out = len;
  *start_out = start;
  return (int)((lim + kTile - 1) / kTile);
}

// The list of all pairs' tiles is cut into equal ranges, one per CTA, or several one behind the other where one would
// be longer than a stretch.  Starting a pair costs a CTA about as
// much as kStart tiles (an epilogue, an empty pipeline), so each pair with tiles has kStart places in front;
// none where every tile can have its own CTA.  0 / 2 / 4, 64 x 4,608, width 1536: 24 heads 147 / 143 / 142 us,
// 12 heads 112 / 109 / 112, 3 heads 85.4 / 83.8 / 85.4.
constexpr int kStart = 2;

// This CTA's share of the list, walked segment by segment (every role walks it on its own).
struct Share {
  int v, t;        // the first pair and tile
  int place, end;  // their place in the list, and where the CTA's ranges end
  int per;         // places of a range
};
struct Walk {
  int v, place;  // pair, place in the list behind the segment
  int t0, t1;    // the segment: tiles [t0, t1) of the pair
  int range;     // that the segment lies in; -1 when it is the whole pair
  int64_t len, start;
  KIMI_D explicit Walk(const Share& s) : v(s.v), place(s.place), t0(0), t1(s.t), range(0), len(0), start(0) {}
  KIMI_D bool next(const TcParams& p, const Share& s, int pairs) {
    while (place < s.end && v < pairs) {
      const int tiles = pair_tiles(p, v, &len, &start);
      if (t1 < tiles) {
        t0 = t1;
        range = place / s.per;
        t1 = min(tiles, t0 + min(s.end, (range + 1) * s.per) - place);
        place += t1 - t0 + (t1 == tiles ? p.start : 0);  // the next pair's places in front
        if (t1 - t0 == tiles) range = -1;
        return true;
      }
      ++v;  // no tiles (left)
      t1 = 0;
    }
    return false;
  }
};

// Number of the part that range c holds of a pair v that it does not hold whole.  A range holds one such part that does not
// start the pair, its first, and one that does, its last: two numbers a range, or, where the pairs are fewer, c + v.
KIMI_D int64_t part_of(const TcParams& p, int c, int v, bool starts) {
  return p.part_c == 1 ? (int64_t)c + v : 2 * (int64_t)c + (starts ? 1 : 0);
}

template <typename T>
struct alignas(16) Oct8 {
  T v[8];
};

// Query parts, one block per row and one thread per 8 elements.  64 x 24 rows of 1,536 in bf16 (4.7 MB in, 4.7 MB
// out) take 4.4 us, most of it a launch, one trip to memory and one back; a warp per row took 5.6, its long code
// fetched cold, and the attention kernel gets its SMs only behind it.
template <typename T, int QP>
__global__ void __launch_bounds__(kPrepThreads) attn_tc_prep_kernel(const __grid_constant__ TcParams p) {
  __shared__ uint32_t stop[kPrepThreads / 32];
  const int o = threadIdx.x, warp = o >> 5, R = p.r_pad, NS = p.ns;
  const int v = blockIdx.x / p.rows_tile, r = blockIdx.x - v * p.rows_tile;
  const int b = v / p.row_tiles, qr = (v - b * p.row_tiles) * p.rows_tile + r;
  const int qi = qr / p.a.heads, h = qr - qi * p.a.heads;
  pdl_wait();
  // only now: the attention kernel reads cache and lengths without waiting for this one to end, so it may
  // not start before everything ahead of this kernel is done
  pdl_launch();
  if (qr >= p.rows) return;
  const T* q = static_cast<const T*>(p.a.q) + b * p.a.q_b + qi * p.a.q_i + h * p.a.q_h + o * 8;
  Oct8<T> x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x.v[j] = from_f<T>(0.f);
  if (o < p.a.cache.width >> 3) {
    if (p.q_vec) {
      *reinterpret_cast<int4*>(x.v) = __ldg(reinterpret_cast<const int4*>(q));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x.v[j] = q[j];
    }
  }
  uint32_t top = 0;  // of the magnitudes' bits, which order like the values; infinities and NaN on top
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(to_f<T>(x.v[j])) & 0x7FFFFFFFu);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((o & 31) == 0) stop[warp] = top;
  __syncthreads();
  for (int i = 0; i < (int)blockDim.x / 32; ++i) top = max(top, stop[i]);
  const bool bad = top >= 0x7F800000u;
  const int k = bad ? 0 : min(126, 134 - (int)(top >> 23));  // the maximum to [128, 256)
  const float f = pow2i(k);
  if (o < p.boxes * 16) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = bad ? 0.f : to_f<T>(x.v[j]) * f;
    uint8_t* at = p.q_parts + (int64_t)v * p.q_bytes + (size_t)(o >> 4) * NS * 128 + (o & 1) * 8;
#pragma unroll
    for (int part = 0; part < QP; ++part) {
      const int n = part * R + r;
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[j] = to_codes2(y[2 * j], y[2 * j + 1]);
        const float2 d = codes2(c[j]);
        y[2 * j] = (y[2 * j] - d.x) * 32.f;
        y[2 * j + 1] = (y[2 * j + 1] - d.y) * 32.f;
      }
      *reinterpret_cast<uint2*>(at + (n >> 3) * 1024 + (n & 7) * 128 + ((((o >> 1) & 7) ^ (n & 7)) << 4)) =
          make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
    }
  }
  if (o == 0) p.coef[v * R + r] = bad ? __uint_as_float(0x7FC00000u) : p.a.scale * kLog2e * pow2i(-k);
}

template <typename T, int RH, int QP>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ TcParams p) {
  using S = Shape<RH, QP>;
  constexpr int R = S::R, HR = RH / 2;  // a thread of a compute group handles HR rows of one token
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = smem_raw;                                   // [stages][group][kBox]
  if (tc::smem_u32(smem_raw) & 1023u) {  // the swizzle needs it; no static shared memory is in front
    if (threadIdx.x == 0) atomicCAS(p.status, 0, kMisaligned);
    return;
  }
  uint8_t* sq = ring + (size_t)p.stages * p.group * kBox;     // [boxes][NS][128] query parts
  uint8_t* sp = sq + p.q_bytes;                               // [p_bufs][p_bytes] weight parts
  float2* sfac = reinterpret_cast<float2*>(sp + p.p_bufs * p.p_bytes);  // [R] normalisation of a row
  float* sref = reinterpret_cast<float*>(sfac + R);           // [R] weight references
  float* sreft = sref + R;                                    // [R] sum references
  float* sdel = sreft + R;                                    // [R] change of a weight reference
  float* smul = sdel + R;                                     // [R] factor of a sum
  float* sred = smul + R;                                     // [2 kinds][4 warps][R]
  uint64_t* full = reinterpret_cast<uint64_t*>(sred + 8 * R);
  uint64_t* empty = full + kMaxStages;
  uint64_t* s_full = empty + kMaxStages;
  uint64_t* s_empty = s_full + 2;
  uint64_t* p_full = s_empty + 2;
  uint64_t* pv_done = p_full + 2;
  uint64_t* q_full = pv_done + 2;
  uint64_t* drain = q_full + 1;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
  Share& share = *reinterpret_cast<Share*>(tslot + 1);
  int* swsum = reinterpret_cast<int*>(&share + 1);            // [10] tiles counted by each warp
  volatile int* svoid = swsum + kThreads / 32;                // a wait has given up: what this CTA has is void

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pairs = p.a.batch * p.row_tiles;
  const int width = p.a.cache.width;

  // ---- set-up: barriers, TMEM, this CTA's share of the tiles
  if (warp == 1) tc::tmem_alloc(tslot, p.tmem);
  if (tid < p.stages) {
    tc::mbar_init(&full[tid], 1);
    tc::mbar_init(&empty[tid], 1);
  }
  if (tid >= 64 && tid < 66) {
    tc::mbar_init(&s_full[tid - 64], 1);
    tc::mbar_init(&s_empty[tid - 64], 8);
    tc::mbar_init(&p_full[tid - 64], 8);
    tc::mbar_init(&pv_done[tid - 64], 1);
  }
  // a record that nobody has cleared: every wait would give up, so nothing is started
  if (tid == 128) *svoid = tc::status_peek(p.status);
  if (tid == 96) {
    tc::mbar_init(q_full, 1);
    tc::mbar_init(drain, 1);
    tc::tma_prefetch(&p.map);
  }
  // a context product may read weight parts that no row has: zeros (warps 0 and 1 have other things to do)
  for (int i = tid - 64; i >= 0 && i < p.p_bufs * p.p_bytes / 16; i += kThreads - 64)
    reinterpret_cast<int4*>(sp)[i] = make_int4(0, 0, 0, 0);
  tc::fence_barrier_init();
  tc::fence_proxy_async();
  pdl_launch();
  if (p.direct) {
    int64_t len, start;
    if (tid == 0) {
      const int n = pair_tiles(p, blockIdx.x, &len, &start);
      share = {(int)blockIdx.x, 0, 0, n, max(n, 1)};  // all of it
    }
  } else {
    // Every thread counts the tiles of a run of pairs; a block scan places the runs in the tile list.
    int64_t len, start;
    const int run = (pairs + kThreads - 1) / kThreads, v0 = min(tid * run, pairs), v1 = min(v0 + run, pairs);
    int own = 0, last = 0;
    for (int v = v0; v < v1; ++v) {
      last = pair_tiles(p, v, &len, &start);
      own += last > 0 ? last + p.start : 0;
    }
    __syncwarp();
    int incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) swsum[warp] = incl;
    if (tid == 0) share = {pairs, 0, 0, 0, 1};
    __syncthreads();
    int at = incl - own, total = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) at += swsum[i];
      total += swsum[i];
    }
    // as many ranges for each CTA as keep its segments within a stretch; < 2^31: the host bounds the tiles
    int per = (total + p.grid - 1) / p.grid, ranges = 1;
    if (per > p.stretch) {
      ranges = (per - 1) / p.stretch + 1;
      per = (per - 1) / ranges + 1;
    }
    const int mine = (int)blockIdx.x * ranges * per, end = mine + ranges * per;
    if (blockIdx.x == 0 || (mine >= at && mine < at + own)) {
      for (int v = v0; v < v1; ++v) {
        const int n = run == 1 ? last : pair_tiles(p, v, &len, &start), places = n > 0 ? n + p.start : 0;
        if (blockIdx.x == 0) p.prefix[v] = at;
        if (mine >= at && mine < at + places) {
          const int place = max(mine, at + p.start);
          share = {v, place - at - p.start, place, end, per};
        }
        at += places;
      }
    }
    if (blockIdx.x == 0 && tid == 0) {
      p.prefix[pairs] = total;
      p.prefix[pairs + 1] = max(per, 1);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tslot;
  const uint32_t tm_s = tmem + (uint32_t)(p.boxes * p.np);  // score buffers behind the accumulators
  Walk w(share);
  const bool idle = *svoid != 0;

  if (warp == 0) {
    // ---- loads
    if (!idle && elect_one()) {
      bool ok = true;
      uint32_t n = 0;  // stages loaded so far
      int st = 0;
      uint32_t ph = 1;  // parity of the last release of stage `st` before this use
      while (ok && w.next(p, share, pairs)) {
        const int zb = (int)((w.v / p.row_tiles) * p.z_mul);
        for (int t = w.t0; ok && t < w.t1; ++t) {
          const bool fetch = p.fetch > 0 && t + p.fetch < w.t1;
          for (int k = 0; k < p.boxes; k += p.group, ++n) {
            if (n >= (uint32_t)p.stages && !tc::mbar_wait(&empty[st], ph, p.status, tc::kTimeoutEmpty)) {
              ok = false;
              break;
            }
            uint8_t* dst = ring + (size_t)(st * p.group) * kBox;
            if (p.wide) {  // chunks past the latent axis are filled with zeros and count
              tc::mbar_arrive_expect_tx(&full[st], p.group * kBox);
              tma_load_4d(dst, &p.map, &full[st], t * kTile, k, zb);
              if (fetch) tma_prefetch_4d(&p.map, (t + p.fetch) * kTile, k, zb);
            } else {
              const int nb = min(p.group, p.boxes - k);
              tc::mbar_arrive_expect_tx(&full[st], nb * kBox);
              const int y = p.t_first ? t * kTile : zb, z = p.t_first ? zb : t * kTile;
              for (int i = 0; i < nb; ++i) tc::tma_load_3d(dst + i * kBox, &p.map, &full[st], (k + i) * 128, y, z);
            }
            if (++st == p.stages) {
              st = 0;
              ph ^= 1;
            }
          }
        }
      }
      // copies in flight land before the CTA ends
      for (uint32_t i = n > (uint32_t)p.stages ? n - p.stages : 0; i < n; ++i)
        tc::mbar_wait_local(&full[i % p.stages], (i / p.stages) & 1, p.status, tc::kTimeoutDrain, tc::kDrainNs);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMAs.  Issued under elect.sync with descriptors that are sums of precomputed words, an MMA costs
    // what the tensor core takes (28 clocks for a score step of 48 columns, 40 for a context step); behind
    // a plain lane test the issue alone took 90 to 170.
    if (!idle && elect_one()) {
      // Two streams over the same tiles, scores and context, each taken as soon as its operands are there:
      // a context product goes first (it frees its tile's part of the ring), else the next stage of scores.
      int s_st = 0, o_st = 0, s_i = 0;  // ring stages of the streams; stage of the score tile
      uint32_t s_ph = 0, s_n = 0, o_n = 0, s_seg = 0, polls = 0;  // tiles and segments so far
      bool s_open = false;
      const uint32_t id_s = idesc_f8(64, S::NS, false, false), id_o = idesc_f8(128, p.np, true, true);
      const uint64_t ad_k = tc::smem_desc_sw128(tc::smem_u32(ring), 16, 1024);
      const uint64_t ad_mn = tc::smem_desc_sw128(tc::smem_u32(ring), 8192, 1024);
      const uint64_t bd_q = tc::smem_desc_sw128(tc::smem_u32(sq), 16, 1024);
      const uint64_t bd_p = tc::smem_desc_sw128(tc::smem_u32(sp), 16, 1024);
      const uint32_t k_hi = (uint32_t)(ad_k >> 32), mn_hi = (uint32_t)(ad_mn >> 32), q_hi = (uint32_t)(bd_q >> 32),
                     p_hi = (uint32_t)(bd_p >> 32);
      const uint32_t stage16 = (uint32_t)(p.group * (kBox >> 4));
      Walk ws = w, wo = w;
      bool s_have = ws.next(p, share, pairs), o_have = wo.next(p, share, pairs);
      int s_t = ws.t0, o_t = wo.t0;
      uint64_t since = 0;
      while (o_have) {
        const uint32_t pb = o_n & 1;
        if (mbar_over(&p_full[pb], o_n >> 1)) {
          tc::tc_fence_after();
          const uint32_t pd = (uint32_t)bd_p + (p.p_bufs == 2 ? pb : 0) * (uint32_t)(p.p_bytes >> 4);
          uint32_t d = tmem;
          for (int i = 0; i < p.tile_stages; ++i) {
            const int nb = min(p.group, p.boxes - i * p.group);
            uint32_t a = (uint32_t)ad_mn + o_st * stage16;
            for (int k = 0; k < nb; ++k, a += kBox >> 4, d += p.np) {
              mma_f8(d, a, mn_hi, pd, p_hi, id_o, o_t > wo.t0 ? 1u : 0u);
              mma_f8(d, a + (4096 >> 4), mn_hi, pd + 2, p_hi, id_o, 1u);
              for (int run = 1; run < p.runs; ++run) {
                const uint32_t pr = pd + (uint32_t)((run >> 1) * p.np * 8 + (run & 1) * 4);
                mma_f8(d, a, mn_hi, pr, p_hi, id_o, 1u);
                mma_f8(d, a + (4096 >> 4), mn_hi, pr + 2, p_hi, id_o, 1u);
              }
            }
            tc::mma_commit(&empty[o_st]);
            if (++o_st == p.stages) o_st = 0;
          }
          tc::mma_commit(&pv_done[pb]);
          ++o_n;
          if (++o_t == wo.t1) {
            o_have = wo.next(p, share, pairs);
            o_t = wo.t0;
          }
          polls = 0;
          continue;
        }
        if (s_have) {
          const uint32_t buf = p.s_bufs == 2 ? s_n & 1 : 0, use = p.s_bufs == 2 ? s_n >> 1 : s_n;
          if (!s_open && (use == 0 || mbar_over(&s_empty[buf], use - 1)) && (s_t > ws.t0 || mbar_over(q_full, s_seg)))
            s_open = true;
          if (s_open && mbar_over(&full[s_st], s_ph)) {
            tc::tc_fence_after();
            const uint32_t d = tm_s + buf * S::NS;
            const int k0 = s_i * p.group, nb = min(p.group, p.boxes - k0);
            uint32_t a = (uint32_t)ad_k + s_st * stage16, q = (uint32_t)bd_q + k0 * (S::NS * 8);
            for (int k = 0; k < nb; ++k, a += kBox >> 4, q += S::NS * 8) {
#pragma unroll
              for (int j = 0; j < 4; ++j) mma_f8(d, a + 2 * j, k_hi, q + 2 * j, q_hi, id_s, (s_i | k | j) != 0);
            }
            if (++s_st == p.stages) {
              s_st = 0;
              s_ph ^= 1;
            }
            if (++s_i == p.tile_stages) {
              tc::mma_commit(&s_full[buf]);
              s_i = 0;
              s_open = false;
              ++s_n;
              if (++s_t == ws.t1) {
                s_have = ws.next(p, share, pairs);
                s_t = ws.t0;
                ++s_seg;
              }
            }
            polls = 0;
            continue;
          }
        }
        if ((++polls & 1023u) == 0) {  // bounded like every wait
          if (tc::status_peek(p.status) != 0) break;
          const uint64_t now = tc::globaltimer_ns();
          if (polls == 1024) {
            since = now;
          } else if (now - since > tc::kWaitNs) {
            atomicCAS(p.status, 0, (int)tc::kTimeoutTmemFull);
            break;
          }
        }
      }
      tc::mma_commit(drain);
      tc::mbar_wait_local(drain, 0, p.status, tc::kTimeoutDrain, tc::kDrainNs);
    }
    __syncwarp();
  } else {
    // ---- compute groups: rows [grp * RH, grp * RH + RH) of the pair.  The score tile has M = 64: its tokens
    // lie in lanes 0-15 of each warp's quadrant, and the halves of a warp take half of the rows each.
    const int grp = (warp - 2) >> 2, quad = warp & 3, bar_id = 1 + grp;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int tok = quad * 16 + (lane & 15);
    const int r0 = grp * RH, rr = r0 + (lane >> 4) * HR;  // rows of the group and of this thread
    // weight parts: run `part / stack` takes 64 bytes of a 128-byte row, stacked parts take R rows each
    uint32_t part_at[S::WP], row_at[HR];
#pragma unroll
    for (int i = 0; i < S::WP; ++i) {
      const int run = i / p.stack, g = i - run * p.stack;
      part_at[i] = (uint32_t)((run >> 1) * p.np * 128 + g * R * 128) | ((run & 1) << 31);
    }
#pragma unroll
    for (int r = 0; r < HR; ++r) {
      const int n = rr + r;
      row_at[r] = (uint32_t)((n >> 3) * 1024 + (n & 7) * 128 + ((quad ^ (n & 7)) << 4) + (lane & 15));
    }
    // A wait that fails only makes this warp skip its later waits: every warp walks all tiles, so the
    // groups' named barriers always meet and the kernel ends (its results are NaN, and the status says so).
    bool ok = !idle;
    uint32_t n_tile = 0;
    int stage = 0;  // first stage of the tile
    auto wait = [&](uint64_t* bar, uint32_t use, int code) {  // the warp is converged again behind it, and agrees
      ok = __all_sync(0xffffffffu, ok && tc::mbar_wait(bar, use & 1, p.status, code));
      if (!ok) *svoid = 1;  // before this warp arrives anywhere
      tc::tc_fence_after();
    };
    // One copy at a time: the next is issued behind a wait that shows the one before to be read.
    uint32_t n_q = 0;  // warp 2: copies issued
    auto load_q = [&](int v) {
      tc::mbar_arrive_expect_tx(q_full, p.q_bytes);
      bulk_load(sq, p.q_parts + (int64_t)v * p.q_bytes, p.q_bytes, q_full);
    };
    pdl_wait();  // the query parts are there
    bool have = w.next(p, share, pairs);
    if (have && warp == 2 && ok) {
      if (elect_one()) load_q(w.v);
      ++n_q;
    }
    __syncwarp();
    while (have) {
      const int b = w.v / p.row_tiles, row0 = (w.v - b * p.row_tiles) * p.rows_tile;
      const int nrow = min(p.rows_tile, p.rows - row0);
      Walk nx = w;
      const bool more = nx.next(p, share, pairs);
      float coef[HR], ref[HR], reft[HR], sum[HR];
#pragma unroll
      for (int r = 0; r < HR; ++r) {
        coef[r] = rr + r < nrow ? p.coef[w.v * R + rr + r] : 0.f;
        ref[r] = reft[r] = kNoRef;
        sum[r] = 0.f;
      }
      if (quad == 0 && lane < RH) sref[r0 + lane] = sreft[r0 + lane] = kNoRef;
      auto keys = [&](int r) {  // keys that row r sees; rows come in the order of their positions
        const int64_t seen = w.start + 1 + (p.a.queries == 1 ? 0 : (row0 + min(r, nrow - 1)) / p.a.heads);
        return seen < 0 ? 0 : (int)(seen < w.len ? seen : w.len);
      };
      const int lim0 = keys(0);
      const float* scales = p.a.cache.scales + b * p.a.cache.scale_b;
      float st_next = w.t0 * kTile + tok < w.len ? scales[(w.t0 * kTile + tok) * p.a.cache.scale_t] : 0.f;
      for (int t = w.t0; t < w.t1; ++t, ++n_tile) {
        const int at = t * kTile + tok;
        const float st = st_next;
        const float lg = st < INFINITY ? lg2(st) : 0.f;  // a NaN stays in the scores of the rows that see it
        if (t + 1 < w.t1) st_next = at + kTile < w.len ? scales[(at + kTile) * p.a.cache.scale_t] : 0.f;
        const uint32_t buf = p.s_bufs == 2 ? n_tile & 1 : 0, pb = n_tile & 1;
        wait(&s_full[buf], p.s_bufs == 2 ? n_tile >> 1 : n_tile, tc::kTimeoutTmemFull);
        // this segment's score products are done: the next one's queries may come in
        if (t + 1 == w.t1 && more && warp == 2 && ok) {
          if (elect_one()) load_q(nx.v);
          ++n_q;
        }
        __syncwarp();
        float s[HR];
        {
          float v[QP][HR];
#pragma unroll
          for (int part = 0; part < QP; ++part)
            tmem_ld_halves<HR, HR>(tm_s + lanes + buf * S::NS + part * R + r0, v[part]);
          tmem_wait_ld();
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&s_empty[buf]);
#pragma unroll
          for (int r = 0; r < HR; ++r) {
            float x = v[QP - 1][r];
#pragma unroll
            for (int part = QP - 2; part >= 0; --part) x = fmaf(x, 0.03125f, v[part][r]);
            s[r] = x * (coef[r] * st);
          }
        }
        if ((t + 1) * kTile > lim0) {  // a tile that some row does not see whole
#pragma unroll
          for (int r = 0; r < HR; ++r)
            if (at >= keys(rr + r)) s[r] = -INFINITY;
          // slots past the length hold anything: their rows of the tile become zeros
          if ((int64_t)(t + 1) * kTile > w.len) {
            const int from = (int)(w.len - (int64_t)t * kTile), n = (kTile - from) * 8;
            for (int k = 0; k < p.boxes; ++k) {
              const int st_k = (stage + k / p.group) % p.stages;
              uint8_t* box = ring + (size_t)(st_k * p.group + k % p.group) * kBox + from * 128;
              for (int j = tid - 64; j < n; j += 256) reinterpret_cast<int4*>(box)[j] = make_int4(0, 0, 0, 0);
            }
          }
        }
        stage += p.tile_stages;
        if (stage >= p.stages) stage -= p.stages;
        float ev[HR], es[HR];  // log2 of the weights and of the sums' terms
        bool raise = false;
#pragma unroll
        for (int r = 0; r < HR; ++r) {
          ev[r] = s[r] + lg - ref[r];
          es[r] = s[r] - reft[r];
          raise |= ev[r] > kTop || es[r] > kSumRoom;
        }
        if (group_any(bar_id, raise)) {
          // some row outgrew a reference: new ones from the tile's maxima
#pragma unroll
          for (int r = 0; r < HR; ++r) {
            const float ma = half_max(s[r] + lg), ms = half_max(s[r]);
            if ((lane & 15) == 0) {
              sred[quad * R + rr + r] = ma;
              sred[(4 + quad) * R + rr + r] = ms;
            }
          }
          group_sync(bar_id);
          if (quad == 0 && lane < RH) {
            const int r = r0 + lane;
            const float ma = fmaxf(fmaxf(sred[r], sred[R + r]), fmaxf(sred[2 * R + r], sred[3 * R + r]));
            const float ms = fmaxf(fmaxf(sred[4 * R + r], sred[5 * R + r]), fmaxf(sred[6 * R + r], sred[7 * R + r]));
            float del = 0.f, mul = 1.f;
            if (ma > sref[r] + kTop) {
              const float to = ceilf(ma) - (kTop - kRoom<QP>);
              del = sref[r] - to;
              sref[r] = to;
            }
            if (ms > sreft[r] + kSumRoom) {
              const float to = ceilf(ms);
              mul = exp2f(sreft[r] - to);
              sreft[r] = to;
            }
            sdel[r] = del;
            smul[r] = mul;
          }
          group_sync(bar_id);
#pragma unroll
          for (int r = 0; r < HR; ++r) {
            sum[r] *= smul[rr + r];
            ref[r] = sref[rr + r];
            reft[r] = sreft[rr + r];
            ev[r] = s[r] + lg - ref[r];
            es[r] = s[r] - reft[r];
          }
          if (t > w.t0) {  // the accumulators hold something
            bool waited = false;
#pragma unroll 1
            for (int r = r0; r < r0 + RH; ++r) {
              const float del = sdel[r];
              if (del == 0.f) continue;  // uniform over the group
              if (!waited) wait(&pv_done[pb ^ 1], (n_tile - 1) >> 1, tc::kTimeoutTmemEmpty);
              waited = true;
              const float2 f = pow2_pair(del);
#pragma unroll 1
              for (int g = 0; g < p.stack; ++g) {
                const uint32_t c = tmem + lanes + (uint32_t)(g * R + r);
#pragma unroll 1
                for (int k = 0; k < p.boxes; k += 8) {
                  float v[8];
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    if (k + i < p.boxes) v[i] = tmem_ld1(c + (uint32_t)((k + i) * p.np));
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    if (k + i < p.boxes) tmem_st1(c + (uint32_t)((k + i) * p.np), v[i] * f.x * f.y);
                }
              }
            }
            if (waited) tmem_wait_st();
          }
        }
        // weights into parts; the buffer was last read by the context product of p_bufs tiles ago
        const uint32_t before = n_tile - p.p_bufs;
        if (n_tile >= (uint32_t)p.p_bufs) wait(&pv_done[before & 1], before >> 1, tc::kTimeoutTmemEmpty);
        uint8_t* wp = sp + (p.p_bufs == 2 ? pb : 0) * p.p_bytes;
#pragma unroll
        for (int r = 0; r < HR; r += 2) {
          float v[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sum[r + e] += ex2(es[r + e]);
            v[e] = ex2(ev[r + e]);
          }
          // an fp16 holds three parts; the one before them comes off in fp32
          __half2 h;
          if constexpr (S::WP == 3) h = __floats2half2_rn(v[0], v[1]);
#pragma unroll
          for (int part = 0; part < S::WP; ++part) {
            uint32_t c;
            if (part < S::WP - 3) {
              c = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E5M2);
              const float2 d = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c, __NV_E5M2)));
              v[0] -= d.x;
              v[1] -= d.y;
              if (part == S::WP - 4) h = __floats2half2_rn(v[0], v[1]);
            } else {
              c = take_e5m2x2(h);
            }
            uint8_t* to = wp + (part_at[part] & 0x7FFFFFFFu);
            const uint32_t flip = (part_at[part] >> 31) << 6;  // the row's other 64 bytes
            to[row_at[r] ^ flip] = (uint8_t)c;
            to[row_at[r + 1] ^ flip] = (uint8_t)(c >> 8);
          }
        }
        tc::fence_proxy_async();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&p_full[pb]);
      }
      // -- epilogue: normalise, write the output or this CTA's part of it
#pragma unroll
      for (int r = 0; r < HR; ++r) {
        const float x = half_sum(sum[r]);
        if ((lane & 15) == 0) sred[quad * R + rr + r] = x;
      }
      group_sync(bar_id);
      const bool whole = w.range < 0;
      const int64_t part = part_of(p, w.range, w.v, w.t0 == 0);
      if (quad == 0 && lane < RH) {
        const int r = r0 + lane;
        const float x = sred[r] + sred[R + r] + sred[2 * R + r] + sred[3 * R + r];
        // no key: the row is zeros; references are finite otherwise (or the row is NaN)
        const float2 f = x != 0.f ? pow2_pair(sref[r] - sreft[r]) : make_float2(0.f, 0.f);
        sfac[r] = make_float2(f.x, x != 0.f ? f.y / x : 0.f);
        if (!whole && r < nrow) p.part_lse[part * p.rows_tile + r] = x != 0.f ? sreft[r] + log2f(x) : -INFINITY;
      }
      group_sync(bar_id);
      wait(&pv_done[(n_tile - 1) & 1], (n_tile - 1) >> 1, tc::kTimeoutTmemEmpty);
      // a warp that gave up before this segment's last product was issued has said so
      const bool sound = *svoid == 0;
      if (!sound && !whole && quad == 0 && lane < RH && r0 + lane < nrow)
        p.part_lse[part * p.rows_tile + r0 + lane] = __uint_as_float(0x7FC00000u);
      __syncwarp();
      {
        const int elt = whole ? (int)sizeof(T) : 4, have_rows = nrow - r0, l0 = quad * 32 + lane;
        const int64_t row = whole ? (int64_t)b * p.rows + row0 + r0 : part * p.rows_tile + r0;
        uint8_t* to = (whole ? static_cast<uint8_t*>(p.a.out) : reinterpret_cast<uint8_t*>(p.part_o)) +
                      (row * width + l0) * elt;
        const int step = width * elt;
#pragma unroll 1
        for (int k = 0; k < p.boxes; ++k, to += 128 * elt) {
          __syncwarp();  // the box before may have been the end of some lanes' columns
          float v[S::MAX_STACK][RH];
#pragma unroll
          for (int g = 0; g < S::MAX_STACK; ++g)
            if (g < p.stack) tmem_ldn<RH>(tmem + lanes + (uint32_t)(k * p.np + g * R + r0), v[g]);
          tmem_wait_ld();
          const int rows = l0 + k * 128 < width ? have_rows : 0;
          uint8_t* at = to;
#pragma unroll
          for (int r = 0; r < RH; ++r, at += step) {
            const float2 f = sfac[r0 + r];
            float x = v[0][r];
#pragma unroll
            for (int g = 1; g < S::MAX_STACK; ++g)
              if (g < p.stack) x += v[g][r];
            // no key: the accumulator may hold a stale column, the row is zeros
            x = f.y == 0.f ? 0.f : x * f.x * f.y;
            if (!sound) x = __uint_as_float(0x7FC00000u);
            if (r < rows) {
              if (whole) *reinterpret_cast<T*>(at) = from_f<T>(x);
              else *reinterpret_cast<float*>(at) = x;
            }
          }
        }
      }
      tc::tc_fence_before();
      group_sync(bar_id);  // references and sums of the group are rewritten next
      w = nx;
      have = more;
    }
    if (p.direct && share.end == 0) {  // a pair without a key
      const int b = blockIdx.x / p.row_tiles, row0 = (blockIdx.x - b * p.row_tiles) * p.rows_tile;
      const int64_t n = (int64_t)min(p.rows_tile, p.rows - row0) * width;
      T* out = static_cast<T*>(p.a.out) + ((int64_t)b * p.rows + row0) * width;
      for (int64_t i = tid - 64; i < n; i += 256) out[i] = from_f<T>(0.f);
    }
    // a query copy that nobody waited for (a wait failed before its turn) lands before the CTA ends
    if (n_q > 0 && warp == 2 && elect_one())
      tc::mbar_wait_local(q_full, (n_q - 1) & 1, p.status, tc::kTimeoutDrain, tc::kDrainNs);
    __syncwarp();
  }
  tc::tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_relinquish();
    tc::tmem_dealloc(tmem, p.tmem);
  }
}

// Joins the ranges of a pair: weights 2^(lse_c - max), in the order of the ranges.  A pair inside one range is
// already written.  A block takes one row and COLS * V * 4 columns; with many parts (a few long sequences) SL
// groups of threads take every SL-th part each and are added up in shared memory.
template <typename T, int SL>
__global__ void __launch_bounds__(kJoinThreads<SL>) attn_tc_join_kernel(const __grid_constant__ TcParams p) {
  constexpr int COLS = kJoinThreads<SL> / SL, V = SL == 1 ? 2 : 1;  // threads along the columns, V times 4 columns each
  constexpr int U = SL > 2 ? 8 : 4;  // parts in flight
  __shared__ float4 sacc[SL > 1 ? SL : 1][COLS];
  __shared__ float slse[SL > 1 ? kMaxGrid : 1], sstat[SL > 1 ? 8 + SL : 1];
  const int v = blockIdx.x / p.rows_tile, r = blockIdx.x - v * p.rows_tile;
  const int b = v / p.row_tiles, row0 = (v - b * p.row_tiles) * p.rows_tile, width = p.a.cache.width;
  const int pairs = p.a.batch * p.row_tiles;
  const int col = threadIdx.x % COLS, grp = threadIdx.x / COLS, l0 = (blockIdx.y * COLS * V + col) * 4;
  pdl_wait();
  if (row0 + r >= p.rows) return;
  const int at = p.prefix[v], places = p.prefix[v + 1] - at, per = p.prefix[pairs + 1];
  const int n = places - p.start;  // tiles, if any
  const int c0 = n > 0 ? (at + p.start) / per : 0, c1 = n > 0 ? (at + places - 1) / per : -1;
  if (n > 0 && c0 == c1) return;
  // this row of the parts, one behind the other but for the first
  const int step = p.part_c * p.rows_tile;
  const int64_t row0_of = part_of(p, c0, v, false) * p.rows_tile + r;
  const int more = p.part_c == 1 ? 0 : p.rows_tile;
  auto row_of = [&](int i) { return row0_of + (int64_t)i * step + (i == 0 ? more : 0); };
  float4 acc[V];
  float m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  if constexpr (SL > 1) {  // all log-sums at once
    for (int i = threadIdx.x; i <= c1 - c0; i += kJoinThreads<SL>) {
      const float x = p.part_lse[row_of(i)];
      if (i < kMaxGrid) slse[i] = x;
      m = fmaxf(m, x);
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) sstat[threadIdx.x >> 5] = m;
    __syncthreads();
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kJoinThreads<SL> / 32; ++i) m = fmaxf(m, sstat[i]);
  }
  // without the log-sums at hand the weights follow a running maximum
  for (int c = c0 + grp; c <= c1; c += U * SL) {
    float f[U];
    float4 x[U][V];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int ci = c + i * SL;
      const bool on = ci <= c1;
      f[i] = !on ? -INFINITY : SL > 1 && ci - c0 < kMaxGrid ? slse[ci - c0] : p.part_lse[row_of(ci - c0)];
      const float* po = p.part_o + row_of(ci - c0) * width;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int l = l0 + k * COLS * 4;
        x[i][k] = on && l < width ? *reinterpret_cast<const float4*>(po + l)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    if constexpr (SL == 1) {
      float to = m;
#pragma unroll
      for (int i = 0; i < U; ++i) to = fmaxf(to, f[i]);
      const float g = m == to || to == -INFINITY ? 1.f : exp2f(m - to);
      m = to;
      sum *= g;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        acc[k].x *= g;
        acc[k].y *= g;
        acc[k].z *= g;
        acc[k].w *= g;
      }
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float e = exp2f(f[i] - base);  // 0 for a part that is not there
      sum += e;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        acc[k].x += e * x[i][k].x;
        acc[k].y += e * x[i][k].y;
        acc[k].z += e * x[i][k].z;
        acc[k].w += e * x[i][k].w;
      }
    }
  }
  if constexpr (SL > 1) {
    sacc[grp][col] = acc[0];
    if (col == 0) sstat[8 + grp] = sum;
    __syncthreads();
    if (grp != 0) return;
    for (int g = 1; g < SL; ++g) {
      const float4 x = sacc[g][col];
      acc[0].x += x.x;
      acc[0].y += x.y;
      acc[0].z += x.z;
      acc[0].w += x.w;
      sum += sstat[8 + g];
    }
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int l = l0 + k * COLS * 4;
    if (l >= width) continue;
    T* out = static_cast<T*>(p.a.out) + ((int64_t)b * p.rows + row0 + r) * width + l;
    const float o[4] = {acc[k].x, acc[k].y, acc[k].z, acc[k].w};
    struct alignas(4 * sizeof(T)) Four {
      T t[4];
    } four;
#pragma unroll
    for (int i = 0; i < 4; ++i) four.t[i] = from_f<T>(inv == 0.f ? 0.f : o[i] * inv);
    *reinterpret_cast<Four*>(out) = four;
  }
}

// Weight parts on N cost accumulator columns, parts along K cost a pass over the tile (36 + N / 5 clocks
// per 32 tokens x 128 latents as measured, whatever N holds): as many on N as make the passes cheapest.  One
// part on N / as chosen: 64 x 4,608, width 1536 12 heads 121.3 / 108.8 us (two on N), 3 heads 113.2 / 83.8 (three);
// 64 x 4,096, 10 heads, width 640 59.3 / 49.7 (three).
template <int RH, int QP>
bool fit(int boxes, Plan* pl) {
  using S = Shape<RH, QP>;
  bool found = false;
  int best = 0;
  for (int stack = 1; stack <= S::MAX_STACK; ++stack) {
    const int np = pad16(stack * S::R), runs = (S::WP + stack - 1) / stack, cols = boxes * np;
    const int bufs = cols + 2 * S::NS <= 512 ? 2 : cols + S::NS <= 512 ? 1 : 0;
    if (np > 256 || !bufs || (found && bufs < pl->s_bufs)) continue;
    const int cost = runs * (36 * 5 + np);
    if (found && cost >= best && bufs <= pl->s_bufs) continue;
    const int p_bytes = np * 128 * ((runs + 1) / 2);
    // Stages as wide as the ring allows with a tile in it and more to load.  Where the ring holds less than two
    // tiles, a tile's weights are written only once the tile before has left the ring: one weight buffer then
    // costs no time and widens the ring (24 heads, width 1536: 143 us, 152 with two; 12 heads the same).
    int tile_stages = 0, group = 0, stages = 0, p_bufs = 2;
    size_t fixed = 0;
    for (; p_bufs >= 1; --p_bufs) {
      fixed = (size_t)boxes * S::NS * 128 + p_bufs * p_bytes + (2 + 4 + 8) * S::R * 4 + (2 * kMaxStages + 10) * 8 + 80;
      stages = 0;
      for (int g = kMaxGroup; g >= 1 && fixed < kSmemMax; --g) {
        tile_stages = (boxes + g - 1) / g;
        group = (boxes + tile_stages - 1) / tile_stages;
        stages = (int)((kSmemMax - fixed) / (group * kBox));
        stages = stages < kMaxStages ? stages : kMaxStages;
        if (stages > tile_stages) break;
      }
      if (stages >= 2 * tile_stages || p_bufs == 1) break;
    }
    if (stages <= tile_stages) continue;
    found = true;
    best = cost;
    pl->rh = RH;
    pl->boxes = boxes;
    pl->group = group;
    pl->tile_stages = tile_stages;
    pl->stages = stages;
    pl->s_bufs = bufs;
    pl->ns = S::NS;
    pl->stack = stack;
    pl->runs = runs;
    pl->np = np;
    pl->p_bytes = p_bytes;
    pl->p_bufs = p_bufs;
    uint32_t n = 32;
    while (n < (uint32_t)(cols + bufs * S::NS)) n *= 2;
    pl->tmem = n;
    pl->smem = fixed + (size_t)stages * group * kBox;
  }
  return found;
}

// Whether each pair is one CTA's, written without a join.  Against the split list that gives up balance (all of
// `tiles` in a row, a whole wave of CTAs more for a pair too many) and saves the parts' way through memory and
// a launch.  In ns, as measured: 1.2 a tile and latent, 2,000 the join, 1 / 3,000 a byte of the parts, there and back.
// One CTA a pair / split, bf16: 64 x 256 tokens, 16 heads, L 1024 15.0 / 20.4 us; 100 x 400, 10, 640 18.1 / 24.9;
// 32 x 128, 12, 768 10.1 / 11.9; 200 x 500, 10, 640 35.2 / 35.9; 16 x 528, 10, 640 18.7 / 16.2; 4 x 300, 24, 1536
// 31.7 / 24.6; 1 x 512, 10, 640 16.5 / 12.7.  From the slots: the lengths are on the device.  So a buffer longer than what it
// holds is split: 64 x 300 tokens, 24 heads, L 1536 44.0 us in 300 slots, 52 - 54 in 1,024 .. 65,536.
bool one_cta_per_pair(int64_t pairs, int64_t tiles, int sms, int rows, int width) {
  const int64_t whole = (pairs + sms - 1) / sms * (tiles + kStart);
  const int64_t split = std::max<int64_t>((pairs * (tiles + kStart) + sms - 1) / sms, 1 + kStart);
  const int64_t part_bytes = std::min<int64_t>(pairs * tiles, sms) * rows * width * 8;
  return (whole - split) * width * 6 / 5 <= 2000 + part_bytes / 3000;
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
#undef KIMI_MLAC_FIT
  if (best.rh == 0) return false;
  *pl = best;
  pl->row_tiles = (rows + 2 * best.rh - 1) / (2 * best.rh);
  pl->rows_tile = (rows + pl->row_tiles - 1) / pl->row_tiles;
  if (pl->rows_tile <= 24 && best.rh > 12) {  // the rows of a tile pad less
    Plan c;
    if (fit<12, QP>(boxes, &c)) {
      c.row_tiles = pl->row_tiles;
      c.rows_tile = pl->rows_tile;
      *pl = c;
    }
  }
  const int64_t pairs = (int64_t)a.batch * pl->row_tiles, tiles = (a.cache.slots + kTile - 1) / kTile;
  if (pairs > (1 << 20) || pairs * tiles > (1 << 29)) return false;
  const int sms = device_sms() < kMaxGrid ? device_sms() : kMaxGrid;
  pl->direct = tiles <= kStretch && one_cta_per_pair(pairs, tiles, sms, pl->rows_tile, a.cache.width);
  pl->grid = pl->direct ? (int)pairs : (int)(pairs * tiles < sms ? pairs * tiles : sms);
  // as the kernel divides the list, for sequences that fill their slots: shorter ones make no more
  const int64_t whole = (pairs * (tiles + kStart) + pl->grid - 1) / pl->grid;
  pl->stretch = tiles <= kStretch ? 1 << 30 : kStretch;  // no pair is longer than a stretch: only the CTAs divide them
  pl->ranges = pl->grid * ((whole + pl->stretch - 1) / pl->stretch);
  return true;
}

bool plan_for(int dtype, const MlaCacheAttnArgs& a, Plan* pl) {
  return dtype == 1 ? make_plan<2>(a, pl) : make_plan<3>(a, pl);
}

// wide: [B][L / 128][Tmax][128] as a view of the cache, boxes of `group` chunks x 64 tokens.  Else [B][Tmax][L]
// with the smaller of the two outer strides first, boxes of 64 tokens x 128 latents (the last one partly zeros).
bool make_map(CUtensorMap* m, const MlaCacheAttnArgs& a, bool wide, int group, bool t_first, bool one) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  if (!fn) return false;
  const cuuint64_t slots = a.cache.slots, width = a.cache.width, ct = a.cache.code_t;
  const cuuint64_t nb = one ? 1 : a.batch, cb = one ? ct * slots : a.cache.code_b;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  cuuint64_t dims[4], strides[3];
  cuuint32_t box[4];
  if (wide) {
    dims[0] = 128; dims[1] = slots; dims[2] = width / 128; dims[3] = nb;
    strides[0] = ct; strides[1] = 128; strides[2] = cb;
    box[0] = 128; box[1] = kTile; box[2] = group; box[3] = 1;
  } else {
    dims[0] = width; dims[1] = t_first ? slots : nb; dims[2] = t_first ? nb : slots;
    strides[0] = t_first ? ct : cb; strides[1] = t_first ? cb : ct;
    box[0] = 128; box[1] = t_first ? kTile : 1; box[2] = t_first ? 1 : kTile;
  }
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, wide ? 4 : 3, a.cache.codes, dims, strides, box, ones,
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

template <typename K>
cudaError_t launch_dependent(K* kern, dim3 grid, int threads, size_t smem, cudaStream_t s, const TcParams& p) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T, int RH, int QP>
cudaError_t launch(const TcParams& p, const Plan& pl, cudaStream_t s) {
  auto kern = attn_tc_kernel<T, RH, QP>;
  cudaError_t e = ensure_dynamic_smem(kern, (int)pl.smem);
  if (e != cudaSuccess) return e;
  const int pairs = p.a.batch * p.row_tiles;
  e = launch_dependent(attn_tc_prep_kernel<T, QP>, dim3(pairs * p.rows_tile), (p.boxes * 16 + 31) / 32 * 32, 0, s, p);
  if (e != cudaSuccess) return e;
  if ((e = launch_dependent(kern, dim3(pl.grid), kThreads, pl.smem, s, p)) != cudaSuccess || pl.direct) return e;
  const unsigned rows = (unsigned)(pairs * p.rows_tile);
  const int width = p.a.cache.width;
  // Threads along the parts or along the columns: few rows want narrow blocks and many parts at once (one sequence of
  // 131,072, 16 heads, width 1024: all of it 47.3 us with SL = 16, 49.1 with 8; 700 tokens, 10 heads, width 640: 12.7
  // with 8, 13.6 with 2); many rows wide blocks (8 x 2304, 48 rows, width 768: 21.6 with 2, 26.9 with 8).
  const bool narrow = rows * ((width + 63) / 64) <= 600;
  // From the CTAs, not the ranges: a serving buffer is mostly longer than what it holds, and a sequence that fills many
  // stretches takes far longer than its join.  64 sequences of 300 tokens in 65,536 slots, 24 heads, width 1536: 53.2 / 66.6 us
  // by CTAs / by ranges.
  const int sl = pl.grid >= 32 * pairs ? (narrow ? 16 : 8) : pl.grid >= 6 * pairs ? (narrow ? 8 : 2) : 1;
  switch (sl) {
    case 16: return launch_dependent(attn_tc_join_kernel<T, 16>, dim3(rows, (width + 63) / 64), 256, 0, s, p);
    case 8: return launch_dependent(attn_tc_join_kernel<T, 8>, dim3(rows, (width + 127) / 128), 256, 0, s, p);
    case 2: return launch_dependent(attn_tc_join_kernel<T, 2>, dim3(rows, (width + 511) / 512), 256, 0, s, p);
    default: return launch_dependent(attn_tc_join_kernel<T, 1>, dim3(rows, (width + 1023) / 1024), kJoinThreads<1>, 0, s, p);
  }
}

template <typename T, int QP>
cudaError_t launch_rh(const TcParams& p, const Plan& pl, cudaStream_t s) {
  switch (pl.rh) {
    case 4: return launch<T, 4, QP>(p, pl, s);
    case 8: return launch<T, 8, QP>(p, pl, s);
    case 12: return launch<T, 12, QP>(p, pl, s);
    case 16: return launch<T, 16, QP>(p, pl, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

// 16-bit queries, and code rows that TMA can address: 16-byte base and strides.
bool mla_attn_tc_supported(int dtype, const MlaCacheAttnArgs& a) {
  if (dtype != 1 && dtype != 2) return false;
  if (a.cache.width % 16 || a.cache.width < 64 || a.cache.width > 8 * kPrepThreads) return false;
  if (a.cache.slots > (1 << 30)) return false;
  if ((reinterpret_cast<uintptr_t>(a.cache.codes) & 15) || (a.batch > 1 && a.cache.code_b % 16)) return false;
  if (a.cache.slots > 1 && (a.cache.code_t % 16 || a.cache.code_t < a.cache.width)) return false;
  Plan pl;
  return plan_for(dtype, a, &pl);
}

// Layout of the workspace, in floats: query images, score factors, partial contexts and log-sums, the
// tile list's prefix and the CTAs' first pairs.
struct Work {
  int64_t coef, part_o, part_lse, prefix, total;
};
static Work work_of(const MlaCacheAttnArgs& a, const Plan& pl) {
  const int64_t pairs = (int64_t)a.batch * pl.row_tiles, 
                units = pl.direct ? 0 : (pl.ranges + std::min(pl.ranges, pairs)) * pl.rows_tile;
  Work w;
  w.coef = pairs * pl.boxes * pl.ns * 32;
  w.part_o = w.coef + pairs * 2 * pl.rh;
  w.part_lse = w.part_o + units * a.cache.width;
  w.prefix = w.part_lse + units;
  w.total = w.prefix + pairs + 2;
  return w;
}

int64_t mla_attn_tc_workspace(int dtype, const MlaCacheAttnArgs& a) {
  Plan pl;
  return plan_for(dtype, a, &pl) ? work_of(a, pl).total : 0;
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
  p.group = pl.group;
  p.tile_stages = pl.tile_stages;
  p.stages = pl.stages;
  p.s_bufs = pl.s_bufs;
  p.stack = pl.stack;
  p.runs = pl.runs;
  p.r_pad = 2 * pl.rh;
  p.ns = pl.ns;
  p.np = pl.np;
  p.p_bytes = pl.p_bytes;
  p.p_bufs = pl.p_bufs;
  p.q_bytes = pl.boxes * pl.ns * 128;
  p.grid = pl.grid;
  p.start = (a.cache.slots + kTile - 1) / kTile * a.batch * pl.row_tiles <= pl.grid ? 0 : kStart;
  p.part_c = (int64_t)a.batch * pl.row_tiles <= pl.ranges ? 1 : 2;
  p.stretch = pl.stretch;
  p.fetch = kFetch;
  p.direct = pl.direct ? 1 : 0;
  p.tmem = pl.tmem;
  p.q_vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.q_b % 8 == 0 && a.q_i % 8 == 0 && a.q_h % 8 == 0;
  const bool one = a.batch == 1 || a.cache.code_b == 0;  // every sequence reads the same rows
  p.z_mul = one ? 0 : 1;
  p.t_first = one || p.a.cache.code_t <= a.cache.code_b ? 1 : 0;
  // the encoder needs the device's context on this host thread
  static thread_local bool bound = false;
  if (!bound) {
    (void)cudaFree(nullptr);
    bound = true;
  }
  p.wide = a.cache.width % 128 == 0 ? 1 : 0;
  if (!make_map(&p.map, p.a, p.wide, p.group, p.t_first, one)) return cudaErrorInvalidValue;
  const Work wk = work_of(a, pl);
  p.q_parts = reinterpret_cast<uint8_t*>(a.part_acc);
  p.coef = a.part_acc + wk.coef;
  p.part_o = a.part_acc + wk.part_o;
  p.part_lse = a.part_acc + wk.part_lse;
  p.prefix = reinterpret_cast<int*>(a.part_acc + wk.prefix);
  p.status = status_ptr();
  if (!p.status) return cudaErrorInvalidValue;
  return dtype == 1 ? launch_rh<__nv_bfloat16, 2>(p, pl, s) : launch_rh<__half, 3>(p, pl, s);
}

int* mla_cache_default_status() { return status_ptr(); }

}  // namespace kimi
