// Attention over the per-head cache for many query rows per key head: drafted trees of grouped
// heads, chunks of a prompt (kv_attn.cuh has the formulas, the numbers and the cut of the work).
//
// Rows are the MMA's M: S = Q K^T and O += P V on tcgen05 in bf16, scores, weights and outputs
// in tensor memory, the weights as the second product's A operand where the scores were. Keys
// and values come from the cache as codes in registers and are expanded to bf16 in shared
// memory on the way (4 KB of codes are read once per 256 rows; the expansion, ten
// operations per four codes on two pipes, runs beside the products).
//
// Scores come in buffers of 64 keys, two per stream, so that a row's stay in registers from the
// maximum to the weights and the next are there when it is done with them (with one buffer of 128
// the chain scores -> softmax -> output -> scores took 6700 cycles, 5000 of them softmax).  The
// weights of a buffer go where its scores were.
// A CTA works on two streams, so that one's softmax runs under the other's products:
//   D <= 128, more than 128 rows: a stream per 128 rows, on the same keys;
//   D <= 128, up to 128 rows: even and odd tiles of keys, each stream with references, sums and
//     outputs of its own, added up at the end of the row tile;
//   D > 128 (tensor memory holds one output): even and odd tiles, one output; one warpgroup does
//     the softmax of both in turn.
// Warps: 0-3 and 4-7 softmax (thread = row = TMEM lane), also queries and results; 8 issues the
// products; 9 walks the page table and the scales; 10-16 and 17-23 load and expand, every other
// unit (the keys or the values of a tile) each.  Units lie in a ring in the order the products
// take them; a warp's codes are loaded a unit of its own ahead, into the registers just used.
// (Expansion is a chain of latencies: with seven warps that also found the addresses themselves it
// took 3700 cycles a unit, two units a tile, and was what everything waited for.)
//
// Bound by the chain scores -> weights -> output and by the expansion, no unit being full (1024
// tokens of 64 heads of 128 on 8 behind 12288, under a profiler: tensor cores 41 % of their cycles,
// issue 59 %, ALU 44 %, exponentials 41 %).  Measured (one B200): 4096 such tokens 2470 us, 779
// TFLOP/s (2255 in runs too short for the power limit); 2048 tokens of heads of 256 2.5 ms in short
// runs (714 TFLOP/s, expansion bound: a unit is twice as large); 16 trees of 13 tokens, 64 heads on
// 8, up to 6001 keys 92 to 96 us (5 K cycles a tile, 10 us of it the join), chains of 3 tokens 83: a
// product has 128 rows whatever the call has.  The steps that made the 4096 tokens faster, in short
// runs: 3240 us; codes loaded a unit ahead and no rare path unrolled 2560; buffers of 64 keys 2320;
// one issuing thread 2265 to 2339; more registers for the expansion 2240.
// 80 registers at launch make the softmax's code spill: 212 bytes of stores and 420 of loads at heads
// of 256, 228 and 488 at 128, 184 and 384 at 64.
//
// References are raised only when a score passes them by 2^KVA_RISE (rarely after the first
// tiles); then the row's output is scaled in place once its last product is done.
#pragma once
#include "kv_attn.cuh"

namespace ks {

constexpr int KVW_SOFT = 256;                       // softmax threads (the first ones)
constexpr int KVW_CONV_WARPS = 7;                   // of either group of expanding warps (the last ones)
constexpr int KVW_THREADS = KVW_SOFT + 64 + 2 * 32 * KVW_CONV_WARPS;
// 768 threads start with 80 registers; the softmax warpgroups take theirs from the other four.
// (4096 tokens of 64 heads over 12288 keys, softmax / others: 128 / 56 2339 us, 112 / 64 2237 us;
// 2048 tokens at heads of 256 2674 and 2503 us; 96 / 72 is 10 % slower.)
constexpr int KVW_REGS_SOFT = 112, KVW_REGS_REST = 64;
static_assert(KVW_THREADS == 768 && 2 * KVW_REGS_SOFT + 4 * KVW_REGS_REST <= 6 * 80, "register split");
constexpr int KVW_META = 8;                         // units whose addresses are held
constexpr int KVW_UNITS = 8;                        // most units of the ring
constexpr int KVW_HDR = 12288;

template <int D>
constexpr int KVW_STREAM_OUT = D <= 128 ? 2 : 1;    // outputs in tensor memory
template <int D>
constexpr uint32_t KVW_TILE = 128u * D * 2;         // bytes of a unit, and of 128 queries
template <int D>
__host__ __device__ constexpr int kvw_units() {
  const int n = (int)((232448 - 1024 - KVW_HDR - KVW_STREAM_OUT<D> * KVW_TILE<D>) / KVW_TILE<D>);
  // (an odd number, three for D = 192, gives a slot's units to the expanding groups by turns; a group
  // is then at most a phase ahead because units are given back in order.  Two: 8 % slower)
  return n < KVW_UNITS ? n : KVW_UNITS;
}

struct KvwMeta {
  uint32_t place[8];          // of the unit's groups of 16 keys, in 16 rows of the page pool
  uint32_t scale[8];          // their scales' bits, 0: not there
  uint32_t factor[8];         // 2^120 times those, twice
  uint32_t flags;
};
enum : uint32_t { KVW_VALUES = 1, KVW_PLAIN = 2, KVW_END = 4 };  // PLAIN: no larger scale, no mark

struct KvwShared {
  KvaFind find;
  KvwMeta meta[KVW_META];
  uint64_t meta_full[KVW_META], meta_free[KVW_META];
  uint64_t full[KVW_UNITS], free[KVW_UNITS];
  uint64_t s_full[4], p_full[4], o_done[4];  // buffer 2 * stream + half of the tile
  uint64_t q_full, q_free, drain;
  uint64_t pair_full, pair_free;  // the second stream's results are there / have been taken
  uint32_t tmem;
  int abort;
  uint32_t info[16];          // of a tile: bits 0-7 groups of 16 keys that are not there, 8-15 values marked
  float m[128], l[128];       // of the second stream, for the first
  bool nans[128];
  uint32_t nan[2][128][8];    // columns that are NaN of a row's output, where some are
};
static_assert(sizeof(KvwShared) <= KVW_HDR, "KvwShared exceeds its header");

// Products in bf16 with fp32 sums; A in shared memory or in tensor memory, B in shared memory.
// Descriptors as words: the high one (8 rows 1024 bytes apart, 128-byte swizzle) is always the
// same, and the start address sits in the low bits of the low one, so that an operand's steps are
// additions.  (With 64-bit descriptors put together for each product, the one thread that issues
// them took 90 cycles a product, more than the tensor cores.)
constexpr uint32_t KVW_DESC_HI = (1024u >> 4) | 1u << 14 | 1u << 30;
__device__ __forceinline__ uint32_t kvw_desc(uint32_t saddr, uint32_t lbo_bytes) { return saddr >> 4 | lbo_bytes >> 4 << 16; }
__device__ __forceinline__ void kvw_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 ad, bd; setp.ne.b32 p, %4, 0; mov.b64 ad, {%1, %5}; mov.b64 bd, {%2, %5};"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %3, p; }" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(KVW_DESC_HI)
      : "memory");
}
__device__ __forceinline__ void kvw_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{ .reg .pred p; .reg .b64 bd; setp.ne.b32 p, %4, 0; mov.b64 bd, {%2, %5};"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], bd, %3, p; }" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(KVW_DESC_HI)
      : "memory");
}

// Order in which the units of a row tile's n tiles are used; two: both streams take every tile.
//   K0 V0 K1 V1 ..   or   K0 K1 V0 K2 V1 K3 ..
struct KvwUnit {
  int tile;
  bool v;
};
__device__ __forceinline__ KvwUnit kvw_unit(int i, int n, bool two) {
  if (two) return {i >> 1, (i & 1) != 0};
  if (n == 1) return {0, i == 1};
  if (i < 2) return {i, false};
  if (i == 2 * n - 1) return {n - 1, true};
  return (i & 1) ? KvwUnit{(i + 1) >> 1, false} : KvwUnit{(i - 2) >> 1, true};
}

// Columns of the values that are NaN in positions that a row sees.
template <int D>
__device__ __forceinline__ void kvw_nan_columns(const KvAttnParams& p, int b, int h, int len, int n, int t, int pos0,
                                             int keys, uint32_t groups, uint32_t* mask) {
  for (int g = 0; g < 8; ++g) {
    if (!((groups >> g) & 1u)) continue;
    const int at = pos0 + 16 * g, pi = kva_div(at, p.c.page, p.page_shift);
    const int pg = __ldg(p.c.table + (int64_t)b * p.c.max_pages + pi);
    const uint8_t* base = p.c.v8 + (((int64_t)pg * p.c.heads + h) * p.c.page + (at - pi * p.c.page)) * D;
    for (int k = 0; k < 16 && at + k < keys; ++k) {
      if (!kva_sees(p, b, len, n, t, at + k)) continue;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(base + k * D);
      for (int i = 0; i < D / 32; ++i) {
        uint32_t bits = 0;
        for (int j = 0; j < 8; ++j) bits |= kva_nan4_bits(__ldg(w + i * 8 + j)) << (4 * j);
        mask[i] |= bits;
      }
    }
  }
}

__device__ __forceinline__ float kvw_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void kvw_load(uint32_t (&v)[4], const uint8_t* ptr) {
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "l"(ptr));
}
// Two e4m3 codes in the low bytes of two halves to bf16 2^-120 times as large: exponent and
// mantissa move up by four bits and the sign by eight.  (As multiplications, which leave the
// integer pipe to the softmax: shifts and masks there took 4 of every 10 of its cycles.)
__device__ __forceinline__ uint32_t kvw_place(uint32_t x) { return (x & 0x00800080u) * 0xF0u + x * 16u; }

template <int D>
__global__ void __launch_bounds__(KVW_THREADS, 1) kv_attn_wide_kernel(const __grid_constant__ KvAttnParams p) {
  constexpr int UNITS = kvw_units<D>();
  constexpr uint32_t TILE = KVW_TILE<D>;
  constexpr bool ONE_OUT = KVW_STREAM_OUT<D> == 1;
  static_assert(UNITS >= 2, "the ring needs two units");
  extern __shared__ uint8_t kvw_raw[];
  const uint32_t raw = smem_u32(kvw_raw);
  uint8_t* smem = kvw_raw + (((raw + 1023u) & ~1023u) - raw);
  KvwShared* sh = reinterpret_cast<KvwShared*>(smem);
  uint8_t* qs = smem + KVW_HDR;                              // [outputs][D / 64][128 rows x 128 B], swizzled
  uint8_t* ring = qs + KVW_STREAM_OUT<D> * TILE;             // [UNITS][D / 64][128 keys x 128 B], swizzled
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  WaitCtx wc{&sh->abort, p.c.status, p.budget_ns};

  if (tid == 0) {
    for (int i = 0; i < UNITS; ++i) {
      mbar_init(&sh->full[i], KVW_CONV_WARPS);
      mbar_init(&sh->free[i], 1);
    }
    for (int i = 0; i < KVW_META; ++i) {
      mbar_init(&sh->meta_full[i], 1);
      mbar_init(&sh->meta_free[i], KVW_CONV_WARPS);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->p_full[i], 4);
      mbar_init(&sh->o_done[i], 1);
    }
    mbar_init(&sh->q_full, ONE_OUT ? 4 : 8);
    mbar_init(&sh->q_free, 1);
    mbar_init(&sh->drain, 1);
    mbar_init(&sh->pair_full, 4);
    mbar_init(&sh->pair_free, 4);
    sh->abort = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc<1>(&sh->tmem, 512);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may be set up
  kva_find(p, &sh->find);  // (its barriers also publish the above)
  tc_fence_after();
  const uint32_t tmem = sh->tmem;
  KvaWalk w;
  w.start(p, &sh->find);
  if (tid == 0) kva_clear(p, w);
  const bool rows256 = p.nr == 256;

  if (warp < 8) {
    // -------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KVW_REGS_SOFT));
    const int wg = warp >> 2, t128 = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t s_ph = 0;  // phases of the score buffers, a bit each
    // products with the weights of each buffer so far, modulo two.  A buffer's scores come after the
    // product with the weights that were in it before, so at most one of its products is ever
    // waited for, and its parity tells it.
    uint32_t o_ph = 0;
    bool first = true;
    // the scale's sign goes into the queries; times 2^-149 instead of zero, unseen scores stay -inf
    const uint32_t turn = p.scale_log2 < 0.f ? 0x80008000u : 0u;
    const float scale = fmaxf(fabsf(p.scale_log2), __uint_as_float(1u));
    uint32_t item = 0, tiles_before = 0, pair_ph = 0;
    for (; w.left > 0; w.next(p)) {
      const int r0 = w.rt * p.nr;
      if (w.empty()) {
        for (int i = tid; i < p.nr * (D / 8); i += KVW_SOFT) {
          const int row = r0 + i / (D / 8), t = row / p.G;
          if (row < p.rows)
            reinterpret_cast<uint4*>(p.out + (((int64_t)w.b * p.c.T + t) * p.H + w.h * p.G + row % p.G) * D)[i % (D / 8)] =
                make_uint4(0, 0, 0, 0);
        }
      }
      if (!w.any()) continue;
      if (tid == 0 && (int64_t)w.len + w.n > p.c.max_pages * p.c.page)
        report_bounds(p.c.status, w.b, (int)p.c.max_pages);
      const int n = w.t1 - w.t0;
      const bool two = rows256 && r0 + 128 < p.rows;  // both streams on every tile
      // ------------------------------------------------------------ queries
      // (with one output the second warpgroup writes no queries, so nothing waits for it and q_free may
      // complete twice before it looks: it has no part in that barrier)
      if (!ONE_OUT || wg == 0) {
        // (a warp gives up as one: a lane that left alone would be missed at the warp's next barrier)
        if (!first && !__all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->q_free, (item - 1) & 1, wc))) break;
        first = false;
        const int base = !rows256 ? 0 : wg * 128;  // rows of this warpgroup's queries
        if (rows256 || ONE_OUT || wg == 0) {
          uint8_t* dst = qs + (rows256 ? wg : 0) * TILE;
          for (int i = t128; i < 128 * (D / 8); i += 128) {
            const int rr = i / (D / 8), u = i - rr * (D / 8), row = r0 + base + rr;
            const int t = row / p.G;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (row < p.rows)
              x = __ldg(reinterpret_cast<const uint4*>(
                  p.q + (((int64_t)w.b * p.c.T + t) * p.H + w.h * p.G + (row - t * p.G)) * D + u * 8));
            *reinterpret_cast<uint4*>(dst + (u >> 3) * 16384 + rr * 128 + (((u & 7) ^ (rr & 7)) << 4)) =
                make_uint4(x.x ^ turn, x.y ^ turn, x.z ^ turn, x.w ^ turn);
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->q_full);
      }
      ++item;
      if (ONE_OUT && wg == 1) continue;
      // ------------------------------------------------------------ tiles of this warpgroup
      // two: all of them, in the buffers of stream wg; else every other one; one output: all, in the
      // streams' buffers by turns
      const int my_row = r0 + (rows256 ? wg * 128 : 0) + t128;
      const int tok = my_row / p.G;
      const int clear = w.len + (p.mask ? 0 : (my_row - t128) / p.G + 1);
      const int limit = tok < w.n ? (int)min((int64_t)w.len + (p.mask ? 0 : tok + 1), (int64_t)w.keys) : 0;
      const int step = ONE_OUT || two ? 1 : 2;  // tiles
      const bool idle = rows256 && !two && wg == 1;
      float m = -INFINITY, l = 0.f;
      bool nans = false;  // sh->nan is in use
      int last = -1;  // buffer of the last weights
      const uint32_t o_col = tmem + 256 + (ONE_OUT ? 0 : wg * D) + lanes;
      bool ok = true;
      // (a row tile of 256 rows whose second half is empty is done by even and odd tiles too:
      // both warpgroups then have the first 128 rows)
      const int row = idle ? my_row - 128 : my_row;
      const int tk = idle ? row / p.G : tok;
      const int cl = idle ? w.len + (p.mask ? 0 : r0 / p.G + 1) : clear;
      const int lm = idle ? (tk < w.n ? (int)min((int64_t)w.len + (p.mask ? 0 : tk + 1), (int64_t)w.keys) : 0) : limit;
      for (int q = step == 2 ? 2 * wg : 0; q < 2 * n; q += (q & 1) ? 2 * step - 1 : 1) {
        const int j = q >> 1, h = q & 1, buf = 2 * (ONE_OUT ? j & 1 : wg) + h;
        const uint32_t s_col = tmem + buf * 64 + lanes;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->s_full[buf], (s_ph >> buf) & 1, wc));
        if (!ok) break;
        s_ph ^= 1u << buf;
        tc_fence_after();
        float x[64];
        tmem_ld32(s_col, reinterpret_cast<uint32_t*>(x));
        tmem_ld32(s_col + 32, reinterpret_cast<uint32_t*>(x + 32));
        const int pos0 = (w.t0 + j) * 128 + 64 * h;
        const uint32_t info = sh->info[(tiles_before + j) & 15], gone = (info >> (4 * h)) & 15u;
        tmem_wait_ld();
        if (pos0 + 64 > cl || gone) {
          // some rows do not see some of the keys
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int at = pos0 + 32 * c, k = lm - at;
            uint32_t see = k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1u;
            if (p.mask && tk < w.n)
              for (int i = max(w.len - at, 0); i < 32 && at + i < w.keys; ++i)
                if (kva_sees(p, w.b, w.len, w.n, tk, at + i)) see |= 1u << i;
            if ((gone >> (2 * c)) & 1u) see &= 0xFFFF0000u;
            if ((gone >> (2 * c + 1)) & 1u) see &= 0x0000FFFFu;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((see >> i) & 1u)) x[32 * c + i] = -INFINITY;
          }
        }
        // ---------------------------------------------------------- maximum
        float top = kvw_max3(x[0], x[1], x[2]), top1 = kvw_max3(x[3], x[4], x[5]);
#pragma unroll
        for (int i = 6; i < 62; i += 4) {
          top = kvw_max3(top, x[i], x[i + 1]);
          top1 = kvw_max3(top1, x[i + 2], x[i + 3]);
        }
        top = fmaxf(kvw_max3(kvw_max3(top, x[62], x[63]), top1, -INFINITY), -INFINITY);
        top = top == -INFINITY ? top : top * scale;
        // ---------------------------------------------------------- raise the reference
        if (__any_sync(0xFFFFFFFFu, top > m + KVA_RISE)) {
          const float now = fmaxf(m, top);
          const float f = now == -INFINITY ? 1.f : ex2f(m - now);
          m = now;
          l *= f;
          if (last >= 0) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->o_done[last], ((o_ph >> last) & 1) ^ 1, wc));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float y[16];
              tmem_ld16(o_col + c, reinterpret_cast<uint32_t*>(y));
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) y[i] *= f;
              tmem_st16(o_col + c, reinterpret_cast<uint32_t*>(y));
            }
            tmem_wait_st();
          }
        }
        // ---------------------------------------------------------- weights
        const float mu = (m == -INFINITY ? 0.f : m) + KVA_DOWN;
        const float2 sc = make_float2(scale, scale), minus = make_float2(-mu, -mu);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t e[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 y = fma2(make_float2(x[32 * c + 2 * i], x[32 * c + 2 * i + 1]), sc, minus);
            y = make_float2(ex2f(y.x), ex2f(y.y));
            sum = add2(sum, y);
            e[i] = cvt_bf16x2(y.x, y.y);
          }
          tmem_st16(s_col + 16 * c, e);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[buf]);
        o_ph ^= 1u << buf;
        last = buf;
        l += sum.x + sum.y;
        if ((info >> 8) && h == 1) {
          if (!nans)
            for (int i = 0; i < D / 32; ++i) sh->nan[wg][t128][i] = 0;
          nans = true;
          kvw_nan_columns<D>(p, w.b, w.h, w.len, w.n, tk, pos0 - 64, w.keys, info >> 8, sh->nan[wg][t128]);
        }
      }
      if (!ok) break;
      tiles_before += n;
      // ------------------------------------------------------------ results
      if (last >= 0) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->o_done[last], ((o_ph >> last) & 1) ^ 1, wc));
        tc_fence_after();
      }
      if (!ONE_OUT && !two) {
        // even and odd tiles together: the first warpgroup takes the second's
        if (wg == 1) {
          sh->m[t128] = m;
          sh->l[t128] = l;
          sh->nans[t128] = nans;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->pair_full);
          // its output is the first warpgroup's to read until here
          ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->pair_free, pair_ph, wc));
        } else {
          ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->pair_full, pair_ph, wc));
          tc_fence_after();
        }
        pair_ph ^= 1;
      }
      if (ok && (two || wg == 0)) {
        const bool both = !ONE_OUT && !two && n > 1;
        float f0 = 1.f, f1 = 0.f;
        if (both) {
          const float m1 = sh->m[t128], l1 = sh->l[t128];
          const float now = fmaxf(m, m1);
          f0 = now == -INFINITY ? 1.f : ex2f(m - now);
          f1 = now == -INFINITY ? 1.f : ex2f(m1 - now);
          l = l * f0 + l1 * f1;
          m = now;
          if (sh->nans[t128]) {
            for (int i = 0; i < D / 32; ++i) sh->nan[0][t128][i] = (nans ? sh->nan[0][t128][i] : 0u) | sh->nan[1][t128][i];
            nans = true;
          }
        }
        const bool whole = w.whole(), in = row < p.rows;
        const int g = row - tk * p.G;
        float f = 1.f;
        if (whole)
          f = kva_norm(m, l, in && p.sink ? __ldg(p.sink + w.h * p.G + g) * 1.4426950408889634f : 0.f, in && p.sink);
        uint16_t* orow = p.out + (((int64_t)w.b * p.c.T + tk) * p.H + w.h * p.G + g) * D;
        const int64_t prow = (int64_t)w.slot() * p.nr + (row - r0);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float x[32];
          tmem_ld32(o_col + c, reinterpret_cast<uint32_t*>(x));
          tmem_wait_ld();
          if (both) {
            float y[32];
            tmem_ld32(o_col + D + c, reinterpret_cast<uint32_t*>(y));
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = x[i] * f0 + y[i] * f1;
          }
          if (nans) {
            const uint32_t nan = sh->nan[wg][t128][c / 32];
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if ((nan >> i) & 1u) x[i] = __uint_as_float(0x7FC00000u);
          }
          if (whole) {
            if (in) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint4 v = make_uint4(cvt_bf16x2(x[8 * i] * f, x[8 * i + 1] * f), cvt_bf16x2(x[8 * i + 2] * f, x[8 * i + 3] * f),
                                     cvt_bf16x2(x[8 * i + 4] * f, x[8 * i + 5] * f), cvt_bf16x2(x[8 * i + 6] * f, x[8 * i + 7] * f));
                if (tk >= w.n) v = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(orow + c + 8 * i) = v;
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<float4*>(p.part_o + prow * D + c + 4 * i) =
                  make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
          }
        }
        if (!whole) {
          p.part_ml[prow] = make_float2(m, l);
          if (tid == 0 && w.t0 == 0) w.share(p, sh->find.per);
        }
        tc_fence_before();
      }
      if (!ok) break;
      if (!ONE_OUT && !two && wg == 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->pair_free);
      }
    }
  } else if (warp == 8) {
    // -------------------------------------------------------------- products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KVW_REGS_REST));
    // One thread does all of it: every instruction of this warp is in the chain of products.
    if (elect_one()) {
      uint32_t unit = 0, q_ph = 0, p_ph = 0;
      constexpr uint32_t idesc_s = idesc_bf16_f32(128, 64, false, false);
      constexpr uint32_t idesc_o = idesc_bf16_f32(128, D, false, true);
      const uint32_t q_desc = kvw_desc(smem_u32(qs), 16), k_desc = kvw_desc(smem_u32(ring), 16),
                     v_desc = kvw_desc(smem_u32(ring), 16384);
      bool ok = true;
      const auto wait = [&](uint64_t* bar, uint32_t ph) {
        ok = ok && mbar_wait_inl(bar, ph, wc);
        tc_fence_after();
        return ok;
      };
      // scores of half h of the tile whose keys are in `slot`, into the stream's buffer
      const auto qk = [&](int stream, int h, int qt, uint32_t slot) {
        const uint32_t a = q_desc + qt * (TILE >> 4), b = k_desc + slot * (TILE >> 4) + h * (8192 >> 4);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
          kvw_mma_ss(tmem + (2 * stream + h) * 64, a + off, b + off, idesc_s, ks > 0);
        }
        umma_commit(&sh->s_full[2 * stream + h]);
      };
      // a whole tile's, into both of the stream's buffers, which lie side by side
      const auto qk_tile = [&](int stream, uint32_t slot) {
        const uint32_t b = k_desc + slot * (TILE >> 4);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
          kvw_mma_ss(tmem + stream * 128, q_desc + off, b + off, idesc_bf16_f32(128, 128, false, false), ks > 0);
        }
        umma_commit(&sh->s_full[2 * stream]);
        umma_commit(&sh->s_full[2 * stream + 1]);
      };
      const auto pv = [&](int stream, int h, int out, uint32_t slot, bool acc) {
        const uint32_t b = v_desc + slot * (TILE >> 4) + h * (8192 >> 4);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          kvw_mma_ts(tmem + 256 + out * D, tmem + (2 * stream + h) * 64 + ks * 8, b + ks * (2048 >> 4), idesc_o,
                     acc || ks > 0);
        umma_commit(&sh->o_done[2 * stream + h]);
      };
      const auto weights = [&](int stream, int h) {
        const int buf = 2 * stream + h;
        const bool there = wait(&sh->p_full[buf], (p_ph >> buf) & 1);
        p_ph ^= 1u << buf;
        return there;
      };
      for (; w.left > 0 && ok; w.next(p)) {
        if (!w.any()) continue;
        const int n = w.t1 - w.t0;
        const bool two = rows256 && w.rt * 256 + 128 < p.rows;
        if (!wait(&sh->q_full, q_ph)) break;
        q_ph ^= 1;
        // unit i of the row tile: waits for it and gives its slot
        const uint32_t base = unit;
        const auto take = [&](int i, uint32_t* slot) {
          const uint32_t u = base + i;
          *slot = u % UNITS;
          return wait(&sh->full[*slot], (u / UNITS) & 1);
        };
        uint32_t vs, ks;
        if (two) {
          if (!take(0, &ks)) break;
          for (int q = 0; q < 4; ++q) qk(q & 1, q >> 1, q & 1, ks);
          umma_commit(&sh->free[ks]);
          if (n == 1) umma_commit(&sh->q_free);
          for (int j = 0; j < n && ok; ++j) {
            if (!take(2 * j + 1, &vs)) break;
            for (int q = 0; q < 4; ++q) {
              const int s = q & 1, h = q >> 1;
              if (!weights(s, h)) break;
              pv(s, h, s, vs, j > 0 || h > 0);
              if (q == 3) umma_commit(&sh->free[vs]);
              if (j + 1 < n) {
                if (q == 0 && !take(2 * j + 2, &ks)) break;
                qk(s, h, s, ks);
              }
            }
            if (ok && j + 1 < n) {
              umma_commit(&sh->free[ks]);
              if (j + 2 == n) umma_commit(&sh->q_free);
            }
          }
        } else {
          for (int j = 0; j < min(n, 2) && ok; ++j) {
            if (!take(j, &ks)) break;
            // (wide heads wait for the tensor cores, which 64 keys at a time would feed from shared
            // memory at two thirds of their rate)
            if constexpr (ONE_OUT) {
              qk_tile(j, ks);
            } else {
              qk(j, 0, 0, ks);
              qk(j, 1, 0, ks);
            }
            umma_commit(&sh->free[ks]);
            if (j + 1 == n) umma_commit(&sh->q_free);
          }
          for (int j = 0; j < n && ok; ++j) {
            const int s = j & 1;
            // values of tile j: unit 1 of a single tile; else 2 + 2 j, the last one 2 n - 1
            if (!take(n == 1 ? 1 : j + 1 == n ? 2 * n - 1 : 2 + 2 * j, &vs)) break;
            for (int h = 0; h < 2; ++h) {
              if (!weights(s, h)) break;
              pv(s, h, ONE_OUT ? 0 : s, vs, h > 0 || (ONE_OUT ? j > 0 : j > 1));
              if (h == 1) umma_commit(&sh->free[vs]);
              if (j + 2 < n) {
                if (h == (ONE_OUT ? 1 : 0) && !take(2 * j + 3, &ks)) break;
                if constexpr (!ONE_OUT) qk(s, h, 0, ks);
                else if (h == 1) qk_tile(s, ks);
              }
            }
            if (ok && j + 2 < n) {
              umma_commit(&sh->free[ks]);
              if (j + 3 == n) umma_commit(&sh->q_free);
            }
          }
        }
        unit += 2 * n;
      }
      // every product and arrival in flight has landed before the CTA gives its memory back
      umma_commit(&sh->drain);
      mbar_wait_body(&sh->drain, 0, wc, false, true);
    }
    __syncwarp();
  } else if (warp == 9) {
    // -------------------------------------------------------------- addresses
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KVW_REGS_REST));
    const uint32_t per_page = (uint32_t)(p.c.page / p.c.block), page16 = (uint32_t)(p.c.page >> 4);
    uint32_t unit = 0, tiles_before = 0;
    bool ok = true;
    // a unit whose scales are on their way; lanes 0-7: a group of 16 of its keys each
    struct Unit {
      uint32_t place, scale, v_scale, gone;
      int tile;  // of all
      bool v;
    } last{};
    const auto publish = [&](const Unit& a, uint32_t u) {
      const uint32_t slot = u % KVW_META;
      if (u >= KVW_META) ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->meta_free[slot], ((u / KVW_META) & 1) ^ 1, wc));
      if (!ok) return;
      KvwMeta& m = sh->meta[slot];
      float rest;
      const uint32_t scale = a.v ? a.v_scale : a.scale, factor = kva_factor(scale, &rest);
      const bool plain = !__any_sync(0xFFFFFFFFu, rest != 1.f || (scale & 1u));
      const uint32_t marks = __ballot_sync(0xFFFFFFFFu, a.v_scale & 1u) & 255u;
      if (lane < 8) {
        m.place[lane] = a.place;
        m.scale[lane] = scale;
        m.factor[lane] = factor;
      }
      if (lane == 0) {
        m.flags = (a.v ? KVW_VALUES : 0u) | (plain ? KVW_PLAIN : 0u);
        if (!a.v) sh->info[a.tile & 15] = a.gone | marks << 8;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->meta_full[slot]);
    };
    for (; w.left > 0 && ok; w.next(p)) {
      if (!w.any()) continue;
      const int n = w.t1 - w.t0;
      const bool two = rows256 && w.rt * 256 + 128 < p.rows;
      const auto page_of = [&](int tile) {
        const int pos = (w.t0 + tile) * 128 + 16 * lane;
        return lane < 8 && tile < n && pos < w.keys
                   ? __ldg(p.c.table + (int64_t)w.b * p.c.max_pages + kva_div(pos, p.c.page, p.page_shift)) : -2;
      };
      int pg0 = page_of(0), pg1 = page_of(1);  // page numbers of the tiles to come, by tile parity
      for (int i = 0; i < 2 * n && ok; ++i) {
        const KvwUnit u = kvw_unit(i, n, two);
        const int page = (u.tile & 1) ? pg1 : pg0, pos = (w.t0 + u.tile) * 128 + 16 * lane;
        const bool there = page >= 0 && page < p.c.n_pages;
        if (page != -2 && !there) report_bounds(p.c.status, w.b, (int)p.c.n_pages);
        const uint32_t in = there ? (uint32_t)(pos - kva_div(pos, p.c.page, p.page_shift) * p.c.page) : 0u;
        const uint32_t at = (there ? (uint32_t)page : 0u) * (uint32_t)p.c.heads + (uint32_t)w.h;
        Unit now;
        now.place = at * page16 + (in >> 4);  // (the host has checked that it fits)
        const uint32_t si = at * per_page + (uint32_t)kva_div((int)in, p.c.block, p.block_shift);
        now.scale = now.v_scale = 0;
        if (there) {
          now.v_scale = __float_as_uint(__ldg(p.c.v_scale + si));
          if (!u.v) now.scale = __float_as_uint(__ldg(p.c.k_scale + si));
        }
        now.gone = __ballot_sync(0xFFFFFFFFu, !there) & 255u;
        now.tile = (int)tiles_before + u.tile;
        now.v = u.v;
        if (u.v) {  // a tile's values come after its keys
          if (u.tile & 1) pg1 = page_of(u.tile + 2);
          else pg0 = page_of(u.tile + 2);
        }
        if (unit + i > 0) publish(last, unit + i - 1);
        last = now;
      }
      unit += 2 * n;
      tiles_before += n;
    }
    if (unit > 0) publish(last, unit - 1);
    // an end for either group
    for (int i = 0; i < 2 && ok; ++i, ++unit) {
      const uint32_t slot = unit % KVW_META;
      if (unit >= KVW_META) ok = __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->meta_free[slot], ((unit / KVW_META) & 1) ^ 1, wc));
      if (!ok) break;
      if (lane == 0) {
        sh->meta[slot].flags = KVW_END;
        mbar_arrive(&sh->meta_full[slot]);
      }
      __syncwarp();
    }
  } else {
    // -------------------------------------------------------------- keys and values
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KVW_REGS_REST));
    // A warp takes KEYS keys of 16-code pieces at a time, every KVW_CONV_WARPS-th such step of a unit.
    // Codes are loaded AHEAD steps before they are expanded.
    constexpr int P16 = D / 16, KEYS = D == 64 ? 8 : D == 128 ? 4 : 2;
    constexpr int STEPS = 128 / KEYS, NP = (STEPS + KVW_CONV_WARPS - 1) / KVW_CONV_WARPS;
    constexpr int AHEAD = NP > 5 ? 5 : NP;
    static_assert(NP % AHEAD == 0, "whole rounds");
    // lane's key and piece: eight lanes that store together have four pieces of two keys, whose
    // swizzles differ in the lowest bit, so they meet no bank twice
    const int group = (warp - 10) / KVW_CONV_WARPS, cw = (warp - 10) % KVW_CONV_WARPS;
    const int k0 = D == 64 ? lane >> 2 : ((lane >> 2) & 1) + (D == 128 ? 2 * (lane >> 4) : 0);
    // (D = 192: the last eight lanes do what the eight before them do; left out, they made every
    // step a branch of its own: 2048 tokens, 64 heads over 12288 keys 3244 us, so 2446)
    const int c = D == 64 ? lane & 3 : (lane & 3) + 4 * (D == 128 ? (lane >> 3) & 1 : min(lane >> 3, P16 / 4 - 1));
    uint32_t code[AHEAD][4];
    const auto load = [&](int q, const KvwMeta& m, const uint8_t* src, uint32_t (&v)[4]) {
      const int step = cw + q * KVW_CONV_WARPS, key = step * KEYS;
      if (step < STEPS) kvw_load(v, src + (int64_t)m.place[(key >> 4) & 7] * (16 * D) + (key & 15) * D);
    };
    const auto source = [&](uint32_t flags) { return (flags & KVW_VALUES ? p.c.v8 : p.c.k8) + (k0 * D + c * 16); };
    const auto known = [&](uint32_t u, uint32_t* flags) {
      const bool ok = __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->meta_full[u % KVW_META], (u / KVW_META) & 1, wc));
      *flags = ok ? sh->meta[u % KVW_META].flags : KVW_END;
    };
    uint32_t unit = group, flags;
    known(unit, &flags);
    if (!(flags & KVW_END)) {
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) load(q, sh->meta[unit % KVW_META], source(flags), code[q]);
    }
    while (!(flags & KVW_END)) {
      const KvwMeta &m = sh->meta[unit % KVW_META], &next = sh->meta[(unit + 2) % KVW_META];
      uint32_t flags_next;
      known(unit + 2, &flags_next);
      const bool more = !(flags_next & KVW_END);
      const uint8_t *src = source(flags), *src_next = source(flags_next);
      const uint32_t slot = unit % UNITS;
      if (unit >= UNITS && !__all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->free[slot], ((unit / UNITS) & 1) ^ 1, wc))) break;
      uint8_t* dst = ring + slot * TILE + (c >> 2) * 16384 + k0 * 128;
      const auto store = [&](int step, const uint32_t (&x)[8]) {
        const int key = step * KEYS + k0, b = 2 * (c & 3);
        uint8_t* at = dst + step * KEYS * 128;
        *reinterpret_cast<uint4*>(at + ((b ^ (key & 7)) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<uint4*>(at + (((b + 1) ^ (key & 7)) << 4)) = make_uint4(x[4], x[5], x[6], x[7]);
      };
      const auto expand = [&](const uint32_t (&v)[4], uint32_t f, uint32_t (&x)[8]) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          x[2 * h] = mul_bf16x2(kvw_place(__byte_perm(v[h], 0, 0x4140)), f);
          x[2 * h + 1] = mul_bf16x2(kvw_place(__byte_perm(v[h], 0, 0x4342)), f);
        }
      };
      if (flags & KVW_PLAIN) {
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          const int step = cw + q * KVW_CONV_WARPS;
          uint32_t x[8];
          expand(code[q % AHEAD], m.factor[(step * KEYS >> 4) & 7], x);
          if (step < STEPS) store(step, x);
          if (q + AHEAD < NP) load(q + AHEAD, m, src, code[q % AHEAD]);
          else if (more) load(q + AHEAD - NP, next, src_next, code[q % AHEAD]);
        }
      } else {
        // large scales and marked blocks: rare, and read (again) one step at a time
#pragma unroll 1
        for (int q = 0; q < NP; ++q) {
          const int step = cw + q * KVW_CONV_WARPS;
          uint32_t v[4] = {0, 0, 0, 0}, x[8];
          load(q, m, src, v);
          expand(v, m.factor[(step * KEYS >> 4) & 7], x);
          const uint32_t sb = m.scale[(step * KEYS >> 4) & 7];
          float r1;
          kva_factor(sb, &r1);
          const uint32_t r2 = cvt_bf16x2(r1, r1);
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const uint32_t bits = (sb & 1u) ? kva_nan4_bits(v[h]) : 0u;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t z = mul_bf16x2(x[2 * h + y], r2);
              // a key's NaN goes into the scores, a value's is put into the outputs at the end
              const uint32_t nan = flags & KVW_VALUES ? 0u : 0x7FC0u;
              if ((bits >> (2 * y)) & 1u) z = (z & 0xFFFF0000u) | nan;
              if ((bits >> (2 * y + 1)) & 1u) z = (z & 0x0000FFFFu) | nan << 16;
              x[2 * h + y] = z;
            }
          }
          if (step < STEPS) store(step, x);
        }
        if (more) {
#pragma unroll
          for (int q = 0; q < AHEAD; ++q) load(q, next, src_next, code[q]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh->full[slot]);
        mbar_arrive(&sh->meta_free[unit % KVW_META]);
      }
      unit += 2;
      flags = flags_next;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc<1>(tmem, 512);
}

}  // namespace ks
