// Attention over the per-head cache for many query rows per key head: drafted trees of grouped
// heads, chunks of a prompt (kv_attn.cuh has the formulas, the numbers and the cut of the work).
//
// Rows are the MMA's M: S = Q K^T and O += P V on tcgen05 in bf16, scores, weights and outputs
// in tensor memory, the weights as the second product's A operand where the scores were. Keys
// and values come from the cache as codes in registers and are expanded to bf16 in shared
// memory on the way (4 KB of codes are read once per 256 rows; the expansion, ten integer
// operations per four codes, runs beside the products and takes about a third of their time).
//
// A CTA works on two streams of (scores, weights) so that one's softmax runs under the other's
// products:
//   D <= 128, more than 128 rows: a stream per 128 rows, on the same keys;
//   D <= 128, up to 128 rows: even and odd tiles of keys, each stream with references, sums and
//     outputs of its own, added up at the end of the row tile;
//   D > 128 (tensor memory holds one output): even and odd tiles, one output; one warpgroup does
//     the softmax of both in turn.
// Warps: 0-3 and 4-7 softmax (thread = row = TMEM lane), also queries and results; 8 issues the
// products; 9-16 load and expand. Codes of the next unit (the keys or the values of a tile) are in
// flight while one is expanded; units lie in a ring in the order the products take them.
//
// References are raised only when a score passes them by 2^KVA_RISE (rarely after the first
// tiles); then the row's output is scaled in place once its last product is done.
#pragma once
#include "kv_attn.cuh"

namespace ks {

constexpr int KVW_SOFT = 256;                       // softmax threads (the first ones)
constexpr int KVW_CONV = 256;                       // expanding threads (the last ones)
constexpr int KVW_THREADS = KVW_SOFT + 32 + KVW_CONV;
constexpr int KVW_UNITS = 8;                        // most units of the ring
constexpr int KVW_HDR = 6144;

template <int D>
constexpr int KVW_STREAM_OUT = D <= 128 ? 2 : 1;    // outputs in tensor memory
template <int D>
constexpr uint32_t KVW_TILE = 128u * D * 2;         // bytes of a unit, and of 128 queries
template <int D>
__host__ __device__ constexpr int kvw_units() {
  const int n = (int)((232448 - 1024 - KVW_HDR - KVW_STREAM_OUT<D> * KVW_TILE<D>) / KVW_TILE<D>);
  return n < KVW_UNITS ? n : KVW_UNITS;
}

struct KvwShared {
  KvaFind find;
  uint64_t full[KVW_UNITS], free[KVW_UNITS];
  uint64_t s_full[2], p_full[2], o_done[2];
  uint64_t q_full, q_free, drain;
  uint64_t pair_full, pair_free;  // the second stream's results are there / have been taken
  uint32_t tmem;
  int abort;
  uint32_t info[8];           // of a tile: bits 0-7 groups of 16 keys that are not there, 8-15 values marked
  float m[128], l[128];       // of the second stream, for the first
  uint32_t nan[128][8];
};
static_assert(sizeof(KvwShared) <= KVW_HDR, "KvwShared exceeds its header");

// D[tmem] (+)= A[tmem] * B[smem]^T, bf16 inputs, fp32 accumulate.
__device__ __forceinline__ void kvw_mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0;"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)
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
__device__ __noinline__ void kvw_nan_columns(const KvAttnParams& p, int b, int h, int len, int n, int t, int pos0,
                                             int keys, uint32_t groups, uint32_t (&mask)[D / 32]) {
  for (int g = 0; g < 8; ++g) {
    if (!((groups >> g) & 1u)) continue;
    const int at = pos0 + 16 * g, pi = kva_div(at, p.c.page, p.page_shift);
    const int pg = __ldg(p.c.table + (int64_t)b * p.c.max_pages + pi);
    const uint8_t* base = p.c.v8 + (((int64_t)pg * p.c.heads + h) * p.c.page + (at - pi * p.c.page)) * D;
    for (int k = 0; k < 16 && at + k < keys; ++k) {
      if (!kva_sees(p, b, len, n, t, at + k)) continue;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(base + k * D);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) bits |= kva_nan4_bits(__ldg(w + i * 8 + j)) << (4 * j);
        mask[i] |= bits;
      }
    }
  }
}

__device__ __forceinline__ float2 kvw_fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{ .reg .b64 w, x, y, z; mov.b64 w, {%2, %3}; mov.b64 x, {%4, %5}; mov.b64 y, {%6, %7};"
      " fma.rn.f32x2 z, w, x, y; mov.b64 {%0, %1}, z; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 kvw_add2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

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
      mbar_init(&sh->full[i], KVW_CONV / 32);
      mbar_init(&sh->free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
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
    p.owner[blockIdx.x] = make_int4(0, 0, 0, 0);
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
  const bool rows256 = p.nr == 256;

  if (warp < 8) {
    // -------------------------------------------------------------- softmax
    const int wg = warp >> 2, t128 = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t s_ph[2] = {0, 0};  // phases of the score buffers
    // products with the weights of either buffer so far.  A tile's scores come after the product
    // with the weights that were in their buffer before, so at most one of a buffer's products
    // is ever waited for, and its parity tells it.
    uint32_t o_count[2] = {0, 0};
    bool first = true;
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
      if (!first) {
        if (!mbar_wait(&sh->q_free, (item - 1) & 1, wc)) break;
      }
      first = false;
      if (!ONE_OUT || wg == 0) {
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
            *reinterpret_cast<uint4*>(dst + (u >> 3) * 16384 + rr * 128 + (((u & 7) ^ (rr & 7)) << 4)) = x;
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->q_full);
      }
      ++item;
      if (ONE_OUT && wg == 1) continue;
      // ------------------------------------------------------------ tiles of this warpgroup
      // two: all of them, in buffer wg; else every other one in buffer wg; one output: all, in
      // buffers by turns
      const int my_row = r0 + (rows256 ? wg * 128 : 0) + t128;
      const int tok = my_row / p.G;
      const int clear = w.len + (p.mask ? 0 : (my_row - t128) / p.G + 1);
      const int limit = tok < w.n ? (int)min((int64_t)w.len + (p.mask ? 0 : tok + 1), (int64_t)w.keys) : 0;
      const int step = ONE_OUT || two ? 1 : 2;
      const bool idle = rows256 && !two && wg == 1;
      float m = -INFINITY, l = 0.f;
      uint32_t nan[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) nan[i] = 0;
      int done = 0, last = wg;  // buffer of the last tile
      const uint32_t o_col = tmem + 256 + (ONE_OUT ? 0 : wg * D) + lanes;
      bool ok = true;
      // (a row tile of 256 rows whose second half is empty is done by even and odd tiles too:
      // both warpgroups then have the first 128 rows)
      const int row = idle ? my_row - 128 : my_row;
      const int tk = idle ? row / p.G : tok;
      const int cl = idle ? w.len + (p.mask ? 0 : r0 / p.G + 1) : clear;
      const int lm = idle ? (tk < w.n ? (int)min((int64_t)w.len + (p.mask ? 0 : tk + 1), (int64_t)w.keys) : 0) : limit;
      for (int j = step == 2 ? wg : 0; j < n; j += step, ++done) {
        const int buf = ONE_OUT ? (j & 1) : wg;
        const uint32_t s_col = tmem + buf * 128 + lanes;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sh->s_full[buf], s_ph[buf], wc));
        if (!ok) break;
        s_ph[buf] ^= 1;
        tc_fence_after();
        const int pos0 = (w.t0 + j) * 128;
        const uint32_t info = sh->info[(tiles_before + j) & 7];
        const bool open = pos0 + 128 <= cl && (info & 255u) == 0;
        // ---------------------------------------------------------- maximum
        // (a negative softmax scale makes the least product the largest score)
        float top = -INFINITY;
        uint32_t see[4] = {~0u, ~0u, ~0u, ~0u};
        const float sign = p.scale_log2 < 0.f ? -1.f : 1.f;
        if (!open) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int at = pos0 + 32 * c, k = lm - at;
            see[c] = k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1u;
            if (p.mask && tk < w.n)
              for (int i = max(w.len - at, 0); i < 32 && at + i < w.keys; ++i)
                if (kva_sees(p, w.b, w.len, w.n, tk, at + i)) see[c] |= 1u << i;
            if ((info >> (2 * c)) & 1u) see[c] &= 0xFFFF0000u;
            if ((info >> (2 * c + 1)) & 1u) see[c] &= 0x0000FFFFu;
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float x[32];
          tmem_ld32(s_col + 32 * c, reinterpret_cast<uint32_t*>(x));
          tmem_wait_ld();
          if (open && sign > 0.f) {
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, x[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if ((see[c] >> i) & 1u) top = fmaxf(top, x[i] * sign);
          }
        }
        top = top == -INFINITY ? top : top * fabsf(p.scale_log2);
        // ---------------------------------------------------------- raise the reference
        if (__any_sync(0xFFFFFFFFu, top > m + KVA_RISE)) {
          const float now = fmaxf(m, top);
          const float f = now == -INFINITY ? 1.f : kva_ex2(m - now);
          m = now;
          l *= f;
          if (done > 0) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sh->o_done[last], (o_count[last] - 1) & 1, wc));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float x[32];
              tmem_ld32(o_col + c, reinterpret_cast<uint32_t*>(x));
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] *= f;
              tmem_st16(o_col + c, reinterpret_cast<uint32_t*>(x));
              tmem_st16(o_col + c + 16, reinterpret_cast<uint32_t*>(x) + 16);
            }
            tmem_wait_st();
          }
        }
        // ---------------------------------------------------------- weights
        const float mu = (m == -INFINITY ? 0.f : m) + KVA_DOWN;
        const float2 sc = make_float2(p.scale_log2, p.scale_log2), minus = make_float2(-mu, -mu);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float x[32];
          tmem_ld32(s_col + 32 * c, reinterpret_cast<uint32_t*>(x));
          tmem_wait_ld();
          uint32_t e[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 y = kvw_fma2(make_float2(x[2 * i], x[2 * i + 1]), sc, minus);
            if (!open) {
              if (!((see[c] >> (2 * i)) & 1u)) y.x = -INFINITY;
              if (!((see[c] >> (2 * i + 1)) & 1u)) y.y = -INFINITY;
            }
            y = make_float2(kva_ex2(y.x), kva_ex2(y.y));
            sum = kvw_add2(sum, y);
            e[i] = cvt_bf16x2(y.x, y.y);
          }
          tmem_st16(s_col + 16 * c, e);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[buf]);
        ++o_count[buf];
        last = buf;
        l += sum.x + sum.y;
        if (info >> 8) kvw_nan_columns<D>(p, w.b, w.h, w.len, w.n, tk, pos0, w.keys, info >> 8, nan);
      }
      if (!ok) break;
      tiles_before += n;
      // ------------------------------------------------------------ results
      if (done > 0) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sh->o_done[last], (o_count[last] - 1) & 1, wc));
        tc_fence_after();
      }
      if (!ONE_OUT && !two) {
        // even and odd tiles together: the first warpgroup takes the second's
        if (wg == 1) {
          sh->m[t128] = m;
          sh->l[t128] = l;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) sh->nan[t128][i] = nan[i];
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->pair_full);
          // its output is the first warpgroup's to read until here
          ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(&sh->pair_free, pair_ph, wc));
        } else {
          ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(&sh->pair_full, pair_ph, wc));
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
          f0 = now == -INFINITY ? 1.f : kva_ex2(m - now);
          f1 = now == -INFINITY ? 1.f : kva_ex2(m1 - now);
          l = l * f0 + l1 * f1;
          m = now;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) nan[i] |= sh->nan[t128][i];
        }
        const bool whole = w.whole(), in = row < p.rows;
        const int g = row - tk * p.G;
        float f = 1.f;
        if (whole)
          f = kva_norm(m, l, in && p.sink ? __ldg(p.sink + w.h * p.G + g) * 1.4426950408889634f : 0.f, in && p.sink);
        uint16_t* orow = p.out + (((int64_t)w.b * p.c.T + tk) * p.H + w.h * p.G + g) * D;
        const int64_t prow = (int64_t)w.slot() * p.nr + (row - r0);
#pragma unroll
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
          if (nan[c / 32]) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if ((nan[c / 32] >> i) & 1u) x[i] = __uint_as_float(0x7FC00000u);
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
          if (tid == 0 && w.t0 == 0) p.owner[blockIdx.x] = make_int4(w.b, w.rt, w.h, w.parts(sh->find.per));
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
    const bool leader = elect_one();
    uint32_t unit = 0, q_ph = 0, p_ph[2] = {0, 0};
    constexpr uint32_t idesc_s = idesc_bf16_f32(128, 128, false, false);
    constexpr uint32_t idesc_o = idesc_bf16_f32(128, D, false, true);
    bool ok = true;
    const auto wait = [&](uint64_t* bar, uint32_t ph) {
      ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(bar, ph, wc));
      tc_fence_after();
      return ok;
    };
    const auto qk = [&](int buf, int qt, uint32_t slot) {
      if (leader) {
        const uint32_t a = smem_u32(qs + qt * TILE), b = smem_u32(ring + slot * TILE);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = (ks >> 2) * 16384 + (ks & 3) * 32;
          umma_bf16_ss(tmem + buf * 128, sdesc_sw128(a + off, 16, 1024), sdesc_sw128(b + off, 16, 1024), idesc_s, ks > 0);
        }
        umma_commit(&sh->s_full[buf]);
      }
      __syncwarp();
    };
    const auto pv = [&](int buf, int out, uint32_t slot, bool acc) {
      if (leader) {
        const uint32_t b = smem_u32(ring + slot * TILE);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          kvw_mma_ts(tmem + 256 + out * D, tmem + buf * 128 + ks * 8, sdesc_sw128(b + ks * 2048, 16384, 1024), idesc_o,
                     acc || ks > 0);
        umma_commit(&sh->o_done[buf]);
      }
      __syncwarp();
    };
    const auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
      __syncwarp();
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
      uint32_t s0, s1;
      if (two) {
        if (!take(0, &s0)) break;
        qk(0, 0, s0);
        qk(1, 1, s0);
        commit(&sh->free[s0]);
        if (n == 1) commit(&sh->q_free);
        for (int j = 0; j < n && ok; ++j) {
          if (!take(2 * j + 1, &s0)) break;
          for (int s = 0; s < 2; ++s) {
            if (!wait(&sh->p_full[s], p_ph[s])) break;
            p_ph[s] ^= 1;
            pv(s, s, s0, j > 0);
            if (s == 1) commit(&sh->free[s0]);
            if (j + 1 < n) {
              if (s == 0 && !take(2 * j + 2, &s1)) break;
              qk(s, s, s1);
              if (s == 1) {
                commit(&sh->free[s1]);
                if (j + 2 == n) commit(&sh->q_free);
              }
            }
          }
        }
      } else {
        for (int j = 0; j < min(n, 2) && ok; ++j) {
          if (!take(j, &s0)) break;
          qk(j, 0, s0);
          commit(&sh->free[s0]);
          if (j + 1 == n) commit(&sh->q_free);
        }
        for (int j = 0; j < n && ok; ++j) {
          const int s = j & 1;
          // values of tile j: unit 1 of a single tile; else 2 + 2 j, the last one 2 n - 1
          if (!take(n == 1 ? 1 : j + 1 == n ? 2 * n - 1 : 2 + 2 * j, &s0)) break;
          if (!wait(&sh->p_full[s], p_ph[s])) break;
          p_ph[s] ^= 1;
          pv(s, ONE_OUT ? 0 : s, s0, ONE_OUT ? j > 0 : j > 1);
          commit(&sh->free[s0]);
          if (j + 2 < n) {
            if (!take(2 * j + 3, &s0)) break;
            qk(s, 0, s0);
            commit(&sh->free[s0]);
            if (j + 3 == n) commit(&sh->q_free);
          }
        }
      }
      unit += 2 * n;
    }
    // every product and arrival in flight has landed before the CTA gives its memory back
    commit(&sh->drain);
    mbar_wait(&sh->drain, 0, wc, false, true);
  } else {
    // -------------------------------------------------------------- keys and values
    constexpr int P16 = D / 16;                    // 16-code pieces of a row
    constexpr int NP = 128 * P16 / KVW_CONV;       // pieces of a thread per unit
    const int ct = tid - (KVW_SOFT + 32), cw = ct >> 5;
    const int per_page = p.c.page / p.c.block;
    uint32_t unit = 0, tiles_before = 0;
    bool ok = true;
    for (; w.left > 0 && ok; w.next(p)) {
      if (!w.any()) continue;
      const int n = w.t1 - w.t0;
      const bool two = rows256 && w.rt * 256 + 128 < p.rows;
      // lanes 0-7: a group of 16 keys of the tile each
      struct Group {
        int64_t row;      // of the page pool's rows of heads
        uint32_t scale;   // bits, 0: not there
      };
      const auto page_of = [&](int tile) {
        const int pos = (w.t0 + tile) * 128 + 16 * lane;
        return lane < 8 && tile < n && pos < w.keys
                   ? __ldg(p.c.table + (int64_t)w.b * p.c.max_pages + kva_div(pos, p.c.page, p.page_shift)) : -2;
      };
      uint32_t info_next = 0;
      const auto locate = [&](const KvwUnit& u, int pg, Group* g) {
        const int pos = (w.t0 + u.tile) * 128 + 16 * lane;
        const bool ok_pg = pg >= 0 && pg < p.c.n_pages;
        if (pg != -2 && !ok_pg && cw == 0) report_bounds(p.c.status, w.b, (int)p.c.n_pages);
        const int in = ok_pg ? pos - kva_div(pos, p.c.page, p.page_shift) * p.c.page : 0;
        const int64_t at = (int64_t)(ok_pg ? pg : 0) * p.c.heads + w.h;
        g->row = at * p.c.page + in;
        const int64_t si = at * per_page + kva_div(in, p.c.block, p.block_shift);
        const uint32_t vs = ok_pg ? __float_as_uint(__ldg(p.c.v_scale + si)) : 0u;
        if (u.v) {
          g->scale = vs;
        } else {
          g->scale = ok_pg ? __float_as_uint(__ldg(p.c.k_scale + si)) : 0u;
          info_next = (__ballot_sync(0xFFFFFFFFu, !ok_pg) & 255u) | (__ballot_sync(0xFFFFFFFFu, ok_pg && (vs & 1u)) & 255u) << 8;
        }
      };
      uint32_t code[NP][4];
      const auto load = [&](const KvwUnit& u, const Group& g) {
        const uint8_t* src = u.v ? p.c.v8 : p.c.k8;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int e = ct + i * KVW_CONV, key = e / P16, c = e - key * P16;
          const int64_t row = __shfl_sync(0xFFFFFFFFu, g.row, key >> 4);
          kvf_load<4>(code[i], src + (row + (key & 15)) * D + c * 16);
        }
      };
      KvwUnit u = kvw_unit(0, n, two), v{};
      // page numbers of the tiles to come, by tile parity
      int pg[2] = {page_of(0), page_of(1)};
      Group g{}, gn{};
      locate(u, pg[0], &g);
      uint32_t info = info_next;
      load(u, g);
      for (int i = 0; i < 2 * n; ++i) {
        const uint32_t slot = (unit + i) % UNITS, ph = ((unit + i) / UNITS) & 1;
        if (unit + i >= UNITS) {
          ok = __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->free[slot], ph ^ 1, wc));
          if (!ok) break;
        }
        uint8_t* dst = ring + slot * TILE;
        const bool more = i + 1 < 2 * n;
        if (more) {
          v = kvw_unit(i + 1, n, two);
          locate(v, pg[v.tile & 1], &gn);
          if (v.v) pg[v.tile & 1] = page_of(v.tile + 2);  // a tile's values come after its keys
        }
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          const int e = ct + q * KVW_CONV, key = e / P16, c = e - key * P16;
          const uint32_t sb = __shfl_sync(0xFFFFFFFFu, g.scale, key >> 4);
          float rest;
          const uint32_t f = kva_factor(sb, &rest);
          uint32_t x[8];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const uint32_t wd = code[q][h];
            x[2 * h] = mul_bf16x2(kva_place(__byte_perm(wd, 0, 0x1404)), f);
            x[2 * h + 1] = mul_bf16x2(kva_place(__byte_perm(wd, 0, 0x3424)), f);
          }
          if (rest != 1.f || (sb & 1u)) {
            const uint32_t r2 = cvt_bf16x2(rest, rest);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const uint32_t bits = (sb & 1u) ? kva_nan4_bits(code[q][h]) : 0u;
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                uint32_t z = mul_bf16x2(x[2 * h + y], r2);
                // a key's NaN goes into the scores, a value's is put into the outputs at the end
                const uint32_t nan = u.v ? 0u : 0x7FC0u;
                if ((bits >> (2 * y)) & 1u) z = (z & 0xFFFF0000u) | nan;
                if ((bits >> (2 * y + 1)) & 1u) z = (z & 0x0000FFFFu) | nan << 16;
                x[2 * h + y] = z;
              }
            }
          }
          // (neighbouring lanes' halves the other way round: no two of a phase meet a bank)
          uint8_t* at = dst + (c >> 2) * 16384 + key * 128;
          const int a = 2 * (c & 3), flip = (c >> 2) & 1;
          const uint4 lo = make_uint4(x[0], x[1], x[2], x[3]), hi = make_uint4(x[4], x[5], x[6], x[7]);
          *reinterpret_cast<uint4*>(at + (((a + flip) ^ (key & 7)) << 4)) = flip ? hi : lo;
          *reinterpret_cast<uint4*>(at + (((a + 1 - flip) ^ (key & 7)) << 4)) = flip ? lo : hi;
        }
        if (!u.v && cw == 0 && lane == 0) sh->info[(tiles_before + u.tile) & 7] = info;
        if (more) load(v, gn);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->full[slot]);
        u = v;
        g = gn;
        info = info_next;
      }
      unit += 2 * n;
      tiles_before += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc<1>(tmem, 512);
}

}  // namespace ks
