// Attention of drafted tokens over the quantised latent cache.
//
//   s[k] = scale * q . c_k,  o = sum_k exp(s_k - m) v_k / (sum_k exp(s_k - m) + exp(sink - m))
//
// with c_k the cached row of position k (latent_cache.cuh), v_k its first dv columns.
// A drafted token of sequence b sees the lens[b] cached positions and, among the T
// drafted rows that follow them in the cache, those its row of the mask allows (without
// a mask: itself and the ones before it).
//
// The T * H query rows of a sequence share its cached rows, so the product is run with
// keys as the MMA's M dimension (tcgen05, bf16 operands, fp32 accumulators in TMEM):
//   S^T[128 keys, NR rows] = K . Q^T         O^T[dv, NR rows] += V^T . P^T
// K and V are one tile in shared memory: the e4m3 codes are expanded to bf16 (exactly,
// their scale included) once, stored 128-byte swizzled, and read K-major by the first
// product and MN-major (dims contiguous) by the second.  NR = 16, 32 or 64 rows.
//
// Work: a unit is one 128-key tile of one (sequence, NR-row tile).  All units of the
// call in order are cut into equal stretches, one per CTA, whatever the lengths (which
// only the device knows), so a long context is split over the SMs and ragged batches
// balance.  A row tile that spans CTAs leaves (maximum, sum, unnormalised output) per
// part in the workspace; tree_attn_join_kernel adds them up in order (no atomics).
//
// Warps: 8 softmax warps (thread = key = TMEM lane; two warps share a lane quarter and
// split the rows), 8 loader warps, 1 MMA / query-TMA warp.  Two threads load a key: its
// codes for the next tile wait in registers while this tile's are expanded, so the memory
// latency passes behind a whole tile's work.  A 64-column chunk (16 KB) of the tile is
// refilled as soon as the last product that reads it is done.
//
// Softmax: the running maximum of a row is only raised when a score passes it by 2^8
// (one vote per tile); p = 2^(s - m) is then at most 256, fp32 sums are kept per thread
// and reduced once per row tile.
#pragma once
#include "latent_cache.cuh"
#include "sparse_attn.cuh"
#include "sparse_attn_small.cuh"

namespace ks {

constexpr int TA_SOFT = 256;                 // softmax threads (warps 0-7)
constexpr int TA_LOAD = 256;                 // loader threads (warps 8-15)
constexpr int TA_THREADS = TA_SOFT + TA_LOAD + 32;
constexpr int TA_MAX_CHUNKS = 9;             // 64-column chunks of a row
constexpr int TA_MAX_CTAS = 148;             // SMs of a B200: bounds the workspace
constexpr int TA_MAX_ROWS = 64;
constexpr int TA_HDR = 4096;
constexpr float TA_GROW = 8.f;               // log2 of how far scores may pass the maximum

struct TreeAttnParams {
  const uint8_t* kv8;
  const float* scale;
  const uint16_t* tail;
  int64_t n_pages, max_pages;
  int32_t page, dq, dr;
  const int32_t* table;   // [B, max_pages]
  const int32_t* lens;    // [B]
  const uint8_t* mask;    // [B, T, T] or null
  const float* sink;      // [H] or null
  uint16_t* out;          // bf16 [B, T, H, dv]
  int32_t B, T, H, dv;
  int32_t rows;           // T * H
  int32_t row_tiles;      // ceil(rows / NR)
  int32_t nq, nkb, nka;   // e4m3 chunks, all chunks, chunk slots of a stage
  int32_t dv_tiles;       // 128-row M tiles of O^T
  int32_t stages;         // K tiles in shared memory (1 or 2)
  int32_t p_alias;        // P lies in the last (key-only) chunk
  uint32_t k_off, q_off, p_off;
  uint32_t tmem_cols;
  float scale_log2;
  float* part_o;          // [2 * CTAs][NR][dv]
  float* part_ml;         // [2 * CTAs][NR][2]
  int32_t* owner;         // [CTAs][4]: sequence, row tile, parts of the item whose head is here
  int* status;
  uint64_t budget_ns;
};

struct TaShared {
  uint64_t full[2][TA_MAX_CHUNKS];  // a chunk has been written
  uint64_t vfree[2][4];             // the PV products of a 128-dim tile are done
  uint64_t s_full[2];               // scores of a tile are in TMEM (and its K reads done)
  uint64_t p_full[2];               // P of a tile is in shared memory
  uint64_t pv_done[2];              // all PV products of a tile are done
  uint64_t q_full, drain;
  uint32_t tmem_base;
  int abort;
  int64_t total, per;
  int32_t b0, rt0, t0;              // where this CTA's stretch starts
  alignas(16) float m[TA_MAX_ROWS]; // running maximum per row (base 2)
  alignas(16) float mneg[TA_MAX_ROWS];  // its negative (read as float4)
  float f[TA_MAX_ROWS];             // factor of a raise; at the end 1 / sum
  float red[4][TA_MAX_ROWS];
  uint8_t flag[2][128];             // key: 0 fine, 1 absent, 2 marked (scale NaN)
};
static_assert(sizeof(TaShared) <= TA_HDR, "TaShared exceeds its header");

// Keys of sequence b: its cached positions and drafted rows, within the page table.
__device__ __forceinline__ int ta_len(const TreeAttnParams& p, int b) { return max(0, __ldg(p.lens + b)); }
__device__ __forceinline__ int ta_keys(const TreeAttnParams& p, int len) {
  const int64_t cap = p.max_pages * p.page;
  return (int)min((int64_t)len + p.T, cap);
}
__device__ __forceinline__ int ta_tiles(const TreeAttnParams& p, int len) { return (ta_keys(p, len) + 127) >> 7; }

// A CTA's stretch of units, walked by every role on its own.
struct TaWalk {
  int left;       // units from here to the end of the stretch
  int b, rt, t;   // this unit
  int len, nt;    // of sequence b
  __device__ __forceinline__ void start(const TreeAttnParams& p, const TaShared* sh) {
    const int64_t u0 = (int64_t)blockIdx.x * sh->per;
    left = (int)min(sh->per, sh->total - u0);
    b = sh->b0; rt = sh->rt0; t = sh->t0;
    if (left > 0) {
      len = ta_len(p, b);
      nt = ta_tiles(p, len);
    }
  }
  // units of this row tile that are in the stretch, from here
  __device__ __forceinline__ int here() const { return min(nt - t, left); }
  __device__ __forceinline__ void next_item(const TreeAttnParams& p, int done) {
    left -= done;
    t = 0;
    if (left > 0 && ++rt == p.row_tiles) {
      rt = 0;
      ++b;
      len = ta_len(p, b);
      nt = ta_tiles(p, len);
    }
  }
  __device__ __forceinline__ void next_unit(const TreeAttnParams& p) {
    if (t + 1 < nt) {
      ++t;
      --left;
    } else {
      next_item(p, 1);
    }
  }
};

// Slot of the page pool that holds this position, -1 for none (a pool has < 2^31 slots).
__device__ __forceinline__ int ta_slot(const TreeAttnParams& p, const TaWalk& w, int key) {
  const int pos = w.t * 128 + key;
  if (w.left <= 0 || pos >= ta_keys(p, w.len)) return -1;
  return (int)cache_row(p.table, p.max_pages, p.n_pages, p.page, w.b, pos, p.status);
}

// Two e4m3 codes (bytes of w picked by SEL) as bf16, times the powers of two in `mul`.
// A code's exponent and mantissa moved to their places in bf16 give its value times
// 2^-120 (bf16's bias is 120 more than e4m3's; subnormals included), so the one exact
// product with 2^120 * scale is the value.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t ta_expand(uint32_t w, uint32_t mul) {
  const uint32_t t = __byte_perm(w, 0, SEL);
  return mul_bf16x2((t & 0x80008000u) | ((t >> 4) & 0x07F007F0u), mul);
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ldn(uint32_t taddr, uint32_t* r) {
  if constexpr (N == 8) tmem_ld8(taddr, r);
  else if constexpr (N == 16) tmem_ld16(taddr, r);
  else tmem_ld32(taddr, r);
}
// Any thread of the softmax warps (also a barrier among them).
__device__ __forceinline__ bool soft_any(bool x) {
  uint32_t r;
  asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.or.pred q, 1, %2, p; selp.u32 %0, 1, 0, q; }"
               : "=r"(r)
               : "r"((uint32_t)x), "n"(TA_SOFT)
               : "memory");
  return r != 0;
}
__device__ __forceinline__ void soft_sync() { named_bar_sync(1, TA_SOFT); }

// Max or sum over the warp's lanes of CW values each into red[.. + c], c < CW.
template <bool MX, int CW>
__device__ __forceinline__ void ta_reduce(const float (&v)[CW], float* red, int lane) {
#pragma unroll
  for (int g = 0; g < CW; g += 16) {
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = g + i < CW ? v[(g + i) % CW] : 0.f;
    const float r = reduce16_lanes<MX>(w, lane);  // value g + (lane >> 1)
    if ((lane & 1) == 0 && g + (lane >> 1) < CW) red[g + (lane >> 1)] = r;
  }
}

template <int NR, int NQ>
__global__ void __launch_bounds__(TA_THREADS, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap qm, const TreeAttnParams p) {
  constexpr int CW = NR / 2;  // rows of a softmax thread
  extern __shared__ uint8_t ta_raw[];
  const uint32_t raw = smem_u32(ta_raw);
  uint8_t* smem = ta_raw + (((raw + 1023u) & ~1023u) - raw);
  TaShared* sh = reinterpret_cast<TaShared*>(smem);
  uint8_t* ks_ = smem + p.k_off;  // [stages][nka][128 keys x 128 B]
  uint8_t* qs = smem + p.q_off;   // [nkb][NR rows x 128 B]
  uint8_t* ps = smem + p.p_off;   // [stages][128 keys x 128 B], rows contiguous (MN-major)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  WaitCtx wc{&sh->abort, p.status, p.budget_ns};

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      for (int c = 0; c < TA_MAX_CHUNKS; ++c) mbar_init(&sh->full[s][c], TA_LOAD / 32);
      for (int m = 0; m < 4; ++m) mbar_init(&sh->vfree[s][m], 1);
      mbar_init(&sh->s_full[s], 1);
      mbar_init(&sh->p_full[s], TA_SOFT / 32);
      mbar_init(&sh->pv_done[s], 1);
    }
    mbar_init(&sh->q_full, 1);
    mbar_init(&sh->drain, 1);
    sh->abort = 0;
    fence_barrier_init();
    p.owner[(int64_t)blockIdx.x * 4 + 2] = 0;  // no row tile's head here yet
  }
  if (threadIdx.x < TA_MAX_ROWS) {
    sh->m[threadIdx.x] = -INFINITY;
    sh->mneg[threadIdx.x] = INFINITY;
  }
  if (warp == 16) {
    tmem_alloc<1>(&sh->tmem_base, p.tmem_cols);
    tmem_relinquish<1>();
    if (lane == 0) tma_prefetch_desc(&qm);
  }
  if (warp == 8) {  // the call's units, and where this CTA's stretch starts
    int64_t total = 0;
    for (int i = 0; i < p.B; i += 32) {
      int64_t n = 0;
      if (i + lane < p.B) {
        const int len = ta_len(p, i + lane);
        n = ta_tiles(p, len);
        if (blockIdx.x == 0 && (int64_t)len + p.T > p.max_pages * p.page)  // past the table
          report_bounds(p.status, i + lane, (int)p.max_pages);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
      total += n * p.row_tiles;
    }
    const int64_t per = (total + gridDim.x - 1) / gridDim.x;
    const int64_t u0 = (int64_t)blockIdx.x * per;
    int64_t at = 0;
    for (int i = 0; i < p.B && u0 < total; i += 32) {
      const int64_t nt = i + lane < p.B ? ta_tiles(p, ta_len(p, i + lane)) : 0;
      int64_t n = nt * p.row_tiles;  // inclusive sums of the 32 sequences
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xFFFFFFFFu, n, o);
        if (lane >= o) n += v;
      }
      const uint32_t over = __ballot_sync(0xFFFFFFFFu, at + n > u0);
      if (over) {
        if (lane == __ffs(over) - 1) {
          const int64_t in = u0 - (at + n - nt * p.row_tiles);
          sh->b0 = i + lane;
          sh->rt0 = (int)(in / nt);
          sh->t0 = (int)(in % nt);
        }
        break;
      }
      at += __shfl_sync(0xFFFFFFFFu, n, 31);
    }
    if (lane == 0) {
      sh->total = total;
      sh->per = per;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const uint32_t o_col = (uint32_t)(p.stages * NR);
  const int two = p.stages == 2;
  TaWalk w;
  w.start(p, sh);

  if (warp >= 8 && warp < 16) {
    // ================================================================ loaders
    const int lt = threadIdx.x - TA_SOFT, key = lt >> 1, half = lt & 1;
    // r[c]: the codes of chunk c.  The bf16 tail (two chunks' worth of registers) borrows
    // r[0] and r[1] between their use in this unit and their load for the next.
    static_assert(NQ >= 2, "the tail borrows two chunks' registers");
    uint4 r[NQ][2];
    const int last_free = 2 * p.dv_tiles;  // chunks from here on are read by QK only
    TaWalk a = w;                          // the walk of the row addresses: one unit ahead
    int slot = ta_slot(p, a, key), next;
    auto load8 = [&](int c, int s) {
      const uint8_t* g = p.kv8 + (int64_t)s * p.dq + c * 64 + half * 32;
      r[c][0] = ldcg_or_zero(g, s >= 0 && c < p.nq);
      r[c][1] = ldcg_or_zero(g + 16, s >= 0 && c < p.nq);
    };
    auto load_scale = [&](int s) { return __float_as_uint(s >= 0 ? __ldg(p.scale + s) : 0.f); };
#pragma unroll
    for (int c = 0; c < NQ; ++c) load8(c, slot);
    uint32_t sb = load_scale(slot);
    a.next_unit(p);
    next = ta_slot(p, a, key);
    const uint32_t row = (uint32_t)(key * 128), sw = (uint32_t)(key & 7);
    const uint32_t units = (uint32_t)max(w.left, 0);
    bool ok = true;
    for (uint32_t g = 0; g < units && ok; ++g) {
      const int st = two ? (int)(g & 1) : 0;
      const uint32_t use = two ? g >> 1 : g;
      uint8_t* tile = ks_ + (size_t)st * p.nka * 16384 + row;
      const bool bad = (sb & 0x7F800000u) == 0x7F800000u;
      // 2^120 * scale, or two factors where that is beyond bf16
      const int e = (int)((sb >> 23) & 255) + 120;
      const bool fine = slot >= 0 && !bad && (sb & 0x7F800000u) != 0;
      const uint32_t m1 = fine ? (uint32_t)min(e, 254) * 0x00800080u : 0u;
      const bool big = __any_sync(0xFFFFFFFFu, fine && e > 254);
      const uint32_t m2 = (uint32_t)(max(e, 254) - 254 + 127) * 0x00800080u;
      sb = load_scale(next);
      auto wait_free = [&](int cc) {  // the last products that read this chunk slot are done
        if (use > 0) {
          uint64_t* bar = cc < last_free ? &sh->vfree[st][cc >> 1] : p.p_alias ? &sh->pv_done[st] : &sh->s_full[st];
          ok = mbar_wait_inl(bar, (use - 1) & 1, wc) && ok;
        }
      };
      auto filled = [&](int cc) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->full[st][cc]);
      };
#pragma unroll
      for (int c = 0; c < NQ; ++c) {
        if (c < p.nq) {
          wait_free(c);
          if (c == 0 && half == 0) sh->flag[st][key] = slot < 0 ? 1 : bad ? 2 : 0;
          uint8_t* dst = tile + c * 16384;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 v = r[c][i >> 1];
            const uint32_t wa = i & 1 ? v.z : v.x, wb = i & 1 ? v.w : v.y;
            uint4 o;
            o.x = ta_expand<0x1404>(wa, m1);
            o.y = ta_expand<0x3424>(wa, m1);
            o.z = ta_expand<0x1404>(wb, m1);
            o.w = ta_expand<0x3424>(wb, m1);
            if (big) {
              o.x = mul_bf16x2(o.x, m2);
              o.y = mul_bf16x2(o.y, m2);
              o.z = mul_bf16x2(o.z, m2);
              o.w = mul_bf16x2(o.w, m2);
            }
            *reinterpret_cast<uint4*>(dst + (((uint32_t)(half * 4 + i) ^ sw) << 4)) = o;
          }
          filled(c);
        }
        // the next unit's codes take this chunk's registers
        if (c >= 2) {
          load8(c, next);
        } else if (c == 1) {
          const uint16_t* tg = p.tail + (int64_t)slot * p.dr + half * 32;
#pragma unroll
          for (int i = 0; i < 4; ++i) r[i >> 1][i & 1] = ldcg_or_zero(tg + i * 8, slot >= 0 && p.dr > 0 && !bad);
        }
      }
      if (p.dr > 0) {
        wait_free(p.nq);
        uint8_t* dst = tile + p.nq * 16384;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(dst + (((uint32_t)(half * 4 + i) ^ sw) << 4)) = r[i >> 1][i & 1];
        filled(p.nq);
      }
      load8(0, next);
      load8(1, next);
      slot = next;
      a.next_unit(p);
      next = ta_slot(p, a, key);
    }
  } else if (warp == 16) {
    // ================================================================ MMA issue
    if (elect_one()) {
      const uint32_t id_qk = idesc_bf16_f32(128, NR, false, false), id_pv = idesc_bf16_f32(128, NR, true, true);
      uint32_t g = 0, items = 0;
      bool ok = true;
      // the item's query rows (rows past it are other rows or zeros: their columns are not used)
      auto load_q = [&](const TaWalk& x) {
        mbar_expect_tx(&sh->q_full, (uint32_t)p.nkb * NR * 128);
        const int y = x.b * p.rows + x.rt * NR;
        for (int c = 0; c < p.nkb; ++c) tma_load_2d(&qm, &sh->q_full, qs + c * NR * 128, c * 64, y);
      };
      auto qk = [&](uint32_t g) {
        const int st = two ? (int)(g & 1) : 0;
        const uint32_t use = two ? g >> 1 : g;
        for (int c = 0; c < p.nkb && ok; ++c) {
          ok = mbar_wait_inl(&sh->full[st][c], use & 1, wc);
          if (!ok) return;
          tc_fence_after();
          const uint64_t ad = sdesc_sw128(smem_u32(ks_ + ((size_t)st * p.nka + c) * 16384), 16, 1024);
          const uint64_t bd = sdesc_sw128(smem_u32(qs + c * NR * 128), 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16_ss(tmem + st * NR, ad + k * 2, bd + k * 2, id_qk, c > 0 || k > 0 ? 1u : 0u);
        }
        umma_commit(&sh->s_full[st]);
      };
      auto pv = [&](uint32_t g, bool first) {
        const int st = two ? (int)(g & 1) : 0;
        const uint32_t use = two ? g >> 1 : g;
        ok = mbar_wait_inl(&sh->p_full[st], use & 1, wc);
        if (!ok) return;
        tc_fence_after();
        const uint64_t bd = sdesc_sw128(smem_u32(ps + st * 16384), 16, 1024);
        for (int m = 0; m < p.dv_tiles; ++m) {
          const uint64_t ad = sdesc_sw128(smem_u32(ks_ + ((size_t)st * p.nka + 2 * m) * 16384), 16384, 1024);
#pragma unroll
          for (int k = 0; k < 8; ++k)  // 16 keys: 2048 bytes further in both
            umma_bf16_ss(tmem + o_col + m * NR, ad + k * 128, bd + k * 128, id_pv, !first || k > 0 ? 1u : 0u);
          umma_commit(&sh->vfree[st][m]);
        }
        umma_commit(&sh->pv_done[st]);
      };
      bool q_wait = false;
      while (w.left > 0 && ok) {
        const int n = w.here();
        if (g > 0) {  // the previous item's QK products have read its query rows
          const uint32_t l = g - 1;
          ok = mbar_wait_inl(&sh->s_full[two ? l & 1 : 0], (two ? l >> 1 : l) & 1, wc);
          if (!ok) break;
        }
        load_q(w);
        q_wait = true;
        ok = mbar_wait_inl(&sh->q_full, items & 1, wc);
        if (!ok) break;
        q_wait = false;
        if (two) {
          qk(g);
          for (int i = 0; i < n && ok; ++i) {
            if (i + 1 < n) qk(g + i + 1);
            if (ok) pv(g + i, i == 0);
          }
        } else {
          for (int i = 0; i < n && ok; ++i) {
            qk(g + i);
            if (ok) pv(g + i, i == 0);
          }
        }
        g += n;
        ++items;
        w.next_item(p, n);
      }
      // nothing of this CTA is in flight when it gives its memory back
      if (q_wait) mbar_wait(&sh->q_full, items & 1, wc, false, true);
      umma_commit(&sh->drain);
      mbar_wait(&sh->drain, 0, wc, false, true);
    }
    __syncwarp();
  } else {
    // ================================================================ softmax, epilogue
    // After a wait ran out (abort) the loops run on without waiting, so the warps keep
    // meeting at their barriers; nothing here indexes by data.
    const int quarter = warp & 3, hc = (warp >> 2) * CW;  // first row of this thread
    const int key = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    uint32_t g = 0;
    while (w.left > 0) {
      const int n = w.here();
      const int r0 = w.rt * NR;                      // first row of the tile in the sequence
      const int nrows = min(NR, p.rows - r0);
      const bool whole = w.t == 0 && n == w.nt;      // no other CTA has a part
      float l[CW];
#pragma unroll
      for (int i = 0; i < CW; ++i) l[i] = 0.f;
      for (int i = 0; i < n; ++i, ++g) {
        const int st = two ? (int)(g & 1) : 0;
        const uint32_t use = two ? g >> 1 : g;
        const int tile = w.t + i;
        // what this key's column entries may be: ~0 everything, else a bit per row
        uint32_t allow = 0xFFFFFFFFu;
        const int pos = tile * 128 + key, j = pos - w.len;
        if (j >= 0) {  // a drafted row, or past them (absent)
          allow = 0;
          if (j < p.T) {
            int t = (r0 + hc) / p.H, h = (r0 + hc) - t * p.H;
            const uint8_t* mk = p.mask + ((int64_t)w.b * p.T) * p.T + j;
            uint32_t bit = 0;
            bool fresh = true;
#pragma unroll 1
            for (int c = 0; c < CW; ++c) {
              if (fresh) bit = t < p.T && (p.mask ? mk[(int64_t)t * p.T] != 0 : j <= t);
              allow |= bit << c;
              fresh = ++h == p.H;
              if (fresh) {
                h = 0;
                ++t;
              }
            }
          }
        }
        mbar_wait(&sh->full[st][0], use & 1, wc);  // the key's flag
        const int flag = sh->flag[st][key];
        if (flag == 1) allow = 0;
        mbar_wait(&sh->s_full[st], use & 1, wc);
        tc_fence_after();
        constexpr uint32_t ALL = CW == 32 ? 0xFFFFFFFFu : (1u << CW) - 1u;
        const bool plain = __all_sync(0xFFFFFFFFu, (allow & ALL) == ALL && flag == 0);
        // exponents: scaled score minus the row's maximum
        float d[CW];
        auto exponents = [&] {
          uint32_t s[CW];
          tmem_ldn<CW>(tmem + st * NR + hc + lane_off, s);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < CW; c += 4) {
            const float4 mn = *reinterpret_cast<const float4*>(&sh->mneg[hc + c]);
            d[c] = fmaf(__uint_as_float(s[c]), p.scale_log2, mn.x);
            d[c + 1] = fmaf(__uint_as_float(s[c + 1]), p.scale_log2, mn.y);
            d[c + 2] = fmaf(__uint_as_float(s[c + 2]), p.scale_log2, mn.z);
            d[c + 3] = fmaf(__uint_as_float(s[c + 3]), p.scale_log2, mn.w);
          }
          if (!plain) {
#pragma unroll
            for (int c = 0; c < CW; ++c)
              d[c] = !((allow >> c) & 1u) ? -INFINITY : flag == 2 ? __uint_as_float(0x7FC00000u) : d[c];
          }
        };
        exponents();
        // a score past the row's maximum by more than TA_GROW?
        bool need = false;
#pragma unroll
        for (int c = 0; c < CW; ++c) need |= d[c] > TA_GROW;
        if (soft_any(need)) {
          {
            uint32_t s[CW];
            tmem_ldn<CW>(tmem + st * NR + hc + lane_off, s);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < CW; ++c)
              d[c] = plain || ((allow >> c) & 1u) ? __uint_as_float(s[c]) * p.scale_log2 : -INFINITY;
          }
          ta_reduce<true, CW>(d, &sh->red[quarter][hc], lane);
          soft_sync();
          if (threadIdx.x < NR) {
            const int c = threadIdx.x;
            const float mo = sh->m[c];
            const float tm = fmaxf(fmaxf(sh->red[0][c], sh->red[1][c]), fmaxf(sh->red[2][c], sh->red[3][c]));
            const float mn = tm > mo + TA_GROW || mo == -INFINITY ? tm : mo;
            sh->f[c] = mn == mo || mo == -INFINITY ? 1.f : ex2f(mo - mn);
            sh->m[c] = mn;
            sh->mneg[c] = -mn;
          }
          soft_sync();
          exponents();
#pragma unroll
          for (int c = 0; c < CW; ++c) l[c] *= sh->f[hc + c];
          if (i > 0) {  // raise the output's columns too, once the products before are in it
            const uint32_t lg = g - 1;
            mbar_wait(&sh->pv_done[two ? lg & 1 : 0], (two ? lg >> 1 : lg) & 1, wc);
            tc_fence_after();
            for (int m = 0; m < p.dv_tiles; ++m) {
#pragma unroll
              for (int c = 0; c < CW; c += 8) {
                uint32_t o[8];
                tmem_ld8(tmem + o_col + m * NR + hc + c + lane_off, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * sh->f[hc + c + k]);
                tmem_st8(tmem + o_col + m * NR + hc + c + lane_off, o);
              }
            }
            tmem_wait_st();
          }
        }
        uint8_t* pr = ps + st * 16384 + key * 128;
#pragma unroll
        for (int c = 0; c < CW; c += 8) {
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float e0 = ex2f(d[c + 2 * k]), e1 = ex2f(d[c + 2 * k + 1]);
            l[c + 2 * k] += e0;
            l[c + 2 * k + 1] += e1;
            o[k] = cvt_bf16x2(e0, e1);
          }
          *reinterpret_cast<uint4*>(pr + ((((hc + c) >> 3) ^ (key & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[st]);
      }
      // the row tile's part is complete
      {
        const uint32_t lg = g - 1;
        ta_reduce<false, CW>(l, &sh->red[quarter][hc], lane);
        soft_sync();
        // a part of a longer row tile: the head of it, or a later piece
        const int slot = 2 * (int)blockIdx.x + (w.t == 0 ? 1 : 0);
        if (threadIdx.x < NR) {
          const int c = threadIdx.x;
          const float m = sh->m[c];
          float sum = sh->red[0][c] + sh->red[1][c] + sh->red[2][c] + sh->red[3][c];
          if (whole) {
            if (p.sink && m != -INFINITY)  // (without a key the output is 0 either way)
              sum += ex2f(__ldg(p.sink + (r0 + c) % p.H) * 1.4426950408889634f - m);
            sh->f[c] = sum == 0.f ? 0.f : 1.f / sum;
          } else {
            *reinterpret_cast<float2*>(p.part_ml + ((int64_t)slot * NR + c) * 2) = make_float2(m, sum);
          }
          sh->m[c] = -INFINITY;
          sh->mneg[c] = INFINITY;
        }
        if (!whole && threadIdx.x == 0 && w.t == 0) {
          int32_t* ow = p.owner + (int64_t)blockIdx.x * 4;
          ow[0] = w.b;
          ow[1] = w.rt;
          // CTAs from this one to the one that holds the last unit
          ow[2] = 1 + (int)((w.nt - n + sh->per - 1) / sh->per);
        }
        soft_sync();
        mbar_wait(&sh->pv_done[two ? lg & 1 : 0], (two ? lg >> 1 : lg) & 1, wc);
        tc_fence_after();
        for (int m = 0; m < p.dv_tiles; ++m) {
          uint32_t o[CW];
          tmem_ldn<CW>(tmem + o_col + m * NR + hc + lane_off, o);
          tmem_wait_ld();
          const int dim = m * 128 + quarter * 32 + lane;
          if (dim < p.dv) {
            if (whole) {
              uint16_t* op = p.out + ((int64_t)w.b * p.rows + r0 + hc) * p.dv + dim;
#pragma unroll
              for (int c = 0; c < CW; ++c)
                if (hc + c < nrows)
                  op[(int64_t)c * p.dv] =
                      __bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float(o[c]) * sh->f[hc + c]));
            } else {
              float* op = p.part_o + ((int64_t)slot * NR + hc) * p.dv + dim;
#pragma unroll
              for (int c = 0; c < CW; ++c)
                if (hc + c < nrows) op[(int64_t)c * p.dv] = __uint_as_float(o[c]);
            }
          }
        }
        tc_fence_before();
        soft_sync();  // f is read by all before the next item's raises
      }
      w.next_item(p, n);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) tmem_dealloc<1>(tmem, p.tmem_cols);
}

// Adds up the parts of row tiles that span CTAs, in order: the tile whose head CTA x holds
// has its parts in slots 2 x + 1, 2 (x + 1), 2 (x + 2), ...  blockIdx.y: TA_JOIN_ROWS rows.
constexpr int TA_JOIN_THREADS = 128;
constexpr int TA_JOIN_ROWS = 1;

template <int NR>
__global__ void __launch_bounds__(TA_JOIN_THREADS) tree_attn_join_kernel(const TreeAttnParams p) {
  const int32_t* ow = p.owner + (int64_t)blockIdx.x * 4;
  const int parts = ow[2];
  const int c = blockIdx.y;
  const int64_t row = (int64_t)ow[1] * NR + c;
  if (parts == 0 || row >= p.rows) return;
  auto slot = [&](int i) { return i == 0 ? 2 * (int64_t)blockIdx.x + 1 : 2 * ((int64_t)blockIdx.x + i); };
  float m = -INFINITY;
  for (int i = 0; i < parts; ++i) m = fmaxf(m, p.part_ml[(slot(i) * NR + c) * 2]);
  const float mu = m == -INFINITY ? 0.f : m;
  float sum = p.sink && m != -INFINITY ? ex2f(__ldg(p.sink + row % p.H) * 1.4426950408889634f - m) : 0.f;
  for (int i = 0; i < parts; ++i) {
    const float2 v = *reinterpret_cast<const float2*>(p.part_ml + (slot(i) * NR + c) * 2);
    sum += v.y * ex2f(v.x - mu);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  for (int d = threadIdx.x * 4; d < p.dv; d += TA_JOIN_THREADS * 4) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < parts; ++i) {
      const float f = ex2f(p.part_ml[(slot(i) * NR + c) * 2] - mu);
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (slot(i) * NR + c) * p.dv + d);
      o.x += v.x * f;
      o.y += v.y * f;
      o.z += v.z * f;
      o.w += v.w * f;
    }
    *reinterpret_cast<uint2*>(p.out + ((int64_t)ow[0] * p.rows + row) * p.dv + d) =
        make_uint2(cvt_bf16x2(o.x * inv, o.y * inv), cvt_bf16x2(o.z * inv, o.w * inv));
  }
}

}  // namespace ks
