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
// Warps: 4 softmax warps (thread = key = TMEM lane), 8 loader warps, one MMA / query-TMA
// warp and one address warp: 14, so that four share a scheduler and a thread may hold 128
// registers (with 18 warps, 96: the loaders spilled, and a spill waits for its load).  The
// address warp walks the page table ahead of the loads (slot, scale factor and state of
// each key, in shared memory).  A loader warp owns 16 keys: its codes of the next tile wait
// in registers, so the memory latency passes behind a whole tile's work, and a pair of
// 64-column chunks is refilled as soon as the last product that reads it is done.  No load
// is in flight while a tile is converted: the proxy fence that hands a chunk to the tensor
// cores waits for all of its thread's loads.  The bf16 tail goes from global to shared
// memory directly (cp.async).
//
// Softmax: p = 2^(s - m) with a reference m that need not be the running maximum: p, its
// sum and the output are floating point, so only overflow limits how far s may pass m.
// A tile is worked on in one pass with the m it finds; if a score passed it by more than
// TA_GROW (base 2), m is raised, and sum and output scaled, after the tile's product; only
// a score that passes it by TA_MOST raises it before, and the tile is done again.  A row
// tile's first tile finds its maxima first.  Sums are kept per thread in fp32 and reduced
// once per row tile.
#pragma once
#include "latent_cache.cuh"
#include "sparse_attn.cuh"
#include "sparse_attn_small.cuh"

namespace ks {

constexpr int TA_SOFT = 128;                 // softmax threads (warps 0-3)
constexpr int TA_LOAD = 256;                 // loader threads (warps 4-11)
constexpr int TA_W_LOAD = 4, TA_W_MMA = 12, TA_W_ADDR = 13;
constexpr int TA_THREADS = TA_SOFT + TA_LOAD + 64;
constexpr int TA_MAX_CHUNKS = 9;             // 64-column chunks of a row
constexpr int TA_MAX_CTAS = 148;             // SMs of a B200: bounds the workspace
constexpr int TA_MAX_ROWS = 64;
constexpr int TA_HDR = 8192;
constexpr int TA_AHEAD = 4;                  // tiles whose addresses are held
constexpr float TA_GROW = 8.f, TA_MOST = 24.f;  // how far a score may pass m (base 2)

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
  uint64_t full[2][5];              // a pair of chunks (4: the tail) has been written
  uint64_t vfree[2][4];             // the PV products of a 128-dim tile are done
  uint64_t s_full[2];               // scores of a tile are in TMEM (and its K reads done)
  uint64_t p_full[2];               // P of a tile is in shared memory
  uint64_t pv_done[2];              // all PV products of a tile are done
  uint64_t a_full[TA_AHEAD], a_free[TA_AHEAD];  // a tile's addresses are in place / used
  uint64_t q_full, drain;
  uint32_t tmem_base;
  int abort;
  int64_t total, per;
  int32_t b0, rt0, t0;              // where this CTA's stretch starts
  alignas(16) float m[TA_MAX_ROWS];     // reference of each row (base 2)
  alignas(16) float mneg[TA_MAX_ROWS];  // its negative (read as float4)
  float f[TA_MAX_ROWS];             // factor of a raise; at the end 1 / sum
  float red[4][TA_MAX_ROWS];
  int32_t slot[TA_AHEAD][128];      // row of the page pool, -1: nothing to load
  uint32_t mul[TA_AHEAD][128];      // 2^120 * scale as two bf16 factors (low half, high half)
  // key: 0 fine, 1 absent, 2 marked (scale NaN); read by the softmax, which is up to two
  // tiles behind the loaders that free the addresses
  uint8_t flag[2 * TA_AHEAD][128];
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

// Two e4m3 codes (bytes 0, 1 of w with SEL = 0x9180, bytes 2, 3 with 0xB3A2) as bf16,
// times the powers of two in `mul`.  A code s eeee mmm is placed in its 16-bit lane sign
// extended, moved up by 4 and masked: s 0000 eeee mmm 0000, its value times 2^-120 (bf16's
// bias is 120 more than e4m3's; subnormals included).  The one exact product with 2^120 *
// scale is the value.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t ta_expand(uint32_t w, uint32_t mul) {
  uint32_t t;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(t) : "r"(w), "n"(SEL));
  return mul_bf16x2((t * 16u) & 0x87F087F0u, mul);
}

// ldcg_or_zero at a constant offset: one address for a whole row.
template <int OFF>
__device__ __forceinline__ uint4 ta_ld(const void* base, bool pred) {
  uint4 v;
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %5, 0;"
      " mov.b32 %0, 0; mov.b32 %1, 0; mov.b32 %2, 0; mov.b32 %3, 0;"
      " @p ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4 + %6]; }"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(base), "r"((int)pred), "n"(OFF));
  return v;
}
// Chunks C .. NQ - 1 of two rows.
template <int C, int NQ>
__device__ __forceinline__ void ta_load_rows(uint4 (&r)[NQ][2], const uint8_t* c0, const uint8_t* c1, bool ok0,
                                             bool ok1, int nq) {
  if constexpr (C < NQ) {
    r[C][0] = ta_ld<C * 64>(c0, ok0 && C < nq);
    r[C][1] = ta_ld<C * 64>(c1, ok1 && C < nq);
    ta_load_rows<C + 1, NQ>(r, c0, c1, ok0, ok1, nq);
  }
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
  constexpr int CB = NR < 32 ? NR : 32;  // rows that a softmax thread works on at a time
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
      for (int c = 0; c < 5; ++c) mbar_init(&sh->full[s][c], TA_LOAD / 32);
      for (int m = 0; m < 4; ++m) mbar_init(&sh->vfree[s][m], 1);
      mbar_init(&sh->s_full[s], 1);
      mbar_init(&sh->p_full[s], TA_SOFT / 32);
      mbar_init(&sh->pv_done[s], 1);
    }
    for (int s = 0; s < TA_AHEAD; ++s) {
      mbar_init(&sh->a_full[s], 1);
      mbar_init(&sh->a_free[s], TA_LOAD / 32);
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
  if (warp == TA_W_MMA) {
    tmem_alloc<1>(&sh->tmem_base, p.tmem_cols);
    tmem_relinquish<1>();
    if (lane == 0) tma_prefetch_desc(&qm);
  }
  if (warp == TA_W_ADDR) {  // the call's units, and where this CTA's stretch starts
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

  if (warp >= TA_W_LOAD && warp < TA_W_MMA) {
    // ================================================================ loaders
    // lane: 16 codes (part) of keys key0, key0 + 8 in each chunk; a warp's load covers
    // 64-byte stretches of 8 rows
    const int lw = warp - TA_W_LOAD, part = lane & 3, key0 = lw * 16 + (lane >> 2);
    const uint32_t sw = (uint32_t)(key0 & 7), units = (uint32_t)max(w.left, 0);
    const uint32_t at0 = (uint32_t)key0 * 128 + (((uint32_t)(part * 2) ^ sw) << 4);
    const uint32_t at1 = (uint32_t)key0 * 128 + (((uint32_t)(part * 2 + 1) ^ sw) << 4);
    uint4 r[NQ][2];
    auto load = [&](uint32_t g) {
      const int s0 = sh->slot[g % TA_AHEAD][key0], s1 = sh->slot[g % TA_AHEAD][key0 + 8];
      const uint8_t* c0 = p.kv8 + (int64_t)s0 * p.dq + part * 16;
      const uint8_t* c1 = p.kv8 + (int64_t)s1 * p.dq + part * 16;
      ta_load_rows<0, NQ>(r, c0, c1, s0 >= 0, s1 >= 0, p.nq);
    };
    bool ok = units > 0;
    if (ok) {
      ok = mbar_wait_inl(&sh->a_full[0], 0, wc);
      load(0);
    }
    // The tail is early where only the scores read it; it waits for the second product
    // where that reads it too, or P takes its place (p_alias).
    const bool tail_pv = p.nq < 2 * p.dv_tiles, tail_early = p.dr > 0 && !tail_pv && !p.p_alias;
    for (uint32_t g = 0; g < units && ok; ++g) {
      const int st = two ? (int)(g & 1) : 0, ad = (int)(g % TA_AHEAD);
      const uint32_t use = two ? g >> 1 : g, last = (use - 1) & 1;
      uint8_t* tile = ks_ + (size_t)st * p.nka * 16384;
      const uint32_t ma = sh->mul[ad][key0], mb = sh->mul[ad][key0 + 8];
      const uint32_t m1[2] = {(ma & 0xFFFFu) * 0x10001u, (mb & 0xFFFFu) * 0x10001u};
      const bool big = __any_sync(0xFFFFFFFFu, (ma >> 16) != 0x3F80u || (mb >> 16) != 0x3F80u);
      auto tail = [&] {
        if (use > 0)
          ok = mbar_wait_inl(tail_pv     ? &sh->vfree[st][p.nq >> 1]
                             : p.p_alias ? &sh->pv_done[st]
                                         : &sh->s_full[st], last, wc) && ok;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = lw * 16 + j * 4 + (lane >> 3), piece = lane & 7;
          const int s = sh->slot[ad][key];
          cp_async16(tile + p.nq * 16384 + key * 128 + ((piece ^ (key & 7)) << 4),
                     p.tail + (int64_t)max(s, 0) * p.dr + piece * 8, s >= 0 ? 16u : 0u);
        }
      };
      if (tail_early) tail();
#pragma unroll
      for (int m = 0; m < NQ / 2; ++m) {
        if (2 * m < p.nq) {
          const bool end = 2 * m + 2 >= p.nq;
          if (use > 0)
            ok = mbar_wait_inl(m < p.dv_tiles ? &sh->vfree[st][m] : &sh->s_full[st], last, wc) && ok;
          if (end && p.dr > 0 && !tail_early) tail();
#pragma unroll
          for (int c = 2 * m; c < 2 * m + 2; ++c) {
            if (c >= p.nq) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint4 v = r[c][j];
              uint4 lo, hi;
              lo.x = ta_expand<0x9180>(v.x, m1[j]);
              lo.y = ta_expand<0xB3A2>(v.x, m1[j]);
              lo.z = ta_expand<0x9180>(v.y, m1[j]);
              lo.w = ta_expand<0xB3A2>(v.y, m1[j]);
              hi.x = ta_expand<0x9180>(v.z, m1[j]);
              hi.y = ta_expand<0xB3A2>(v.z, m1[j]);
              hi.z = ta_expand<0x9180>(v.w, m1[j]);
              hi.w = ta_expand<0xB3A2>(v.w, m1[j]);
              if (big) {  // a scale beyond 2^7
                const uint32_t m2 = ((j ? mb : ma) >> 16) * 0x10001u;
                lo.x = mul_bf16x2(lo.x, m2);
                lo.y = mul_bf16x2(lo.y, m2);
                lo.z = mul_bf16x2(lo.z, m2);
                lo.w = mul_bf16x2(lo.w, m2);
                hi.x = mul_bf16x2(hi.x, m2);
                hi.y = mul_bf16x2(hi.y, m2);
                hi.z = mul_bf16x2(hi.z, m2);
                hi.w = mul_bf16x2(hi.w, m2);
              }
              *reinterpret_cast<uint4*>(tile + c * 16384 + j * 1024 + at0) = lo;
              *reinterpret_cast<uint4*>(tile + c * 16384 + j * 1024 + at1) = hi;
            }
          }
          if (p.dr > 0 && (tail_early ? m == 0 : end)) cp_async_wait_all();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&sh->full[st][m]);
            if (p.dr > 0 && (tail_early ? m == 0 : end)) mbar_arrive(&sh->full[st][4]);
            if (end) mbar_arrive(&sh->a_free[ad]);
          }
        }
      }
      if (g + 1 < units) {
        ok = mbar_wait_inl(&sh->a_full[(g + 1) % TA_AHEAD], ((g + 1) / TA_AHEAD) & 1, wc) && ok;
        load(g + 1);
      }
    }
  } else if (warp == TA_W_ADDR) {
    // ================================================================ addresses
    const uint32_t units = (uint32_t)max(w.left, 0);
    bool ok = true;
    for (uint32_t g = 0; g < units && ok; ++g, w.next_unit(p)) {
      int s[4];
      uint32_t sb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = ta_slot(p, w, i * 32 + lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sb[i] = s[i] >= 0 ? __float_as_uint(__ldg(p.scale + s[i])) : 0u;
        if (s[i] >= 0 && p.dr > 0)  // the tail is fetched when its place is free: have it near
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p.tail + (int64_t)s[i] * p.dr));
      }
      const int ad = (int)(g % TA_AHEAD);
      if (g >= TA_AHEAD) ok = mbar_wait_inl(&sh->a_free[ad], (g / TA_AHEAD - 1) & 1, wc);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = i * 32 + lane;
        const bool bad = (sb[i] & 0x7F800000u) == 0x7F800000u;
        // 2^120 * scale, in two factors where that is beyond bf16 (0 for a scale of 0)
        const int e = (int)((sb[i] >> 23) & 255) + 120;
        const uint32_t m1 = (sb[i] & 0x7F800000u) && !bad ? (uint32_t)min(e, 254) << 7 : 0u;
        const uint32_t m2 = bad ? 127u : (uint32_t)(max(e, 254) - 254 + 127);
        sh->flag[g % (2 * TA_AHEAD)][key] = s[i] < 0 ? 1 : bad ? 2 : 0;
        sh->slot[ad][key] = bad ? -1 : s[i];
        sh->mul[ad][key] = m1 | (m2 << 23);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->a_full[ad]);
    }
  } else if (warp == TA_W_MMA) {
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
      // descriptors: only the start address (low word, 16-byte units) changes
      const uint64_t k_desc = sdesc_sw128(smem_u32(ks_), 16, 1024), q_desc = sdesc_sw128(smem_u32(qs), 16, 1024);
      const uint64_t v_desc = sdesc_sw128(smem_u32(ks_), 16384, 1024), p_desc = sdesc_sw128(smem_u32(ps), 16, 1024);
      const uint32_t stage16 = (uint32_t)p.nka * 1024;
      auto qk = [&](uint32_t g) {
        const int st = two ? (int)(g & 1) : 0;
        const uint32_t use = two ? g >> 1 : g;
        for (int c = 0; c < p.nkb; ++c) {
          if (c == p.nq || !(c & 1)) {
            ok = mbar_wait_inl(&sh->full[st][c == p.nq ? 4 : c >> 1], use & 1, wc);
            if (!ok) return;
            tc_fence_after();
          }
          const uint64_t ad = k_desc + st * stage16 + c * 1024, bd = q_desc + c * (NR * 8);
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
        const uint64_t bd = p_desc + st * 1024;
        for (int m = 0; m < p.dv_tiles; ++m) {
          const uint64_t ad = v_desc + st * stage16 + m * 2048;
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
    const int key = warp * 32 + lane;
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    uint32_t g = 0;
    while (w.left > 0) {
      const int n = w.here();
      const int r0 = w.rt * NR;                      // first row of the tile in the sequence
      const int nrows = min(NR, p.rows - r0);
      const bool whole = w.t == 0 && n == w.nt;      // no other CTA has a part
      float l[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) l[i] = 0.f;
      for (int i = 0; i < n; ++i, ++g) {
        const int st = two ? (int)(g & 1) : 0;
        const uint32_t use = two ? g >> 1 : g;
        const int tile = w.t + i;
        // which rows see this key: all, or a bit per row
        uint64_t allow = ~0ull;
        const int pos = tile * 128 + key, j = pos - w.len;
        if (j >= 0) {  // a drafted row, or past them (absent)
          allow = 0;
          if (j < p.T) {
            int t = r0 / p.H, h = r0 - t * p.H;
            const uint8_t* mk = p.mask + ((int64_t)w.b * p.T) * p.T + j;
            uint64_t bit = 0;
            bool fresh = true;
#pragma unroll 1
            for (int c = 0; c < NR; ++c) {
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
        mbar_wait_inl(&sh->full[st][0], use & 1, wc);  // the key's flag
        const int flag = sh->flag[g % (2 * TA_AHEAD)][key];
        if (flag == 1) allow = 0;
        mbar_wait_inl(&sh->s_full[st], use & 1, wc);
        tc_fence_after();
        constexpr uint64_t ALL = NR == 64 ? ~0ull : (1ull << NR) - 1;
        const bool plain = __all_sync(0xFFFFFFFFu, (allow & ALL) == ALL && flag == 0);
        // rows c0 .. c0 + CB - 1: scaled scores minus their references (raw: themselves)
        auto exponents = [&](int c0, float (&d)[CB], bool raw) {
          tmem_ldn<CB>(tmem + st * NR + c0 + lane_off, reinterpret_cast<uint32_t*>(d));
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < CB; c += 4) {
            const float4 mn = raw ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(&sh->mneg[c0 + c]);
            d[c] = fmaf(d[c], p.scale_log2, mn.x);
            d[c + 1] = fmaf(d[c + 1], p.scale_log2, mn.y);
            d[c + 2] = fmaf(d[c + 2], p.scale_log2, mn.z);
            d[c + 3] = fmaf(d[c + 3], p.scale_log2, mn.w);
          }
          if (!plain) {
            const uint32_t al = (uint32_t)(allow >> c0);
#pragma unroll
            for (int c = 0; c < CB; ++c)
              d[c] = !((al >> c) & 1u) ? -INFINITY : flag == 2 ? __uint_as_float(0x7FC00000u) : d[c];
          }
        };
        uint8_t* pr = ps + st * 16384 + key * 128;
        // P of this key, its sums where `add`; returns the largest exponent
        auto weights = [&](auto add) {
          float most = -INFINITY;
#pragma unroll
          for (int c0 = 0; c0 < NR; c0 += CB) {
            float d[CB];
            exponents(c0, d, false);
#pragma unroll
            for (int c = 0; c < CB; c += 8) {
              uint32_t o[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                most = fmaxf(most, fmaxf(d[c + 2 * k], d[c + 2 * k + 1]));
                const float e0 = ex2f(d[c + 2 * k]), e1 = ex2f(d[c + 2 * k + 1]);
                add(c0 + c + 2 * k, e0);
                add(c0 + c + 2 * k + 1, e1);
                o[k] = cvt_bf16x2(e0, e1);
              }
              *reinterpret_cast<uint4*>(pr + ((((c0 + c) >> 3) ^ (key & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
          return most;
        };
        // The tile's maxima, and references raised to them where they pass by `limit`.
        auto raise = [&](float limit) {
#pragma unroll
          for (int c0 = 0; c0 < NR; c0 += CB) {
            float d[CB];
            exponents(c0, d, true);
            ta_reduce<true, CB>(d, &sh->red[warp][c0], lane);
          }
          soft_sync();
          if (threadIdx.x < NR) {
            const int c = threadIdx.x;
            const float mo = sh->m[c];
            const float tm = fmaxf(fmaxf(sh->red[0][c], sh->red[1][c]), fmaxf(sh->red[2][c], sh->red[3][c]));
            const float mn = tm > mo + limit || mo == -INFINITY ? tm : mo;
            sh->f[c] = mn == mo ? 1.f : ex2f(mo - mn);
            sh->m[c] = mn;
            sh->mneg[c] = -mn;
          }
          soft_sync();
        };
        // The output's columns by the factors of a raise, once every product up to tile x is in them.
        auto scale_output = [&](uint32_t x) {
          mbar_wait_inl(&sh->pv_done[two ? x & 1 : 0], (two ? x >> 1 : x) & 1, wc);
          tc_fence_after();
#pragma unroll 1
          for (int m = 0; m < p.dv_tiles; ++m) {
#pragma unroll 1
            for (int c = 0; c < NR; c += 8) {
              uint32_t o[8];
              tmem_ld8(tmem + o_col + m * NR + c + lane_off, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * sh->f[c + k]);
              tmem_st8(tmem + o_col + m * NR + c + lane_off, o);
            }
          }
          tmem_wait_st();
        };
        auto publish = [&] {
          fence_proxy_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->p_full[st]);
        };
        auto sums = [&](int c, float e) { l[c] += e; };
        if (i == 0) {  // no reference yet
          raise(0.f);
          weights(sums);
          publish();
        } else {
          const float most = weights(sums);
          if (!soft_any(most > TA_GROW)) {
            publish();
          } else if (!soft_any(most > TA_MOST)) {
            raise(TA_GROW);  // (reads the scores, so before the next ones may come)
            publish();
#pragma unroll
            for (int c = 0; c < NR; ++c) l[c] *= sh->f[c];
            scale_output(g);
          } else {
            // Take the weights out of the sums again (to 2^-24 of the weight that passes m,
            // which becomes 1 at most; an infinite one leaves nothing worth keeping), raise m
            // and repeat the tile.
            auto undo = [&](int c, float e) { l[c] = l[c] == INFINITY ? 0.f : l[c] - e; };
            weights(undo);
            raise(TA_GROW);
#pragma unroll
            for (int c = 0; c < NR; ++c) l[c] *= sh->f[c];
            weights(sums);
            scale_output(g - 1);
            publish();
          }
        }
      }
      // the row tile's part is complete
      {
        const uint32_t lg = g - 1;
        ta_reduce<false, NR>(l, sh->red[warp], lane);
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
        mbar_wait_inl(&sh->pv_done[two ? lg & 1 : 0], (two ? lg >> 1 : lg) & 1, wc);
        tc_fence_after();
        for (int m = 0; m < p.dv_tiles; ++m) {
          const int dim = m * 128 + key;
#pragma unroll
          for (int c0 = 0; c0 < NR; c0 += CB) {
            uint32_t o[CB];
            tmem_ldn<CB>(tmem + o_col + m * NR + c0 + lane_off, o);
            tmem_wait_ld();
            if (dim < p.dv) {
              if (whole) {
                uint16_t* op = p.out + ((int64_t)w.b * p.rows + r0 + c0) * p.dv + dim;
#pragma unroll
                for (int c = 0; c < CB; ++c)
                  if (c0 + c < nrows)
                    op[(int64_t)c * p.dv] =
                        __bfloat16_as_ushort(__float2bfloat16_rn(__uint_as_float(o[c]) * sh->f[c0 + c]));
              } else {
                float* op = p.part_o + ((int64_t)slot * NR + c0) * p.dv + dim;
#pragma unroll
                for (int c = 0; c < CB; ++c)
                  if (c0 + c < nrows) op[(int64_t)c * p.dv] = __uint_as_float(o[c]);
              }
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
  if (warp == TA_W_MMA) tmem_dealloc<1>(tmem, p.tmem_cols);
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
