// Attention of drafted tokens over the quantised latent cache.
//
//   s[k] = scale * q . c_k,  o = sum_k exp(s_k - m) v_k / (sum_k exp(s_k - m) + exp(sink - m))
//
// with c_k the cached row of position k (latent_cache.cuh), v_k its first dv columns.
// A drafted token of sequence b sees the lens[b] cached positions and, among the T
// drafted rows that follow them in the cache, those its row of the mask allows (without
// a mask: itself and the ones before it).
//
// The T * H query rows of a sequence share its cached rows, so the products run with keys
// as the MMA's M dimension:
//   S^T[128 keys, rows] = K . Q^T         O^T[dims, rows] += V^T . P^T
// and on the cache's own e4m3 codes (tcgen05 kind::f8f6f4): a code tile is loaded once, by
// TMA where the pages allow, and read K-major by the first product and MN-major (dims
// contiguous) by the second.  Nothing is expanded.  What meets the codes is split into
// 8-bit numbers, several columns per row:
//   * a query element is 8 significant bits of bf16: q 2^-e = hi + lo / 16 exactly, hi and
//     lo with 4 bits each (e: the exponent of the row's code columns, hi below 256; elements
//     under 2^-14 of their largest are rounded to 2^-21 of it).  S = S_hi + S_lo / 16.  The
//     rotary columns are scaled alike; where they are more than 2^TA_ROTARY times as large, e
//     goes by them (an exponent of their own made ragged trees 2 % slower).
//   * a weight is taken to fp16 and split into three e5m2 numbers of 3 bits and a sign, the
//     high bytes of P, P - P0 and P - P0 - P1 as fp16, each rounded to nearest, which
//     together are the 11 bits exactly; each product goes to columns of its own and the
//     three are added at the end.  Off by at most 2^-11 of the weight (fp16; a bf16 weight:
//     2^-8), or 2^-26 of the row's largest weight times scale where that is more.  (Parts
//     cut off instead of rounded: 2^-9 more, at the same time.)
// A key's scale multiplies its scores (thread = key) and its weight.  A row has two
// references: m of its scores, for the weights and their sum, and m + ceil(mr) of its scores
// + log2 of scale, for P = 2^(TA_TOP + s - m - ceil(mr)) * scale.  (m is the largest score
// itself, so that the weight that counts most is a power of two and not rounded: with m
// rounded up, results were up to 1.6 times as far from those of exact weights.)  So P keeps
// within e5m2's range by what the row itself weighs: a key that it does not see, or that has
// no weight, takes no precision from the others, however large its values.  (One reference
// of the scales for the CTA, the largest scale present, lost rows beside one 2^56 larger.)
// Products stay finite where the result is: scores are added up 2^-TA_DOWN as large, with the
// softmax scale's power of two put back last (exactly, so that the largest score's distance
// to its reference is right at any size), and the weights of the bf16 columns 2^-TA_VT.
// The rotary columns are bf16 and have a bf16 product of their own; where v reaches into
// them (dv > dq), so do they.
//
// Why split: with bf16 operands every tile's codes are expanded in shared memory, 147 KB
// stored and read back per tile, next to MMAs that read their operands from the same
// memory ((4 KB + N * 32 B) / 128 B cycles for M128 N16..128: 40 at N = 16, 49 at 64, 65
// at 128).  That form took 10.5 K cycles per 64-row tile; a code tile is half the bytes,
// K = 32 per instruction halves the operand reads, and two tiles fit, so loads run ahead.
//
// Work: a unit is one 128-key tile of one (sequence, NR-row tile), NR = 16 or 32 (three
// output columns per row fill TMEM at 32).  Setting up a row tile's queries and storing its
// output count as TA_SETUP units more.  The call's units in order are cut into equal
// stretches, one per CTA, whatever the lengths (which only the device knows), so a long
// context is split over the SMs and ragged batches balance (16 trees of 13 tokens, 64
// heads, up to 6001 keys: 270 us with TA_SETUP = 0, when CTAs with many short sequences
// ran twice as long as the others; 179, 168 and 170 us with 3, 4 and 5).  A row tile that
// spans CTAs leaves (references, sum, unnormalised output) per part in the workspace;
// tree_attn_join_kernel adds them up in order (no atomics).  Short tables take a CTA per
// row tile and need no join (the host code has the rule and its figures).
//
// Warps: a softmax warp for each lane quarter and 8 rows (thread = key = TMEM lane: 16 warps
// at NR = 32; 8 warps of 16 rows took 1 % less on large trees and 3 % more on ragged ones),
// 5 loader warps, a warp that issues the first product and one that issues the
// second (each waits for its own inputs; one thread for both made each wait for the
// other's), one address warp that walks the page table ahead of
// the loads.  A tile whose keys are all present and unmarked comes by TMA in boxes of r
// rows (r: the power of two that divides page and 128, at least 8); others (the last of a
// sequence, odd pages) by cp.async with absent and marked rows zeroed, so that no garbage
// meets a zero weight.  Codes lie in a ring of chunks (128 keys of 128 columns, 16 KB), nine
// of them at 576 columns: a chunk goes back to the loads when its dim tile's product is done.
//
// Softmax: references are raised only when some weight passes 2^TA_RISE or some P 2^(TA_TOP
// + TA_GROW), together with sum and output (one vote per tile).  A raise costs more than a
// tile, so the limit is what e5m2's range allows, and all rows that have grown are raised at
// once: large trees (below) take 751 us so, 778 where only rows past the limit are raised,
// 808 with TA_GROW = 5 too (one run); all raises together are 1 to 5 % of a call.  Sums are
// kept per thread in fp32 and reduced once per row tile.
//
// Measured (device time, one B200): 8 trees of 32 tokens, 128 heads, 8192 keys 750 us (585
// GFLOP of scores and outputs: 780 TFLOP/s); 16 trees of 13 tokens, 64 heads, up to 6001 keys
// 173 us; one token of 128 heads over 131069 keys 69.8 us; 48 sequences of up to 8000 keys, 16
// heads 36.9 us (128 MB: 3.5 TB/s).  Bound: at 32 rows a tile takes about 2.8 K cycles, the
// MMAs 1.9 K of them (counters: tensor pipe 42 %, shared memory 61 %); the rest is the chain
// chunk given back -> load (1.3 K from L2) -> scores -> softmax (2.2 K) -> output, of which
// two tiles are in flight, because nine chunks and a row tile's queries fill shared memory
// and its outputs TMEM.  A row tile's beginning and end cost about 10 K cycles.  At 16 rows a
// tile's 82 KB are the larger part: 3.4 K cycles, the rate of HBM with all SMs at work.
#pragma once
#include "latent_cache.cuh"
#include "sparse_attn.cuh"
#include "sparse_attn_small.cuh"

namespace ks {

constexpr int TA_CW = 8;                     // rows of a softmax thread
constexpr int TA_LOADERS = 5;                // loader warps: a chunk each, the tail
template <int NR>
constexpr int TA_SOFT = NR / TA_CW * 128;    // softmax threads (the first ones)
template <int NR>
constexpr int TA_THREADS = TA_SOFT<NR> + (TA_LOADERS + 3) * 32;
constexpr int TA_MAX_CTAS = 148;             // SMs of a B200: bounds the workspace
constexpr int TA_MAX_ROWS = 32;
constexpr int TA_SLOTS = 12;                 // most code chunks in shared memory
constexpr uint32_t TA_CHUNK = 16384;         // 128 keys of 128 bytes
constexpr int TA_AHEAD = 4;                  // tiles whose addresses are held
constexpr int TA_HDR = 6144;
constexpr int TA_SETUP = 4;                  // units that a row tile costs beyond its tiles
constexpr int TA_SOLO = 512;                 // keys of a table up to which a CTA takes a row tile whole (see the host code)
constexpr int TA_LEVELS = 3;                 // e5m2 columns per weight
constexpr float TA_TOP = 10.f;               // P at the reference m + mr is 2^TA_TOP
constexpr float TA_GROW = 5.75f;             // how far it may grow past that (base 2): 2^(TA_TOP + TA_GROW) < 57344
constexpr float TA_RISE = 7.f;               // how far a score may pass m (base 2)
constexpr int TA_DOWN = 24;                  // scores are added up 2^24 too small: 256 * 448 * 512 * 2^(119 - 24) is finite
constexpr int TA_ROTARY = 9;                 // bits by which rotary elements may be larger: 64 * 2^(8 + 9 - 24) * 2^128 is finite
constexpr int TA_VT = 24;                    // bf16 weights are 2^24 too small: 2^(TA_RISE - 24) * 2^17 keys * 2^128 is finite
constexpr float TA_SPAN = 110.f;             // how far m + mr may lie below m: 2^(TA_TOP + TA_SPAN + TA_RISE) is finite

struct TreeAttnParams {
  const uint16_t* q;      // bf16 [B, T * H, dq + dr]
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
  int32_t nc;             // 128-column chunks of codes
  int32_t dt;             // 128-dim tiles of O^T from codes
  int32_t slots, tails;   // code chunks and tail chunks in shared memory
  int32_t s_bufs;
  int32_t box;            // rows of a TMA box, 0: no TMA
  int32_t solo;           // a CTA per row tile, nothing to join
  uint32_t k_off, t_off, q_off, p_off, pb_off;
  uint32_t tmem_cols;
  float scale_in, scale_up;  // product: softmax scale * log2 e * 2^TA_DOWN; scale_up is a power of two
  float* part_o;          // [2 * CTAs][NR][dv]
  float* part_ml;         // [2 * CTAs][NR][4]: m, sum, ceil(mr)
  int32_t* owner;         // [CTAs][4]: sequence, row tile, parts (0: none to join), CTA of the head
  int32_t by_item;        // owner is indexed by row tile of the call (there are few), else by CTA
  int* status;
  uint64_t budget_ns;
};

struct TaShared {
  uint64_t full[TA_SLOTS + 2];                  // a chunk is in place (the last two: the tail)
  uint64_t kfree[TA_SLOTS + 2];                 // it has been used
  uint64_t s_full[2], s_free[2];                // scores are in TMEM / in registers
  uint64_t p_full, pv_done;                     // weights are in shared memory / have been used
  uint64_t a_full[TA_AHEAD], a_free[TA_AHEAD];  // a tile's addresses are in place / used
  uint64_t sk_full[TA_AHEAD];                   // its scales are in place
  uint64_t q_full, drain[2];
  uint32_t tmem_base;
  int abort;
  uint32_t issued[TA_SLOTS + 2];                // loads of the chunk so far
  float tp_max;                                 // log2 of the largest tp
  int wide;                                     // some m is so large that m + mr would be rounded
  int64_t per;                                  // units of a stretch
  int32_t left0, b0, rt0, t0, len0;             // its first tile, see TaWalk
  alignas(16) float mneg[TA_MAX_ROWS];          // minus m, the reference of each row's scores (base 2)
  alignas(16) float mr[TA_MAX_ROWS];            // its largest score + log2 of the key's scale, from m on
  alignas(16) float qs[TA_MAX_ROWS];            // 2^e * scale_in of each row
  float red[4][TA_MAX_ROWS];
  union {  // a row's four maxima are read by the thread that then writes its factors
    alignas(16) float red_s[4][TA_MAX_ROWS];
    struct {
      float f[TA_MAX_ROWS];                     // factor of a raise of m; at the end 2^TA_VT / sum
      float fs[TA_MAX_ROWS];                    // of a raise of m + mr; at the end what a unit of P stands for / sum
      float tp[TA_MAX_ROWS];                    // 2^(TA_TOP - ceil(mr)): weight times scale to P, until the next raise
    };
  };
  int32_t whole[TA_AHEAD];                      // every key of the tile can come by TMA
  int32_t slot[TA_AHEAD][128];                  // row of the page pool, -1: zeros
  float sk[TA_AHEAD][128];                      // key's scale; -1: absent, NaN: marked
};
static_assert(sizeof(TaShared) <= TA_HDR, "TaShared exceeds its header");

// Keys of sequence b: its cached positions and drafted rows, within the page table.
__device__ __forceinline__ int ta_len(const TreeAttnParams& p, int b) { return max(0, __ldg(p.lens + b)); }
__device__ __forceinline__ int ta_keys(const TreeAttnParams& p, int len) {
  const int64_t cap = min(p.max_pages * p.page, (int64_t)0x7FFFFF00);
  return (int)min((int64_t)len + p.T, cap);
}
__device__ __forceinline__ int ta_tiles(const TreeAttnParams& p, int len) { return (ta_keys(p, len) + 127) >> 7; }

// A CTA's stretch of units, walked by every role on its own.  Tile t of a row tile lies
// TA_SETUP + t units after the row tile's beginning.
struct TaWalk {
  int left;       // units from here to the end of the stretch (0: no tile is left)
  int b, rt, t;   // this tile
  int len, nt;    // of sequence b
  __device__ __forceinline__ void start(const TreeAttnParams& p, const TaShared* sh) {
    left = sh->left0; b = sh->b0; rt = sh->rt0; t = sh->t0;
    len = sh->len0;
    nt = left > 0 ? ta_tiles(p, len) : 0;
  }
  // tiles of this row tile that are in the stretch, from here
  __device__ __forceinline__ int here() const { return min(nt - t, left); }
  __device__ __forceinline__ void next_item(const TreeAttnParams& p, int done) {
    left = max(left - done - TA_SETUP, 0);
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

// A ring position: slot and phase parity.
struct TaRing {
  int i = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next(int n) {
    if (++i == n) {
      i = 0;
      ph ^= 1;
    }
  }
};

// Slots of the page pool that hold this lane's four keys of a tile (lane, lane + 32, ..),
// -1 for none.  The four table entries are loaded at once.  (A pool has < 2^31 slots.)
__device__ __forceinline__ void ta_slots(const TreeAttnParams& p, const TaWalk& w, int lane, int (&s)[4]) {
  const int keys = ta_keys(p, w.len);
  const int32_t* table = p.table + (int64_t)w.b * p.max_pages;
  int pg[4], in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int pos = w.t * 128 + i * 32 + lane, pi = pos / p.page;  // within the table: keys is
    in[i] = pos - pi * p.page;
    pg[i] = ldg_s32_or(table + pi, pos < keys, -1);
    s[i] = pos < keys;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool ok = pg[i] >= 0 && pg[i] < p.n_pages;
    if (s[i] && !ok) report_bounds(p.status, w.b, (int)p.n_pages);
    s[i] = ok ? pg[i] * p.page + in[i] : -1;
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
__device__ __forceinline__ void tmem_ldn(uint32_t taddr, float* r) {
  if constexpr (N == 8) tmem_ld8(taddr, reinterpret_cast<uint32_t*>(r));
  else tmem_ld16(taddr, reinterpret_cast<uint32_t*>(r));
}
template <int N>
__device__ __forceinline__ void tmem_stn(uint32_t taddr, const float* r) {
  if constexpr (N == 8) tmem_st8(taddr, reinterpret_cast<const uint32_t*>(r));
  else tmem_st16(taddr, reinterpret_cast<const uint32_t*>(r));
}
// Any thread of the softmax warps (also a barrier among them).
template <int SOFT>
__device__ __forceinline__ bool soft_any(bool x) {
  uint32_t r;
  asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.or.pred q, 1, %2, p; selp.u32 %0, 1, 0, q; }"
               : "=r"(r)
               : "r"((uint32_t)x), "n"(SOFT)
               : "memory");
  return r != 0;
}

// 2^x of a whole x (0 below 2^-126; x at most 127; 1 for a NaN: what meets it is one).
__device__ __forceinline__ float ta_pow2(float x) {
  return __uint_as_float((uint32_t)(min(max(__float2int_rz(x), -127), 127) + 127) << 23);
}

// log2 of a power of two (-127: of less than 2^-126).
__device__ __forceinline__ float ta_log2(float x) { return (float)((int)(__float_as_uint(x) >> 23) - 127); }

// Sum over the warp's lanes of CW <= 16 values each into red[c], c < CW.
template <int CW>
__device__ __forceinline__ void ta_reduce(const float (&v)[CW], float* red, int lane) {
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = i < CW ? v[i % CW] : 0.f;
  const float r = reduce16_lanes<false>(w, lane);  // value lane >> 1
  if ((lane & 1) == 0 && (lane >> 1) < CW) red[lane >> 1] = r;
}
// Max over the warp's lanes of 8 values each into red[c], and of the values + a into red_s[c].
__device__ __forceinline__ void ta_maxima(const float (&v)[8], float a, float* red, float* red_s, int lane) {
  float w[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = v[i];
    w[i + 8] = v[i] + a;
  }
  const float r = reduce16_lanes<true>(w, lane);  // value lane >> 1
  if ((lane & 1) == 0) (lane < 16 ? red : red_s)[(lane >> 1) & 7] = r;
}

// MN-major operand of 64-byte rows (32 bf16) with the 64-byte swizzle: 16-byte unit u of
// row r lies at u ^ ((r >> 1) & 3); 8 rows are 512 bytes.
__device__ __forceinline__ uint64_t sdesc_sw64(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(16 >> 4) << 16 | (uint64_t)(512 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)4 << 61;
}

__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint16_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  return h;
}
// Two fp32 per instruction.
struct TaF2 {
  uint64_t v;
};
__device__ __forceinline__ TaF2 f2(float a, float b) {
  TaF2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_get(TaF2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ TaF2 fma2(TaF2 a, TaF2 b, TaF2 c) {
  TaF2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ TaF2 add2(TaF2 a, TaF2 b) {
  TaF2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ TaF2 mul2(TaF2 a, TaF2 b) {
  TaF2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint16_t e4m3x2_of_f16x2(uint32_t x) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(c) : "r"(x));
  return c;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <int NR, bool VT>
__global__ void __launch_bounds__(TA_THREADS<NR>, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap tm,
                     const TreeAttnParams p) {
  constexpr int CW = TA_CW, SOFT = TA_SOFT<NR>;
  constexpr int W_LOAD = SOFT / 32, W_QK = W_LOAD + TA_LOADERS, W_PV = W_QK + 1, W_ADDR = W_PV + 1;
  constexpr int NP = TA_LEVELS * NR;     // columns of P and of a dim tile of O^T
  extern __shared__ uint8_t ta_raw[];
  const uint32_t raw = smem_u32(ta_raw);
  uint8_t* smem = ta_raw + (((raw + 1023u) & ~1023u) - raw);
  TaShared* sh = reinterpret_cast<TaShared*>(smem);
  uint8_t* ks_ = smem + p.k_off;  // [slots][128 keys x 128 B] codes: a ring of chunks, nc a tile
  uint8_t* kt = smem + p.t_off;   // [tails][128 keys x 128 B] bf16 tail
  uint8_t* qs = smem + p.q_off;   // [nc][NR hi rows, NR lo rows x 128 B], [NR x 128 B] bf16 tail
  uint8_t* ps = smem + p.p_off;   // [128 keys x 128 B]: level, row (MN-major)
  uint8_t* pb = smem + p.pb_off;  // [128 keys x 64 B]: bf16 weights (MN-major), with vt
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  WaitCtx wc{&sh->abort, p.status, p.budget_ns};

  if (threadIdx.x == 0) {
    for (int s = 0; s < TA_SLOTS + 2; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->kfree[s], 1);
      sh->issued[s] = 0;
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sh->s_full[s], 1);
      mbar_init(&sh->s_free[s], SOFT / 32);
    }
    mbar_init(&sh->p_full, SOFT / 32);
    mbar_init(&sh->pv_done, 1);
    for (int s = 0; s < TA_AHEAD; ++s) {
      mbar_init(&sh->a_full[s], 1);
      mbar_init(&sh->sk_full[s], 1);
      mbar_init(&sh->a_free[s], TA_LOADERS + SOFT / 32);
    }
    mbar_init(&sh->q_full, SOFT / 32);
    mbar_init(&sh->drain[0], 1);
    mbar_init(&sh->drain[1], 1);
    sh->abort = 0;
    fence_barrier_init();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may be set up
    if (!p.by_item) p.owner[(int64_t)blockIdx.x * 4 + 2] = 0;  // no row tile's head here yet
  }
  if (threadIdx.x < TA_MAX_ROWS) {
    sh->mneg[threadIdx.x] = INFINITY;
  }
  if (warp == W_QK) {
    tmem_alloc<1>(&sh->tmem_base, p.tmem_cols);
    tmem_relinquish<1>();
    if (lane == 0 && p.box) {
      tma_prefetch_desc(&km);
      if (p.dr) tma_prefetch_desc(&tm);
    }
  }
  if (warp == W_ADDR && p.solo) {
    const int b = (int)blockIdx.x / p.row_tiles, rt = (int)blockIdx.x - b * p.row_tiles, len = ta_len(p, b);
    if (lane == 0) {
      sh->per = 0;
      sh->b0 = b;
      sh->rt0 = rt;
      sh->t0 = 0;
      sh->len0 = len;
      sh->left0 = ta_tiles(p, len);
      if (rt == 0 && (int64_t)len + p.T > p.max_pages * p.page)  // past the table
        report_bounds(p.status, b, (int)p.max_pages);
    }
  } else if (warp == W_ADDR) {  // the call's units, and where this CTA's stretch starts
    // 128 sequences at a time, their lengths loaded at once (and kept where that is all)
    int len[4];
    auto lengths = [&](int i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) len[k] = i + k * 32 + lane < p.B ? ta_len(p, i + k * 32 + lane) : -1;
    };
    int64_t total = 0;
    for (int i = 0; i < p.B; i += 128) {
      lengths(i);
      int64_t n = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (len[k] < 0) continue;
        n += ta_tiles(p, len[k]) + TA_SETUP;
        if (blockIdx.x == 0 && (int64_t)len[k] + p.T > p.max_pages * p.page)  // past the table
          report_bounds(p.status, i + k * 32 + lane, (int)p.max_pages);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
      total += n * p.row_tiles;
    }
    const int64_t per = total < (1ll << 31) ? (int64_t)(((uint32_t)total + gridDim.x - 1) / gridDim.x)
                                            : (total + gridDim.x - 1) / gridDim.x;
    const int64_t u0 = (int64_t)blockIdx.x * per;
    if (lane == 0) {
      sh->per = per;
      sh->left0 = 0;
    }
    __syncwarp();
    int64_t at = 0;
    bool found = u0 >= total;
    for (int i = 0; i < p.B && !found; i += 128) {
      if (p.B > 128) lengths(i);
#pragma unroll 1
      for (int k = 0; k < 4 && !found; ++k) {
        const int ln = k == 0 ? len[0] : k == 1 ? len[1] : k == 2 ? len[2] : len[3];
        const int64_t un = ln >= 0 ? ta_tiles(p, ln) + TA_SETUP : 0;  // of a row tile
        int64_t n = un * p.row_tiles;  // inclusive sums of the 32 sequences
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t v = __shfl_up_sync(0xFFFFFFFFu, n, o);
          if (lane >= o) n += v;
        }
        const uint32_t over = __ballot_sync(0xFFFFFFFFu, at + n > u0);
        if (over && lane == __ffs(over) - 1) {
          const int64_t in = u0 - (at + n - un * p.row_tiles);  // units into the sequence
          const int rt = in < (1ll << 31) ? (int)((uint32_t)in / (uint32_t)un) : (int)(in / un);
          const int into = (int)(in - rt * un);                 // and into the row tile
          sh->b0 = i + k * 32 + lane;
          sh->rt0 = rt;
          sh->t0 = max(into - TA_SETUP, 0);
          sh->len0 = ln;
          sh->left0 = (int)max(min(per, total - u0) - max(TA_SETUP - into, 0), (int64_t)0);
        }
        found = over != 0;
        at += __shfl_sync(0xFFFFFFFFu, n, 31);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const uint32_t o_col = (uint32_t)(p.s_bufs * 3 * NR);       // S: hi, lo, tail columns
  const uint32_t ot_col = o_col + (uint32_t)(p.dt * NP);      // O^T of the bf16 columns
  TaWalk w;
  w.start(p, sh);

  if (warp >= W_LOAD && warp < W_QK) {
    // ================================================================ loaders
    // Warp c loads chunk c, warp 4 the tail.
    const int lw = warp - W_LOAD, piece = lane & 7;
    const bool is_tail = lw == 4;
    const int x = is_tail ? 0 : lw * 128;
    const bool mine = is_tail ? p.dr > 0 : lw < p.nc;
    const int step = is_tail ? 1 : p.nc, ring = is_tail ? p.tails : p.slots;
    int at = is_tail ? 0 : lw;  // place in the ring, its phase
    uint32_t ph = 0;
    TaRing ad;
    bool ok = true;
    for (; w.left > 0 && ok; w.next_unit(p), ad.next(TA_AHEAD)) {
      ok = __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->a_full[ad.i], ad.ph, wc));
      if (!ok) break;
      const bool whole = p.box && sh->whole[ad.i];
      const int32_t* sl = sh->slot[ad.i];
      if (mine) {
        // The second product's dim tiles free their chunks one by one, chunks that only the
        // scores read go with theirs.
        const int bar = is_tail ? TA_SLOTS + at : at;
        uint64_t* full = &sh->full[bar];
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->kfree[bar], ph ^ 1, wc));
        if (!ok) break;
        uint8_t* dst = (is_tail ? kt : ks_) + (size_t)at * TA_CHUNK;
        if (lane == 0) ++sh->issued[bar];
        if (whole) {
          if (elect_one()) {
            mbar_expect_tx(full, TA_CHUNK);
            for (int r = 0; r < 128; r += p.box) tma_load_2d(is_tail ? &tm : &km, full, dst + r * 128, x, sl[r]);
          }
          __syncwarp();
        } else {
          // 8 lanes per row; rows that are not there and columns past dq become zeros
          for (int k = lane >> 3; k < 128; k += 4) {
            const int s = sl[k];
            const bool in = s >= 0 && (is_tail || x + piece * 16 < p.dq);
            const void* src = is_tail ? static_cast<const void*>(p.tail + (int64_t)s * p.dr + piece * 8)
                                      : p.kv8 + (int64_t)s * p.dq + x + piece * 16;
            cp_async16(dst + k * 128 + ((piece ^ (k & 7)) << 4), in ? src : p.kv8, in ? 16u : 0u);
          }
          cp_async_wait_all();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full);
        }
        at += step;  // (step <= ring)
        if (at >= ring) {
          at -= ring;
          ph ^= 1;
        }
      }
      if (lane == 0) mbar_arrive(&sh->a_free[ad.i]);
    }
  } else if (warp == W_ADDR) {
    // ================================================================ addresses
    TaRing ad;
    bool ok = true;
    for (; w.left > 0 && ok; ad.next(TA_AHEAD), w.next_unit(p)) {
      int s[4];
      float k[4];
      auto scales = [&] {
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = s[i] >= 0 ? __ldg(p.scale + s[i]) : -1.f;
      };
      auto marked = [&](int i) { return (__float_as_uint(k[i]) & 0x7F800000u) == 0x7F800000u; };
      ta_slots(p, w, lane, s);
      // A marked row among the drafted ones is not read (it meets zero weights).  In the
      // context, which every row sees, it may be: the loads need not wait for the scales.
      const bool drafted = (w.t + 1) * 128 > w.len;
      if (drafted) scales();
      ok = __all_sync(0xFFFFFFFFu, mbar_wait_inl(&sh->a_free[ad.i], ad.ph ^ 1, wc));
      bool whole = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = drafted && marked(i) ? -1 : s[i];
        whole &= at >= 0;
        sh->slot[ad.i][i * 32 + lane] = at;
      }
      whole = __all_sync(0xFFFFFFFFu, whole);
      if (lane == 0) sh->whole[ad.i] = whole;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->a_full[ad.i]);
      if (!drafted) scales();
#pragma unroll
      for (int i = 0; i < 4; ++i) sh->sk[ad.i][i * 32 + lane] = marked(i) ? __uint_as_float(0x7FC00000u) : k[i];
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->sk_full[ad.i]);
    }
  } else if (warp == W_QK) {
    // ================================================================ scores
    if (elect_one()) {
      // descriptors: only the start address (low word, 16-byte units) changes
      const uint64_t k_desc = sdesc_sw128(smem_u32(ks_), 16, 1024), q_desc = sdesc_sw128(smem_u32(qs), 16, 1024);
      const uint32_t id_qk = idesc_e4m3_f32(128, 2 * NR), id_qt = idesc_bf16_f32(128, NR, false, false);
      const uint64_t t_desc = sdesc_sw128(smem_u32(kt), 16, 1024);
      TaRing sl, st, sq;
      uint32_t items = 0;
      bool ok = true;
      for (; w.left > 0 && ok; ++items) {
        const int n = w.here();
        ok = mbar_wait_inl(&sh->q_full, items & 1, wc);
        for (int i = 0; i < n && ok; ++i, sq.next(p.s_bufs)) {
          ok = mbar_wait_inl(&sh->s_free[sq.i], sq.ph ^ 1, wc);
          const uint32_t d = tmem + sq.i * 3 * NR;
          for (int c = 0; c < p.nc && ok; ++c, sl.next(p.slots)) {
            ok = mbar_wait_inl(&sh->full[sl.i], sl.ph, wc);
            tc_fence_after();
            if (!ok) break;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f8_ss(d, k_desc + sl.i * (TA_CHUNK >> 4) + k * 2, q_desc + c * (2 * NR * 8) + k * 2, id_qk,
                         c > 0 || k > 0 ? 1u : 0u);
            if (c >= p.dt) umma_commit(&sh->kfree[sl.i]);
          }
          if (p.dr && ok) {
            ok = mbar_wait_inl(&sh->full[TA_SLOTS + st.i], st.ph, wc);
            tc_fence_after();
            if (ok)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_bf16_ss(d + 2 * NR, t_desc + st.i * (TA_CHUNK >> 4) + k * 2, q_desc + p.nc * (2 * NR * 8) + k * 2,
                             id_qt, k > 0 ? 1u : 0u);
          }
          if (!ok) break;
          umma_commit(&sh->s_full[sq.i]);
          if (p.dr) {
            if (!VT) umma_commit(&sh->kfree[TA_SLOTS + st.i]);
            st.next(p.tails);
          }
        }
        w.next_item(p, n);
      }
      // nothing of this CTA is in flight when it gives its memory back
      umma_commit(&sh->drain[0]);
      mbar_wait(&sh->drain[0], 0, wc, false, true);
    }
    __syncwarp();
  } else if (warp == W_PV) {
    // ================================================================ outputs
    if (elect_one()) {
      const uint64_t v_desc = sdesc_sw128(smem_u32(ks_), TA_CHUNK, 1024), p_desc = sdesc_sw128(smem_u32(ps), 16, 1024);
      const uint64_t pb_desc = sdesc_sw64(smem_u32(pb));
      const uint32_t id_pv = idesc_e4m3_f32(128, NP) | (1u << 10) | (1u << 15) | (1u << 16);  // B e5m2, both MN-major
      const uint32_t id_pt = idesc_bf16_f32(128, NR, true, true);
      const uint64_t vt_desc = sdesc_sw128(smem_u32(kt), TA_CHUNK, 1024);
      TaRing sl, st;
      uint32_t g = 0;
      bool ok = true;
      while (w.left > 0 && ok) {
        const int n = w.here();
        for (int i = 0; i < n; ++i, ++g) {
          ok = mbar_wait_inl(&sh->p_full, g & 1, wc);
          if (!ok) break;
          tc_fence_after();
          for (int m = 0; m < p.nc; ++m, sl.next(p.slots)) {
            if (m >= p.dt) continue;  // read by the scores alone
#pragma unroll
            for (int k = 0; k < 4; ++k)  // 32 keys: 4096 bytes further in both
              umma_f8_ss(tmem + o_col + m * NP, v_desc + sl.i * (TA_CHUNK >> 4) + k * 256, p_desc + k * 256, id_pv,
                         i > 0 || k > 0 ? 1u : 0u);
            umma_commit(&sh->kfree[sl.i]);
          }
          if (VT) {  // 64 dims (the other 64 lanes hold what lies behind them, unused)
#pragma unroll
            for (int k = 0; k < 8; ++k)  // 16 keys: 2048 and 1024 bytes further
              umma_bf16_ss(tmem + ot_col, vt_desc + st.i * (TA_CHUNK >> 4) + k * 128, pb_desc + k * 64, id_pt,
                           i > 0 || k > 0 ? 1u : 0u);
            umma_commit(&sh->kfree[TA_SLOTS + st.i]);
            st.next(p.tails);
          }
          umma_commit(&sh->pv_done);
        }
        w.next_item(p, n);
      }
      umma_commit(&sh->drain[1]);
      mbar_wait(&sh->drain[1], 0, wc, false, true);
    }
    __syncwarp();
  } else {
    // ================================================================ softmax, epilogue
    // After a wait ran out (abort) the loops run on without waiting, so the warps keep
    // meeting at their barriers; nothing here indexes by data.
    const int quarter = warp & 3, hc = (warp >> 2) * CW;  // first row of this thread
    const int key = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    TaRing sq, ad;
    uint32_t g = 0;  // tiles so far: pv_done's phase g - 1 is the last tile's product
    // The queries of item x: hi and lo codes and the bf16 tail, scaled by a power of two
    // per row.  The last scores of the item before are in registers.
    auto queries = [&](const TaWalk& x) {
      constexpr int LR = 16;  // lanes of a row, 8 columns each at a time
      static_assert(NR / (SOFT / 32) == 32 / LR, "every warp takes 32 / LR rows");
      constexpr int QV = 64 / LR;
      const int row = warp * (32 / LR) + lane / LR, at = lane % LR;
      const bool in = x.rt * NR + row < p.rows;
      const uint16_t* q = p.q + ((int64_t)x.b * p.rows + x.rt * NR + row) * (p.dq + p.dr);
      uint4 v[QV], t;
#pragma unroll
      for (int k = 0; k < QV; ++k) v[k] = ldcg_or_zero(q + (k * LR + at) * 8, in && (k * LR + at) * 8 < p.dq);
      t = ldcg_or_zero(q + p.dq + at * 8, in && at * 8 < p.dr);
      // the largest magnitudes, as bf16 bits (in order as integers; from 0x7F80 on not
      // finite): of the code columns in the low half of `top`, of the rotary ones in the high
      auto larger = [](uint32_t& a, uint32_t b) { asm("max.u16x2 %0, %0, %1;" : "+r"(a) : "r"(b)); };
      constexpr uint32_t ABS = 0x7FFF7FFFu;
      uint32_t mc = 0, mt = t.x & ABS;
#pragma unroll
      for (int k = 0; k < QV; ++k) {
        const uint32_t y[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
        for (int z = 0; z < 4; ++z) larger(mc, y[z] & ABS);
      }
      larger(mt, t.y & ABS);
      larger(mt, t.z & ABS);
      larger(mt, t.w & ABS);
      uint32_t top = __byte_perm(mc, mt, 0x5410);  // low halves, then high ones
      larger(top, __byte_perm(mc, mt, 0x7632));
#pragma unroll
      for (int o = LR / 2; o > 0; o >>= 1) larger(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      const uint32_t top_c = top & 0xFFFFu, top_t = top >> 16;
      const bool bad = top_c >= 0x7F80u || top_t >= 0x7F80u;
      // largest code column into [128, 256), rotary ones below 2^(8 + TA_ROTARY)
      const int e = bad ? 0 : max(max((int)(top_c >> 7), (int)(top_t >> 7) - TA_ROTARY) - 127 - 7, -126);
      const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int k = 0; k < QV; ++k) {
        const int c8 = k * LR + at;  // columns 8 c8 .. 8 c8 + 7
        if (c8 >= p.nc * 16) continue;
        const uint32_t y[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
        uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          // (in fp16: below 256 the 8 bits of a bf16 are exact down to 2^-17)
          const uint32_t a = f16x2_of(bf16lo_f32(y[z]) * inv, bf16hi_f32(y[z]) * inv);
          const uint16_t h = e4m3x2_of_f16x2(a);
          const uint32_t rest = mul_f16x2(sub_f16x2(a, f16x2_of_e4m3x2(h)), 0x4C004C00u);  // x 16
          hi[z >> 1] |= (uint32_t)h << (16 * (z & 1));
          lo[z >> 1] |= (uint32_t)e4m3x2_of_f16x2(rest) << (16 * (z & 1));
        }
        uint8_t* dst = qs + (c8 >> 4) * (2 * NR * 128) + row * 128 + ((((c8 & 15) >> 1) ^ (row & 7)) << 4) + (c8 & 1) * 8;
        // a row with a NaN or an infinity scores NaN
        *reinterpret_cast<uint2*>(dst) = bad ? make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu) : make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(dst + NR * 128) = bad ? make_uint2(0u, 0u) : make_uint2(lo[0], lo[1]);
      }
      if (at * 8 < p.dr) {
        const uint32_t m2 = (uint32_t)(127 - e) * 0x00800080u, down = (127u - TA_DOWN) * 0x00800080u;
        auto scaled = [&](uint32_t x) { return bad ? 0u : mul_bf16x2(mul_bf16x2(x, m2), down); };
        *reinterpret_cast<uint4*>(qs + p.nc * (2 * NR * 128) + row * 128 + ((at ^ (row & 7)) << 4)) =
            make_uint4(scaled(t.x), scaled(t.y), scaled(t.z), scaled(t.w));
      }
      if (at == 0) sh->qs[row] = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale_in;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->q_full);
    };
    if (w.left > 0) queries(w);
    named_bar_sync(1, SOFT);
    while (w.left > 0) {
      const int n = w.here();
      const int r0 = w.rt * NR;                      // first row of the tile in the sequence
      const int nrows = min(NR, p.rows - r0);
      const bool whole = w.t == 0 && n == w.nt;      // no other CTA has a part
      TaF2 l2[CW / 2];  // this key lane's sums
#pragma unroll
      for (int c = 0; c < CW / 2; ++c) l2[c] = f2(0.f, 0.f);
      for (int i = 0; i < n; ++i, ++g, sq.next(p.s_bufs), ad.next(TA_AHEAD)) {
        // which rows see this key: all, or a bit per row
        uint32_t allow = 0xFFFFFFFFu;
        const int j = (w.t + i) * 128 + key - w.len;
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
        mbar_wait_inl(&sh->sk_full[ad.i], ad.ph, wc);
        float sk = sh->sk[ad.i][key];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->a_free[ad.i]);
        const bool marked = sk != sk;
        if (sk < 0.f) allow = 0;
        constexpr uint32_t ALL = (1u << CW) - 1u;
        const bool plain = __all_sync(0xFFFFFFFFu, (allow & ALL) == ALL && !marked);
        if (marked || sk < 0.f) sk = 0.f;
        const float sk_log2 = sk > 0.f ? ta_log2(sk) : -INFINITY;
        const float grow = TA_TOP + TA_GROW - sk_log2, tp_max = sh->tp_max;  // (before the scores are there)
        mbar_wait_inl(&sh->s_full[sq.i], sq.ph, wc);
        tc_fence_after();
        TaF2 x[CW / 2];  // scores (base 2) / scale_up
        {
          float hi[CW], lo[CW], tl[CW];
          const uint32_t at = tmem + sq.i * 3 * NR + hc + lane_off;
          tmem_ldn<CW>(at, hi);
          tmem_ldn<CW>(at + NR, lo);
          if (p.dr) tmem_ldn<CW>(at + 2 * NR, tl);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->s_free[sq.i]);
          const float down = sk * (1.f / (1 << TA_DOWN));
          const TaF2 sixteenth = f2(0.0625f, 0.0625f), sk2 = f2(down, down);
#pragma unroll
          for (int c = 0; c < CW; c += 4) {
            const ulonglong2 s4 = *reinterpret_cast<const ulonglong2*>(&sh->qs[hc + c]);
#pragma unroll
            for (int z = c; z < c + 4; z += 2)
              x[z / 2] = mul2(fma2(fma2(f2(lo[z], lo[z + 1]), sixteenth, f2(hi[z], hi[z + 1])), sk2,
                                   p.dr ? f2(tl[z], tl[z + 1]) : f2(0.f, 0.f)),
                              TaF2{z == c ? s4.x : s4.y});
          }
        }
        float d[CW];
        // (scale_up * x is exact, so the difference to a maximum of it is rounded once)
        auto exponents = [&](bool raw) {
          const TaF2 up2 = f2(p.scale_up, p.scale_up);
#pragma unroll
          for (int c = 0; c < CW; c += 4) {
            const ulonglong2 mn = raw ? make_ulonglong2(0, 0) : *reinterpret_cast<const ulonglong2*>(&sh->mneg[hc + c]);
            f2_get(fma2(x[c / 2], up2, TaF2{mn.x}), d[c], d[c + 1]);
            f2_get(fma2(x[c / 2 + 1], up2, TaF2{mn.y}), d[c + 2], d[c + 3]);
          }
          if (!plain) {
#pragma unroll
            for (int c = 0; c < CW; ++c)
              d[c] = !((allow >> c) & 1u) ? -INFINITY : marked ? __uint_as_float(0x7FC00000u) : d[c];
          }
        };
        bool raise = i == 0;
        if (i > 0) {
          exponents(false);
          float most = fmaxf(d[0], d[1]);
#pragma unroll
          for (int c = 2; c < CW; c += 2) most = fmaxf(most, fmaxf(d[c], d[c + 1]));
          bool up = most > TA_RISE;
          if (most + tp_max > grow) {  // some row's P may be too large: which tp has it?
#pragma unroll
            for (int c = 0; c < CW; ++c) up |= d[c] + ta_log2(sh->tp[hc + c]) > grow;
          }
          raise = soft_any<SOFT>(up);
        }
        if (raise) {
          // m goes up to the tile's largest score, m + mr to its largest score + log2 of scale,
          // of every row that has a larger one
          exponents(true);
          ta_maxima(d, sk_log2, &sh->red[quarter][hc], &sh->red_s[quarter][hc], lane);
          named_bar_sync(1, SOFT);
          const int row = lane & (NR - 1);  // (of warp 0, which works on the references)
          auto most = [&](const float (&r)[4][TA_MAX_ROWS]) {
            return fmaxf(fmaxf(r[0][row], r[1][row]), fmaxf(r[2][row], r[3][row]));
          };
          // mr from the tile's largest, which lies `tile` above the new m, and the one before;
          // a row that has seen no key needs none.  m fell by `down`.
          auto settle = [&](float tile, float down) {
            const float old = sh->mr[row];
            const float mr = sh->mneg[row] == INFINITY ? TA_TOP : fmaxf(fmaxf(old + down, tile), -TA_SPAN);
            const float tp = ta_pow2(TA_TOP - ceilf(mr));
            const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(tp));
            if (lane == 0) sh->tp_max = ta_log2(__uint_as_float(top));
            sh->tp[row] = tp;
            sh->mr[row] = mr;
            sh->fs[row] = ex2f(ceilf(old) + down - ceilf(mr));
          };
          float down = 0.f;
          if (warp == 0) {
            const float mo = -sh->mneg[row], mt = most(sh->red), st = most(sh->red_s), mn = fmaxf(mo, mt);
            down = mo == mn ? 0.f : mo - mn;
            const bool wide = __any_sync(0xFFFFFFFFu, fabsf(mn) > 16384.f && fabsf(mn) < INFINITY);
            if (lane == 0) sh->wide = wide;
            sh->f[row] = ex2f(down);
            sh->mneg[row] = -mn;
            __syncwarp();
            if (!wide) settle(st - mn, down);
          }
          named_bar_sync(1, SOFT);
          if (sh->wide) {  // the largest score + log2 of scale from the new m on, exactly
            exponents(false);
#pragma unroll
            for (int c = 0; c < CW; ++c) d[c] += sk_log2;
            ta_maxima(d, 0.f, &sh->red[quarter][hc], &sh->red[quarter][hc], lane);
            named_bar_sync(1, SOFT);
            if (warp == 0) settle(most(sh->red), down);
            named_bar_sync(1, SOFT);
          }
          exponents(false);
          if (i > 0) {  // sums and output follow, once every product before is in it
            bool same = true;
#pragma unroll
            for (int c = 0; c < CW; c += 2) {
              l2[c / 2] = mul2(l2[c / 2], f2(sh->f[hc + c], sh->f[hc + c + 1]));
              same &= sh->f[hc + c] == 1.f && sh->f[hc + c + 1] == 1.f && sh->fs[hc + c] == 1.f && sh->fs[hc + c + 1] == 1.f;
            }
            mbar_wait_inl(&sh->pv_done, (g - 1) & 1, wc);
            tc_fence_after();
            if (!same) {  // (the same for the whole warp)
#pragma unroll 1
              for (int b = 0; b < p.dt * TA_LEVELS + VT; ++b) {
                const float* fr = b < p.dt * TA_LEVELS ? sh->fs : sh->f;
                float o[CW];
                const uint32_t at = tmem + o_col + b * NR + hc + lane_off;
                tmem_ldn<CW>(at, o);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < CW; ++c) o[c] *= fr[hc + c];
                tmem_stn<CW>(at, o);
              }
            }
            tmem_wait_st();
          }
        }
        // weights, their sums, and the three parts of each times scale
        const TaF2 sk2 = f2(sk, sk);
        uint32_t pc[TA_LEVELS][CW / 4], pw[VT ? CW / 2 : 1];
#pragma unroll
        for (int c = 0; c < CW; c += 4) {
          const ulonglong2 tp = *reinterpret_cast<const ulonglong2*>(&sh->tp[hc + c]);
          uint32_t h[2], h1[2], h2[2];
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const float e0 = ex2f(d[c + 2 * z]), e1 = ex2f(d[c + 2 * z + 1]);
            const TaF2 e = f2(e0, e1);
            l2[c / 2 + z] = add2(l2[c / 2 + z], e);
            if constexpr (VT) pw[c / 2 + z] = cvt_bf16x2(e0 * (1.f / (1 << TA_VT)), e1 * (1.f / (1 << TA_VT)));
            float w0, w1;
            f2_get(mul2(mul2(e, TaF2{z ? tp.y : tp.x}), sk2), w0, w1);
            // rounded to nearest: half a last place is added to the magnitude and the low byte
            // dropped (a P of 55109 goes to 57344, the largest e5m2)
            const uint32_t w = f16x2_of(w0, w1);
            h[z] = w + 0x00800080u;
            const uint32_t w_1 = sub_f16x2(w, h[z] & 0xFF00FF00u);
            h1[z] = w_1 + 0x00800080u;
            h2[z] = sub_f16x2(w_1, h1[z] & 0xFF00FF00u) + 0x00800080u;
          }
          pc[0][c / 4] = __byte_perm(h[0], h[1], 0x7531);
          pc[1][c / 4] = __byte_perm(h1[0], h1[1], 0x7531);
          pc[2][c / 4] = __byte_perm(h2[0], h2[1], 0x7531);
        }
        // the previous tile's product has read P
        if (g > 0) mbar_wait_inl(&sh->pv_done, (g - 1) & 1, wc);
#pragma unroll
        for (int v = 0; v < TA_LEVELS; ++v) {
          const int byte = v * NR + hc;
          uint8_t* at = ps + key * 128 + (((byte >> 4) ^ (key & 7)) << 4) + (byte & 15);
          *reinterpret_cast<uint2*>(at) = make_uint2(pc[v][0], pc[v][1]);
        }
        if constexpr (VT) {
          *reinterpret_cast<uint4*>(pb + key * 64 + (((hc >> 3) ^ ((key >> 1) & 3)) << 4)) =
              make_uint4(pw[0], pw[1], pw[2], pw[3]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full);
      }
      // ---- the row tile's part is complete
      {
        float l[CW];
#pragma unroll
        for (int c = 0; c < CW; c += 2) f2_get(l2[c / 2], l[c], l[c + 1]);
        ta_reduce<CW>(l, &sh->red[quarter][hc], lane);
        named_bar_sync(1, SOFT);
        TaWalk x = w;
        x.next_item(p, n);
        if (x.left > 0) queries(x);  // their first scores run during this epilogue
        // a part of a longer row tile: the head of it, or a later piece
        const int slot = 2 * (int)blockIdx.x + (w.t == 0 ? 1 : 0);
        if (threadIdx.x < NR) {
          const int c = threadIdx.x;
          const float m = -sh->mneg[c], mr = ceilf(sh->mr[c]);
          float sum = sh->red[0][c] + sh->red[1][c] + sh->red[2][c] + sh->red[3][c];
          if (whole) {
            if (p.sink && m != -INFINITY)  // (without a key the output is 0 either way)
              sum += ex2f(__ldg(p.sink + (r0 + c) % p.H) * 1.4426950408889634f - m);
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            sh->f[c] = inv * (float)(1 << TA_VT);
            sh->fs[c] = inv * ta_pow2(mr - TA_TOP);
          } else {
            *reinterpret_cast<float4*>(p.part_ml + ((int64_t)slot * NR + c) * 4) = make_float4(m, sum, mr, 0.f);
          }
          sh->mneg[c] = INFINITY;
        }
        if (threadIdx.x == 0 && w.t == 0 && !p.solo && (!whole || p.by_item)) {
          // This CTA's part ends with its stretch; the CTAs after it take `per` tiles each.
          const int parts = whole ? 0 : 1 + (int)((w.nt - n + sh->per - 1) / sh->per);
          *reinterpret_cast<int4*>(p.owner + 4 * (p.by_item ? w.b * p.row_tiles + w.rt : (int)blockIdx.x)) =
              make_int4(w.b, w.rt, parts, (int)blockIdx.x);
        }
        named_bar_sync(1, SOFT);
        mbar_wait_inl(&sh->pv_done, (g - 1) & 1, wc);
        tc_fence_after();
        // dims `dim` (even lanes) and dim + 1 (the next lane) of a row go out together: the
        // even lane stores row c, the odd one row c + 1
        const bool odd = lane & 1;
        auto store = [&](int dim, int dims, const float (&o)[CW], const float* f) {
          if (whole) {
            uint16_t* op = p.out + ((int64_t)w.b * p.rows + r0 + hc + odd) * p.dv + (dim - odd);
#pragma unroll
            for (int c = 0; c < CW; c += 2) {
              const float a = o[c] * f[hc + c], b = o[c + 1] * f[hc + c + 1];
              const float got = __shfl_xor_sync(0xFFFFFFFFu, odd ? a : b, 1);
              if (dim < dims && hc + c + odd < nrows)
                *reinterpret_cast<uint32_t*>(op + (int64_t)c * p.dv) = odd ? cvt_bf16x2(got, b) : cvt_bf16x2(a, got);
            }
          } else {
            float* op = p.part_o + ((int64_t)slot * NR + hc) * p.dv + dim;
#pragma unroll
            for (int c = 0; c < CW; ++c)
              if (dim < dims && hc + c < nrows) op[(int64_t)c * p.dv] = o[c];
          }
        };
#pragma unroll 1
        for (int m = 0; m < p.dt; ++m) {
          float o[CW], o1[CW], o2[CW];
          const uint32_t at = tmem + o_col + m * NP + hc + lane_off;
          tmem_ldn<CW>(at, o);
          tmem_ldn<CW>(at + NR, o1);
          tmem_ldn<CW>(at + 2 * NR, o2);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < CW; ++c) o[c] += o1[c] + o2[c];
          store(m * 128 + key, min(p.dv, p.dq), o, sh->fs);
        }
        if (VT) {
          float o[CW];
          tmem_ldn<CW>(tmem + ot_col + hc + lane_off, o);
          tmem_wait_ld();
          store(p.dq + key, p.dv, o, sh->f);
        }
        tc_fence_before();
        named_bar_sync(1, SOFT);  // f and qs are read by all before the next item's
      }
      w.next_item(p, n);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == W_QK) tmem_dealloc<1>(tmem, p.tmem_cols);
  // after a timed-out wait: no load of this CTA may land once it has gone
  if (threadIdx.x == 0 && sh->abort)
    for (int s = 0; s < TA_SLOTS + 2; ++s)
      if (sh->issued[s]) mbar_wait(&sh->full[s], (sh->issued[s] - 1) & 1, wc, false, true);
}

// Adds up the parts of row tiles that span CTAs, in order: the tile whose head CTA x holds
// has its parts in slots 2 x + 1, 2 (x + 1), 2 (x + 2), ...  A block per row of each entry of
// `owner`; most find no parts where entries are by CTA.  Launched while tree_attn_kernel
// still runs; it waits for its end here.  A chain of load latencies: which tile, the parts'
// maxima and sums, the parts.  Where few row tiles have many parts, entries are by row tile
// and four groups of 128 threads share a row, 16 parts each in flight; else one group with
// 4 in flight (most rows have a few; with 8, 48 ragged sequences take 1 us more).  128 rows
// of 37 parts: 73 us for the call with one group, 69 with four.
constexpr int TA_JOIN_GROUP = 128;  // threads of a row: dv <= 512

template <int NR, int GROUPS>
__global__ void __launch_bounds__(TA_JOIN_GROUP* GROUPS) tree_attn_join_kernel(const TreeAttnParams p) {
  constexpr int FLY = GROUPS > 1 ? 16 : 4;     // parts in flight
  constexpr int PL = (TA_MAX_CTAS + 31) / 32;  // parts of a lane
  // factor of each part, a copy per warp: [0] of columns in units of P, [1] of the bf16 ones
  __shared__ float fs[TA_JOIN_GROUP * GROUPS / 32][2][PL * 32];
  __shared__ float4 sums[GROUPS][TA_JOIN_GROUP];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 ow = *reinterpret_cast<const int4*>(p.owner + (int64_t)blockIdx.x * 4);
  const int parts = ow.z, c = blockIdx.y;
  const int64_t row = (int64_t)ow.y * NR + c;
  if (parts == 0 || row >= p.rows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = threadIdx.x / TA_JOIN_GROUP;
  auto slot = [&](int i) { return i == 0 ? 2 * (int64_t)ow.w + 1 : 2 * ((int64_t)ow.w + i); };
  float4 ml[PL];
#pragma unroll
  for (int k = 0; k < PL; ++k) {
    const int i = k * 32 + lane;
    ml[k] = i < parts ? *reinterpret_cast<const float4*>(p.part_ml + (slot(i) * NR + c) * 4)
                      : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
  }
  float m = ml[0].x;
#pragma unroll
  for (int k = 1; k < PL; ++k) m = fmaxf(m, ml[k].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  float mr = -INFINITY;
#pragma unroll
  for (int k = 0; k < PL; ++k) {
    ml[k].x = ml[k].x == m ? 0.f : ml[k].x - m;
    ml[k].z += ml[k].x;
    mr = fmaxf(mr, ml[k].z);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mr = fmaxf(mr, __shfl_xor_sync(0xFFFFFFFFu, mr, o));
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < PL; ++k) {
    const float f = ex2f(ml[k].x);
    fs[warp][0][k * 32 + lane] = ex2f(ml[k].z - mr);
    fs[warp][1][k * 32 + lane] = f;
    sum += ml[k].y * f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (p.sink && m != -INFINITY) sum += ex2f(__ldg(p.sink + row % p.H) * 1.4426950408889634f - m);
  __syncwarp();
  const int at = threadIdx.x % TA_JOIN_GROUP, d = at * 4, tail = d >= p.dq;  // (dq is a multiple of 4)
  const float inv = (sum == 0.f ? 0.f : 1.f / sum) * (tail ? (float)(1 << TA_VT) : ex2f(mr - TA_TOP));
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d < p.dv)
    for (int base = group; base < parts; base += GROUPS * FLY) {
      float4 v[FLY];
#pragma unroll
      for (int k = 0; k < FLY; ++k) {
        const int i = base + k * GROUPS;
        v[k] = i < parts ? *reinterpret_cast<const float4*>(p.part_o + (slot(i) * NR + c) * p.dv + d)
                         : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < FLY; ++k) {
        const int i = base + k * GROUPS;
        const float f = i < parts ? fs[warp][tail][i] : 0.f;
        o.x += v[k].x * f;
        o.y += v[k].y * f;
        o.z += v[k].z * f;
        o.w += v[k].w * f;
      }
    }
  if constexpr (GROUPS > 1) {
    if (group > 0) sums[group][at] = o;
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int k = 1; k < GROUPS; ++k) {
      const float4 v = sums[k][at];
      o.x += v.x;
      o.y += v.y;
      o.z += v.z;
      o.w += v.w;
    }
  }
  if (d < p.dv)
    *reinterpret_cast<uint2*>(p.out + ((int64_t)ow.x * p.rows + row) * p.dv + d) =
        make_uint2(cvt_bf16x2(o.x * inv, o.y * inv), cvt_bf16x2(o.z * inv, o.w * inv));
}

}  // namespace ks
