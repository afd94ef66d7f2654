// Attention over the per-head cache in 8 bits (kv_cache.cuh): what the kernels share, and the
// kernel for few query rows per key head.
//
//   s[k] = scale * q . c_k,  o = sum_k exp(s_k - m) v_k / (sum_k exp(s_k - m) + exp(sink - m))
//
// The H / heads query heads of a key head and the T tokens are the rows of one product:
// row r is token r / G, head r % G of the group.  Token t of sequence b sees the lens[b] cached
// positions and, of the call's tokens (cached behind them), those its mask row allows, without
// a mask the ones up to itself.
//
// Numbers.  Scores, sums and outputs are fp32; what is rounded to 16 bits are the weights, and
// what a key or value holds is exact in either 16-bit type (4 significant bits).
//   few rows: fp16 products on the codes themselves, converted by the hardware.  A query row
//     enters times a power of two that brings its largest element below 2^15; elements 2^-30 of
//     that and less go into further terms (rarely: then the scores take another pass).  Weights
//     are off by at most 2^-11 of themselves, or 2^-32 of the reference's (which no largest
//     weight is below): they show where all larger ones meet zeros.  A chunk's scale
//     multiplies its scores, and its part of the output when that is added up.
//   many rows: a tile's output is added up in tensor memory, so scales have to be in the
//     operands: bf16, the code's bits moved into place and one multiplication by 2^120 * scale to
//     put the exponent right (e4m3's small numbers included).  Weights are rounded to bf16, off
//     by at most 2^-8 of themselves, with a random sign; the result is rounded by as much.
// Weights are taken relative to a reference that is raised when a score passes it by
// 2^KVA_RISE, and 2^-KVA_DOWN smaller in outputs and sums, so that sums of values at the top of
// the range stay finite.
//
// Work: a unit is a tile of 128 keys of one (sequence, row tile, key head); setting one up counts
// as KVA_SETUP more.  The call's units in order are cut into equal stretches, one per CTA,
// whatever the lengths (which only the device knows).  What a CTA has of a row tile that
// others share goes to the workspace (reference, sum, unnormalised output), and
// kv_attn_join_kernel adds the parts up in order (no atomics).
//
// kv_attn_few_kernel: up to 16 rows.  Decoding is bound by reading the cache.  Every warp works on
// its own: it takes 16 keys at a time (their codes are one stretch of memory), has those of two
// more such chunks on their way into its ring in shared memory (cp.async; no barrier but the
// warp's), and reads a chunk in the layout of mma.m16n8k16's operands, keys as M, rows as N:
// S^T = K Q^T, then O^T = V^T P^T.  8 warps of a CTA take a tile's chunks in turn, each with
// references, sums and outputs of its own, joined once per row tile.
// A column of a product may come from any column of the head as long as both operands agree,
// and a row of it from any key: a lane reads 16 contiguous bytes of a key's row, for V^T 16 bytes
// of four keys, and keys are assigned to the product's rows (kvf_key) so that neither read has
// bank conflicts.
// Measured (one B200, join included): 64 heads on 8 key heads of 128, one token over 131069 keys
// (268 MB) 66 us, 4.1 TB/s: the loop alone runs at 0.84 of a copy's rate, and 25 us are start, ends
// and join.  48 sequences up to 8000 keys, 40 heads on 8 (403 MB) 108 to 112 us, 3.7 TB/s; with 128
// heads (16 rows a key head: 254 registers, one CTA an SM) 184.  Short contexts are bound by row tiles
// taken one after the other, each a chain of lookups and loads, and four barriers: 300 sequences up
// to 60 keys, 2400 row tiles, 78 us for 24 MB.  At heads of 128 (and of 64 with 16 rows) the cap of 128
// registers, which two CTAs an SM need, spills 60 bytes of stores and 88 of loads (44 and 76).  The first
// form (operands from global memory to registers, bf16 by integer operations, one join group a
// row) took 82 us: ALU 60 % of its cycles, now 45 %.  Not taken: the next row tile's queries and
// places fetched ahead (spills: 109 us), the rare further terms of a query out of line (68 us).
#pragma once
#include "kv_cache.cuh"

namespace ks {

// Units that a row tile costs beyond its tiles, for both kernels.  Measured (us, L2 flushed) with 1, 2, 4, 6,
// 10: one sequence of 509 keys 16.5, 16.5, 16.6, 18.2, 18.4, since CTAs of nothing but setting up come
// on top of the parts; 40 sequences up to 500 keys 31.8, 31.6, 32.8, 33.4, 32.7; 48 up to 8000 keys 129,
// 118, 105, 100, 100; 16 trees of 13 129, 108, 102, 97, 99; one of 131069 keys 82, 79, 78, 78, 77; a chunk
// of 4096 tokens the same with all.  Two keeps the small calls; a value for each kernel and size,
// which the ragged ones ask for, is not built.
constexpr int KVA_SETUP = 2;
constexpr float KVA_RISE = 8.f;   // how far a score may pass its reference (base 2)
constexpr float KVA_DOWN = 24.f;  // weights are 2^-24: 2^(8 - 24) * 2^14 keys * 2^128 is finite
constexpr int KVF_WARPS = 8;
constexpr float KVF_TOP = 7.f;    // weights of the few-row kernel are 2^7 at the reference: below 2^16 in fp16
constexpr int KVF_TERM = 30;      // exponents of a query row that one term holds

struct KvAttnParams {
  KvCache c;
  const uint16_t* q;      // bf16 [B, T, H, D]
  uint16_t* out;          // bf16 [B, T, H, D]
  const uint8_t* mask;    // [B, T, T] or null
  const float* sink;      // [H] or null
  int32_t H, G, rows;     // rows: T * G of a (sequence, key head)
  int32_t nr, row_tiles;  // rows of a row tile
  int32_t page_shift, block_shift;  // -1: not a power of two
  float scale_log2;       // softmax scale * log2 e
  float* part_o;          // [2 * CTAs][nr][D]
  float2* part_ml;        // [2 * CTAs][nr]: reference, sum
  int4* owner;            // sequence, row tile, key head, parts << 10 | CTA of the first one (0: none to join)
  int32_t by_item;        // owner is indexed by row tile of the call (they are fewer), else by CTA
  uint64_t budget_ns;
};

struct KvaFind {
  uint32_t warp_sum[32];
  uint32_t per;
  int32_t left, b, rt, h, u;
};

// Keys that row tile rt of a sequence may see.
__device__ __forceinline__ int kva_keys(const KvAttnParams& p, int len, int n, int rt) {
  if (rt * p.nr >= n * p.G) return 0;  // none of its tokens is there
  const int t1 = min((min((rt + 1) * p.nr, p.rows) - 1) / p.G, n - 1);
  const int64_t keys = (int64_t)len + (p.mask ? n : t1 + 1);
  return (int)min(keys, p.c.max_pages * p.c.page);
}
__device__ __forceinline__ int kva_tiles(const KvAttnParams& p, int len, int n, int rt) {
  return (kva_keys(p, len, n, rt) + 127) >> 7;
}

// This CTA's stretch: its first row tile, the unit in it, and how many units.  All threads.
__device__ __forceinline__ void kva_find(const KvAttnParams& p, KvaFind* f) {
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
  // (sequence, row tile) pairs, so many per thread; all units together are below 2^31
  const uint32_t tiles = (uint32_t)p.row_tiles, pairs = (uint32_t)p.c.B * tiles;
  const uint32_t each = (pairs + threads - 1) / threads, i0 = min(tid * each, pairs), i1 = min(i0 + each, pairs);
  const auto cost = [&](uint32_t i) {
    const int b = (int)(i / tiles), rt = (int)(i - b * tiles);
    return (uint32_t)(KVA_SETUP + kva_tiles(p, kv_len(p.c, b), kv_new(p.c, b), rt));
  };
  uint32_t sum = 0;
  for (uint32_t i = i0; i < i1; ++i) sum += p.c.heads * cost(i);
  uint32_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) f->warp_sum[warp] = incl;
  if (tid == 0) f->left = 0;
  __syncthreads();
  uint32_t total = 0, before = 0;
  for (int w = 0; w < threads >> 5; ++w) {
    if (w < warp) before += f->warp_sum[w];
    total += f->warp_sum[w];
  }
  const uint32_t per = (total + gridDim.x - 1) / gridDim.x;
  const uint64_t start = (uint64_t)blockIdx.x * per;
  uint32_t at = before + incl - sum;
  if (start >= at && start < (uint64_t)at + sum) {
    for (uint32_t i = i0; i < i1; ++i) {
      const uint32_t c = cost(i), in = (uint32_t)start - at;
      if (in < p.c.heads * c) {
        f->b = (int)(i / tiles);
        f->rt = (int)(i % tiles);
        f->h = (int)(in / c);
        f->u = (int)(in % c);
        f->left = (int)min(per, total - (uint32_t)start);
        break;
      }
      at += p.c.heads * c;
    }
  }
  if (tid == 0) f->per = per;
  __syncthreads();
}

// A CTA's stretch, walked row tile by row tile; the same in every thread.
struct KvaWalk {
  int left, b, rt, h, u;  // units to go; the row tile and the unit in it
  int len, n, keys, nt;   // of the sequence; keys and tiles of the row tile
  int t0, t1;             // tiles that are this CTA's
  int64_t at;             // the row tile's first unit in the call
  __device__ __forceinline__ void item(const KvAttnParams& p) {
    keys = kva_keys(p, len, n, rt);
    nt = (keys + 127) >> 7;
    t0 = max(u - KVA_SETUP, 0);
    t1 = min(max(u + left - KVA_SETUP, 0), nt);
  }
  __device__ __forceinline__ void start(const KvAttnParams& p, const KvaFind* f) {
    left = f->left; b = f->b; rt = f->rt; h = f->h; u = f->u;
    at = (int64_t)blockIdx.x * f->per - u;
    if (left <= 0) return;
    len = kv_len(p.c, b);
    n = kv_new(p.c, b);
    item(p);
  }
  __device__ __forceinline__ void next(const KvAttnParams& p) {
    left -= KVA_SETUP + nt - u;
    at += KVA_SETUP + nt;
    u = 0;
    if (left <= 0) return;
    if (++h == p.c.heads) {
      h = 0;
      if (++rt == p.row_tiles) {
        rt = 0;
        ++b;
        len = kv_len(p.c, b);
        n = kv_new(p.c, b);
      }
    }
    item(p);
  }
  __device__ __forceinline__ bool any() const { return t1 > t0; }
  // nothing to see: the CTA that has the first unit writes the zeros
  __device__ __forceinline__ bool empty() const { return nt == 0 && u == 0; }
  __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == nt; }
  // where a part goes: a CTA shares its first row tile with the CTAs before it, its last one
  // with those behind
  __device__ __forceinline__ int slot() const { return 2 * (int)blockIdx.x + (t0 > 0 ? 0 : 1); }
  // what the CTA that has a shared row tile's first tile leaves for the join
  __device__ __forceinline__ void share(const KvAttnParams& p, uint32_t per) const {
    const int parts = (int)((at + KVA_SETUP + nt - 1) / per) - (int)blockIdx.x + 1;
    p.owner[p.by_item ? (b * p.row_tiles + rt) * p.c.heads + h : (int)blockIdx.x] = make_int4(b, rt, h, parts << 10 | (int)blockIdx.x);
  }
};
// Nothing to join yet.  A thread clears what it alone may set later: its CTA's entry, or those of
// the row tiles whose first tile (or nothing at all) is in its stretch.
__device__ __forceinline__ void kva_clear(const KvAttnParams& p, KvaWalk w) {
  if (!p.by_item) {
    p.owner[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  for (; w.left > 0; w.next(p))
    if (w.empty() || (w.any() && w.t0 == 0)) p.owner[(w.b * p.row_tiles + w.rt) * p.c.heads + w.h] = make_int4(0, 0, 0, 0);
}

__device__ __forceinline__ bool kva_sees(const KvAttnParams& p, int b, int len, int n, int t, int pos) {
  const int j = pos - len;
  if (t >= n || j >= n) return false;
  if (j < 0) return true;
  return p.mask ? __ldg(p.mask + ((int64_t)b * p.c.T + t) * p.c.T + j) != 0 : j <= t;
}

__device__ __forceinline__ int kva_div(int x, int d, int shift) { return shift >= 0 ? x >> shift : x / d; }

// 2^120 * scale as bf16 (twice), or the largest power of two there is; *rest is what is missing.
__device__ __forceinline__ uint32_t kva_factor(uint32_t scale_bits, float* rest) {
  const uint32_t e = (scale_bits >> 23) & 255u;
  const uint32_t f = e ? min(e + 120u, 254u) : 0u;
  *rest = __uint_as_float((e + 120u > 254u ? e + 120u - 254u + 127u : 127u) << 23);
  return (f << 7) * 0x00010001u;
}

// Codes that are NaN among four, as bits 7, 15, 23, 31.
__device__ __forceinline__ uint32_t kva_nan4(uint32_t w) {
  return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
}
// The same, each in the lowest of four bits.
__device__ __forceinline__ uint32_t kva_nan4_bits(uint32_t w) {
  const uint32_t x = kva_nan4(w) >> 7;
  return (x | x >> 7 | x >> 14 | x >> 21) & 15u;
}

// A row's result: bf16 of o / den, zeros where nothing is seen.
__device__ __forceinline__ float kva_norm(float m, float l, float sink_log2, bool has_sink) {
  if (has_sink) l += ex2f(sink_log2 - (m == -INFINITY ? 0.f : m) - KVA_DOWN);
  return l == 0.f ? 0.f : 1.f / l;  // (a NaN stays one)
}

// ------------------------------------------------------------------ few rows
__device__ __forceinline__ void kvf_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t kvf_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t kvf_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Codes 0, 1 and codes 2, 3 of a word as fp16 pairs.
__device__ __forceinline__ void kvf_codes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h; }"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float kvf_pow2(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }

// A query row's 16 columns from d on, as the second operand of four steps: those elements of
// 2^sh times the row that are in [2^-15, 2^15), the first term's also above (infinite, NaN).
__device__ __forceinline__ void kvf_query(const uint16_t* q, bool in, int sh, bool first, uint32_t (&b)[4][2]) {
  uint4 x = make_uint4(0, 0, 0, 0), y = x;
  if (in) {
    x = __ldg(reinterpret_cast<const uint4*>(q));
    y = __ldg(reinterpret_cast<const uint4*>(q + 8));
  }
  const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  const float f = kvf_pow2(sh);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float lo = bf16lo_f32(w[i]) * f, hi = bf16hi_f32(w[i]) * f;
    if (fabsf(lo) < 0x1p-15f || (!first && fabsf(lo) >= 0x1p15f)) lo = 0.f;
    if (fabsf(hi) < 0x1p-15f || (!first && fabsf(hi) >= 0x1p15f)) hi = 0.f;
    b[i >> 1][i & 1] = kvf_f16x2(lo, hi);
  }
}

template <int W>
__device__ __forceinline__ void kvf_lds(uint32_t (&v)[W], uint32_t addr) {
  if constexpr (W == 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr));
  else
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr));
}

// Key (of 8, and of the 8 behind) that row i of a product stands for, and where 16-byte piece u
// of a key's row lies in a chunk.  Of a quarter warp's lanes, two product rows and four
// pieces meet in a read of keys, four product rows (every other one) and two pieces in one of
// values: all eight in different banks.
template <int D>
__device__ __forceinline__ int kvf_key(int i) {
  return (int)((D % 128 == 0 ? 0x37156240u : 0x67324510u) >> (4 * i)) & 7;
}
template <int D>
__device__ __forceinline__ int kvf_at(int key, int u) {
  return key * D + (D % 128 == 0 ? ((u & ~7) | ((u ^ key) & 7)) : (u ^ (key & 2))) * 16;
}
constexpr int KVF_STAGES = 3;

constexpr int KVF_HDR = 2048;
template <int NR>
struct KvfShared {
  KvaFind find;
  float m[KVF_WARPS][NR], l[KVF_WARPS][NR];  // of the warps
};
static_assert(sizeof(KvfShared<16>) <= KVF_HDR, "KvfShared exceeds its header");

// Scales (bits) of a chunk; ks = KVF_GONE: the page is not there (the first page's codes stand in for
// it, in bounds, with weights and a value scale of zero).
struct KvfChunk {
  uint32_t ks, vs;
};
constexpr uint32_t KVF_GONE = 0xFFFFFFFFu;

// D: columns of a head, NT: 8-row groups.
template <int D, int NT>
__global__ void __launch_bounds__(KVF_WARPS * 32, D * NT <= 128 ? 2 : 1) kv_attn_few_kernel(const __grid_constant__ KvAttnParams p) {
  constexpr int NR = 8 * NT, KJ = D / 64;        // 64-column pieces of a key row
  constexpr int VW = D % 128 == 0 ? 4 : 2;       // words of a value piece
  constexpr int VU = D / (32 * VW);              // value pieces of a lane per key
  extern __shared__ __align__(16) uint8_t kvf_raw[];
  KvfShared<NR>& sh = *reinterpret_cast<KvfShared<NR>*>(kvf_raw);
  KvaFind& find = sh.find;
  auto& sm_m = sh.m;
  auto& sm_l = sh.l;
  float* kvf_smem = reinterpret_cast<float*>(kvf_raw + KVF_HDR);  // [4][NR][D] outputs of four warps, at the end
  // a warp's ring: [stages][keys, values][16 keys x D]
  const uint32_t ring = smem_u32(kvf_raw + KVF_HDR) + (threadIdx.x >> 5) * (KVF_STAGES * 32 * D);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join may be set up
  kva_find(p, &find);
  KvaWalk w;
  w.start(p, &find);
  if (tid == 0) kva_clear(p, w);
  const int per_page = p.c.page / p.c.block;
  const int key_r = kvf_key<D>(r), key_v[2] = {kvf_key<D>(2 * c), kvf_key<D>(2 * c + 1)};

  for (; w.left > 0; w.next(p)) {
    const int r0 = w.rt * NR;
    if (w.empty()) {
      for (int i = tid; i < NR * (D / 8); i += KVF_WARPS * 32) {
        const int row = r0 + i / (D / 8), t = row / p.G;
        if (row < p.rows)
          reinterpret_cast<uint4*>(p.out + (((int64_t)w.b * p.c.T + t) * p.H + w.h * p.G + row % p.G) * D)[i % (D / 8)] =
              make_uint4(0, 0, 0, 0);
      }
    }
    if (!w.any()) continue;
    if (tid == 0 && (int64_t)w.len + w.n > p.c.max_pages * p.c.page)
      report_bounds(p.c.status, w.b, (int)p.c.max_pages);
    const int chunks = min(w.t1 * 8, (w.keys + 15) >> 4);

    int ci = w.t0 * 8 + warp;
    // Lane l knows where the l-th chunk from here is and its scales, for 32 chunks at a time.
    // (A chunk's rows lie at 16 D times its place; places fit 32 bits.)
    uint32_t place = 0, ks32 = KVF_GONE, vs32 = 0;
    const auto locate = [&](int first) {
      const int pos = (first + KVF_WARPS * lane) * 16;
      if (pos < chunks * 16) {
        const int pi = kva_div(pos, p.c.page, p.page_shift), in = pos - pi * p.c.page;
        const int pg = __ldg(p.c.table + (int64_t)w.b * p.c.max_pages + pi);
        const bool ok = pg >= 0 && pg < p.c.n_pages;
        if (!ok) report_bounds(p.c.status, w.b, (int)p.c.n_pages);
        const uint32_t unit = (ok ? (uint32_t)pg : 0u) * (uint32_t)p.c.heads + (uint32_t)w.h;
        const uint32_t si = unit * (uint32_t)per_page + (uint32_t)kva_div(in, p.c.block, p.block_shift);
        place = unit * (uint32_t)(p.c.page >> 4) + (uint32_t)(in >> 4);
        ks32 = ok ? __float_as_uint(__ldg(p.c.k_scale + si)) : KVF_GONE;
        vs32 = ok ? __float_as_uint(__ldg(p.c.v_scale + si)) : 0u;
      }
    };
    // starts the copies of the n-th chunk from the first
    const auto fetch = [&](int n, int stage, KvfChunk* k) {
      const uint32_t at16 = __shfl_sync(0xFFFFFFFFu, place, n & 31);
      k->ks = __shfl_sync(0xFFFFFFFFu, ks32, n & 31);
      k->vs = __shfl_sync(0xFFFFFFFFu, vs32, n & 31);
      const int64_t at = (int64_t)at16 * (16 * D) + lane * 16;
      const uint8_t *ksrc = p.c.k8 + at, *vsrc = p.c.v8 + at;
      const uint32_t dst = ring + stage * (32 * D);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int e = lane + 32 * i, key = e / (D / 16), u = e - key * (D / 16);
        const uint32_t to = dst + kvf_at<D>(key, u);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(ksrc + 512 * i) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16 * D), "l"(vsrc + 512 * i) : "memory");
      }
    };
    KvfChunk cur{}, n1{}, n2{};
    int stage = 0, n_fetched = 2;
    locate(ci);
    if (ci < chunks) fetch(0, 0, &cur);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (ci + KVF_WARPS < chunks) fetch(1, 1, &n1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    // queries as the second operand: piece j of a lane holds columns 16 (c + 4 j) ..
    uint32_t qf[NT][KJ][4][2];
    int sh[NT];            // exponents that the lane's rows were moved by
    float qsc[NT][2];      // of the lane's score columns: softmax scale, back by as much
    int terms = 1;
    const auto query_row = [&](int g) {
      const int row = min(r0 + g * 8 + r, p.rows - 1), t = row / p.G;
      return p.q + (((int64_t)w.b * p.c.T + t) * p.H + w.h * p.G + (row - t * p.G)) * D + 16 * c;
    };
#pragma unroll
    for (int g = 0; g < NT; ++g) {
      const uint16_t* qp = query_row(g);
      // exponents of the largest and the least element (bits of |x|, zeros left out)
      uint32_t most = 0, least = 0x7F80u;
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(qp + 64 * j)), y = __ldg(reinterpret_cast<const uint4*>(qp + 64 * j + 8));
        const uint32_t e[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t lo = e[i] & 0x7FFFu, hi = (e[i] >> 16) & 0x7FFFu;
          most = max(most, max(lo, hi));
          least = min(least, min(lo ? lo : 0x7F80u, hi ? hi : 0x7F80u));
        }
      }
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, x));
        least = min(least, __shfl_xor_sync(0xFFFFFFFFu, least, x));
      }
      // (numbers below 2^-126 have the exponent of their first bit)
      const int top = (int)(most >> 7) - 127, low = least < 128u ? -102 - __clz(least) : (int)(least >> 7) - 127;
      sh[g] = 14 - top;
      if (r0 + g * 8 + r < p.rows && most < 0x7F80u && low < top) terms = max(terms, (top - low) / KVF_TERM + 1);
    }
    terms = __reduce_max_sync(0xFFFFFFFFu, terms);
#pragma unroll
    for (int g = 0; g < NT; ++g) {
      // Every row goes through as many terms as the one that needs most.  Their windows follow each
      // other without overlap: a row's first factor is small enough for its last one to be at most
      // 2^126, whose window reaches down to 2^-141, below bf16's least number.
      sh[g] = min(sh[g], 126 - KVF_TERM * (terms - 1));
#pragma unroll
      for (int j = 0; j < KJ; ++j) kvf_query(query_row(g) + 64 * j, r0 + g * 8 + r < p.rows, sh[g], true, qf[g][j]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int back = -__shfl_sync(0xFFFFFFFFu, sh[g], (2 * c + i) * 4);
        qsc[g][i] = p.scale_log2 * kvf_pow2(back);
      }
    }
    float m[NT][2], mu[NT][2], l[NT][2], o[NT][D / 16][4];
    uint32_t nanv[NT][2];  // columns of the lane's outputs that are NaN
#pragma unroll
    for (int g = 0; g < NT; ++g) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[g][i] = -INFINITY;
        mu[g][i] = -KVF_TOP;
        l[g][i] = 0.f;
        nanv[g][i] = 0;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[g][i][0] = o[g][i][1] = o[g][i][2] = o[g][i][3] = 0.f;
    }
    // positions below this are seen by every row
    const int clear = w.len + (p.mask ? 0 : r0 / p.G + 1);

    for (; ci < chunks; ci += KVF_WARPS) {
      const int pos = ci * 16;
      // ---------------------------------------------------------- the copies
      __syncwarp();  // the stage that is filled next has been read
      if (ci + 2 * KVF_WARPS < chunks) {
        if ((n_fetched & 31) == 0) locate(ci + 2 * KVF_WARPS);
        fetch(n_fetched++, stage == 0 ? 2 : stage - 1, &n2);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 2;" ::: "memory");
      __syncwarp();
      const uint32_t kb = ring + stage * (32 * D), vb = kb + 16 * D;
      uint32_t kr[2][KJ][4], vr[4][VU][VW];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < KJ; ++j) kvf_lds<4>(kr[i][j], kb + kvf_at<D>(key_r + 8 * i, c + 4 * j));
      // ---------------------------------------------------------- scores
      // (two sums side by side: a product waits for the one before it in its sum)
      float s[NT][4], s_odd[NT][4];
#pragma unroll
      for (int g = 0; g < NT; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[g][i] = s_odd[g][i] = 0.f;
      const bool there = cur.ks != KVF_GONE;
      const bool marked = there && (cur.vs & 1u);
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t a[4];
          kvf_codes(kr[0][j][i], a[0], a[2]);
          kvf_codes(kr[1][j][i], a[1], a[3]);
#pragma unroll
          for (int g = 0; g < NT; ++g) kvf_mma(i & 1 ? s_odd[g] : s[g], a, qf[g][j][i][0], qf[g][j][i][1]);
        }
      // (The product of the factors may pass the range where the score does not, at zero codes; scores
      // beyond 2^103 may come out smaller.  A softmax scale and a power that are below 2^-126 together put
      // a score off by at most 2^-118 times the key scale, which shows for keys above 2^100 alone.)
      const float ks = __uint_as_float(cur.ks & 0x7F800000u), vs = __uint_as_float(cur.vs & 0x7F800000u) * 0x1p-31f;
      const auto factor = [&](float back) { return fminf(fmaxf(back * ks, -3e38f), 3e38f); };
#pragma unroll
      for (int g = 0; g < NT; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[g][i] = (s[g][i] + s_odd[g][i]) * factor(qsc[g][i & 1]);
#pragma unroll 1
      for (int t = 1; t < terms; ++t) {  // elements of a query far below its largest
#pragma unroll
        for (int g = 0; g < NT; ++g) {
          float s1[4] = {0.f, 0.f, 0.f, 0.f};
          const uint16_t* qp = query_row(g);
          const int sh1 = sh[g] + KVF_TERM * t;
#pragma unroll
          for (int j = 0; j < KJ; ++j) {
            uint32_t q1[4][2];
            kvf_query(qp + 64 * j, r0 + g * 8 + r < p.rows, sh1, false, q1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a[4];
              kvf_codes(kr[0][j][i], a[0], a[2]);
              kvf_codes(kr[1][j][i], a[1], a[3]);
              kvf_mma(s1, a, q1[i][0], q1[i][1]);
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float f = factor(p.scale_log2 * kvf_pow2(-__shfl_sync(0xFFFFFFFFu, sh1, (2 * c + i) * 4)));
            s[g][i] += s1[i] * f;
            s[g][i + 2] += s1[i + 2] * f;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VU; ++j) {
          const int u8 = r + 8 * j;  // VW words each
          kvf_lds<VW>(vr[i][j], vb + (VW == 4 ? kvf_at<D>(key_v[i & 1] + 8 * (i >> 1), u8)
                                              : kvf_at<D>(key_v[i & 1] + 8 * (i >> 1), u8 >> 1) + (u8 & 1) * 8));
        }
      // ---------------------------------------------------------- weights
      // lane: product rows r and r + 8, columns 2 c and 2 c + 1 of each group
      bool rise = false;
      const bool open = there && !marked && pos + 16 <= clear;
#pragma unroll
      for (int g = 0; g < NT; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!open) {
            const int row = r0 + g * 8 + 2 * c + (i & 1);
            if (!there || !kva_sees(p, w.b, w.len, w.n, row / p.G, pos + key_r + (i >> 1) * 8)) s[g][i] = -INFINITY;
          }
          rise |= s[g][i] > m[g][i & 1] + KVA_RISE;
        }
      if (__any_sync(0xFFFFFFFFu, rise)) {
#pragma unroll
        for (int g = 0; g < NT; ++g)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(s[g][i], s[g][i + 2]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
            const float now = fmaxf(m[g][i], top);
            const float f = now == -INFINITY ? 1.f : ex2f(m[g][i] - now);
            m[g][i] = now;
            mu[g][i] = (now == -INFINITY ? 0.f : now) - KVF_TOP;
            l[g][i] *= f;
#pragma unroll
            for (int y = 0; y < D / 16; ++y) {
              o[g][y][i] *= f;
              o[g][y][i + 2] *= f;
            }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int g = 0; g < NT; ++g) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = ex2f(s[g][i] - mu[g][i & 1]);
          l[g][i & 1] += e[i];
        }
        pb[g][0] = kvf_trans(kvf_f16x2(e[0], e[1]));
        pb[g][1] = kvf_trans(kvf_f16x2(e[2], e[3]));
      }
      // ---------------------------------------------------------- outputs
      if (!open) {
        // codes that are NaN (also those behind the last row, of which nothing is known) count
        // as zero in the product; the rows that see them get NaN (none sees a page that is not there)
        uint32_t bits[4];  // of the lane's four keys, by its columns
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bits[i] = 0;
#pragma unroll
          for (int j = 0; j < VU; ++j)
#pragma unroll
            for (int x = 0; x < VW; ++x) {
              const uint32_t nan = kva_nan4(vr[i][j][x]);
              bits[i] |= kva_nan4_bits(vr[i][j][x]) << ((j * VW + x) * 4);
              vr[i][j][x] &= ~((nan >> 7) * 255u);
            }
        }
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t of = __shfl_sync(0xFFFFFFFFu, bits[i], (lane & ~3) | y);
            const int at = pos + kvf_key<D>(2 * y + (i & 1)) + (i >> 1) * 8;
            if (of && there) {
#pragma unroll
              for (int g = 0; g < NT; ++g)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                  if (kva_sees(p, w.b, w.len, w.n, (r0 + g * 8 + 2 * c + x) / p.G, at)) nanv[g][x] |= of;
            }
          }
      }
#pragma unroll
      for (int j = 0; j < VU; ++j)
#pragma unroll
        for (int x = 0; x < VW; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // columns 4 x + 2 h, + 1 of the piece
            const uint32_t sel = h ? 0x7362u : 0x5140u;  // two keys' codes of a column side by side
            uint32_t a[4];
            kvf_codes(__byte_perm(vr[0][j][x], vr[1][j][x], sel), a[0], a[1]);
            kvf_codes(__byte_perm(vr[2][j][x], vr[3][j][x], sel), a[2], a[3]);
#pragma unroll
            for (int g = 0; g < NT; ++g) {
              float t[4] = {0.f, 0.f, 0.f, 0.f};
              kvf_mma(t, a, pb[g][0], pb[g][1]);
#pragma unroll
              for (int i = 0; i < 4; ++i) o[g][(j * VW + x) * 2 + h][i] = fmaf(t[i], vs, o[g][(j * VW + x) * 2 + h][i]);
            }
          }
      cur = n1;
      n1 = n2;
      stage = stage == 2 ? 0 : stage + 1;
    }

    // ------------------------------------------------------------ the warps' results together
#pragma unroll
    for (int g = 0; g < NT; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[g][i] += __shfl_xor_sync(0xFFFFFFFFu, l[g][i], x);
        if (r == 0) {
          sm_m[warp][g * 8 + 2 * c + i] = m[g][i];
          sm_l[warp][g * 8 + 2 * c + i] = l[g][i] * 0x1p-31f;  // as the outputs (2^(KVF_TOP - 31) = 2^-KVA_DOWN)
        }
      }
    __syncthreads();
    // (element of output tile y: column base + (y / 2 % VW) * 4 + (y & 1) * 2 + {0, 1})
    const auto put = [&](float* dst, bool add) {
#pragma unroll
      for (int g = 0; g < NT; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int y = 0; y < D / 16; ++y) {
            const int j = y / (2 * VW), at = y % (2 * VW) * 2;
            float2* e = reinterpret_cast<float2*>(dst + (g * 8 + 2 * c + i) * D + (r + 8 * j) * (4 * VW) + at);
            float2 v = make_float2(o[g][y][i], o[g][y][i + 2]);
            if (add) {
              const float2 q = *e;
              v.x += q.x;
              v.y += q.y;
            }
            *e = v;
          }
    };
#pragma unroll
    for (int g = 0; g < NT; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < KVF_WARPS; ++x) top = fmaxf(top, sm_m[x][g * 8 + 2 * c + i]);
        const float f = top == -INFINITY ? 1.f : ex2f(m[g][i] - top);
#pragma unroll
        for (int y = 0; y < D / 16; ++y) {
          o[g][y][i] *= f;
          o[g][y][i + 2] *= f;
          // bits y * 2 and y * 2 + 1: the tile's columns, in the order of the lane's codes
          if ((nanv[g][i] >> (2 * y)) & 1u) o[g][y][i] = __uint_as_float(0x7FC00000u);
          if ((nanv[g][i] >> (2 * y + 1)) & 1u) o[g][y][i + 2] = __uint_as_float(0x7FC00000u);
        }
      }
    // (every warp is past its ring, which lies where the outputs go: the barrier above)
    if (warp >= 4) put(kvf_smem + (warp - 4) * NR * D, false);
    __syncthreads();
    if (warp < 4) put(kvf_smem + warp * NR * D, true);
    __syncthreads();
    const bool whole = w.whole();
    for (int i = tid; i < NR * (D / 4); i += KVF_WARPS * 32) {
      const int row = i / (D / 4), col = (i - row * (D / 4)) * 4;
      const float* e = kvf_smem + row * D + col;
      float4 v = *reinterpret_cast<const float4*>(e);
#pragma unroll
      for (int x = 1; x < 4; ++x) {
        const float4 y = *reinterpret_cast<const float4*>(e + x * NR * D);
        v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
      }
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int x = 0; x < KVF_WARPS; ++x) top = fmaxf(top, sm_m[x][row]);
#pragma unroll
      for (int x = 0; x < KVF_WARPS; ++x)
        sum += top == -INFINITY ? sm_l[x][row] : sm_l[x][row] * ex2f(sm_m[x][row] - top);
      if (whole) {
        const int t = (r0 + row) / p.G, g = (r0 + row) - t * p.G;
        if (r0 + row < p.rows) {
          const float f = t < w.n ? kva_norm(top, sum, p.sink ? __ldg(p.sink + w.h * p.G + g) * 1.4426950408889634f : 0.f, p.sink) : 0.f;
          const uint2 b = t < w.n ? make_uint2(cvt_bf16x2(v.x * f, v.y * f), cvt_bf16x2(v.z * f, v.w * f)) : make_uint2(0, 0);
          *reinterpret_cast<uint2*>(p.out + (((int64_t)w.b * p.c.T + t) * p.H + w.h * p.G + g) * D + col) = b;
        }
      } else {
        const int64_t slot = w.slot();
        *reinterpret_cast<float4*>(p.part_o + (slot * NR + row) * D + col) = v;
        if (col == 0) p.part_ml[slot * NR + row] = make_float2(top, sum);
      }
    }
    if (tid == 0 && !whole && w.t0 == 0) w.share(p, find.per);
    __syncthreads();
  }
}

// Parts of a row tile that several CTAs share, added up.  Blocks (x, y): a row tile, or the one whose
// first tile CTA x has where there are more row tiles than CTAs; some of its rows each.  D / 4
// threads take a row; where there are many parts (one long sequence) up to eight of such groups
// take every eighth part each, with a reference of their own, and are added up in order.  Latency:
// the owner record, then the parts.  (64 heads over 131069 keys, 37 parts a row tile: 6 us under a
// profiler; with one group a row 30 us of the call's 76.)
__global__ void __launch_bounds__(256) kv_attn_join_kernel(const __grid_constant__ KvAttnParams p) {
  __shared__ float4 sv[256];
  __shared__ float2 sml[256];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // until all parts are written
  const int4 own = p.owner[blockIdx.x];
  if (own.w == 0) return;
  const int b = own.x, r0 = own.y * p.nr, h = own.z, parts = own.w >> 10, d = p.c.d, per_row = d >> 2;
  const int64_t cta = own.w & 1023;
  const int n = kv_new(p.c, b), at_once = blockDim.x / per_row;
  int groups = 1;
  while (groups * 2 <= at_once && groups * 4 < parts) groups *= 2;
  const int rows = at_once / groups;
  const int set = threadIdx.x / per_row, col = (threadIdx.x - set * per_row) * 4, grp = set % groups, mine = set / groups;
  for (int first = blockIdx.y * rows; first < p.nr && r0 + first < p.rows; first += gridDim.y * rows) {
    const int row = first + mine;
    const bool in = mine < rows && row < p.nr && r0 + row < p.rows;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, sum = 0.f;
    const auto take = [&](const float2 ml, const float4 y) {
      const float now = fmaxf(top, ml.x);
      const float f0 = now == -INFINITY ? 1.f : ex2f(top - now), f1 = now == -INFINITY ? 1.f : ex2f(ml.x - now);
      top = now;
      sum = f0 * sum + f1 * ml.y;
      v = make_float4(f0 * v.x + f1 * y.x, f0 * v.y + f1 * y.y, f0 * v.z + f1 * y.z, f0 * v.w + f1 * y.w);
    };
    if (in) {
#pragma unroll 4
      for (int i = grp; i < parts; i += groups) {
        const int64_t at = (i ? 2 * (cta + i) : 2 * cta + 1) * p.nr + row;
        take(p.part_ml[at], *reinterpret_cast<const float4*>(p.part_o + at * d + col));
      }
    }
    if (groups > 1) {
      __syncthreads();  // (the row before has been read)
      sv[threadIdx.x] = v;
      sml[threadIdx.x] = make_float2(top, sum);
      __syncthreads();
      if (grp == 0 && in)
        for (int i = 1; i < groups; ++i) take(sml[threadIdx.x + i * per_row], sv[threadIdx.x + i * per_row]);
    }
    if (grp == 0 && in) {
      const int t = (r0 + row) / p.G, g = (r0 + row) - t * p.G;
      const float f = kva_norm(top, sum, p.sink ? __ldg(p.sink + h * p.G + g) * 1.4426950408889634f : 0.f, p.sink);
      *reinterpret_cast<uint2*>(p.out + (((int64_t)b * p.c.T + t) * p.H + h * p.G + g) * d + col) =
          t < n ? make_uint2(cvt_bf16x2(v.x * f, v.y * f), cvt_bf16x2(v.z * f, v.w * f)) : make_uint2(0, 0);
    }
  }
}

}  // namespace ks
