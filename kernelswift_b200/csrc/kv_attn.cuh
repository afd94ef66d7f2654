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
// Numbers.  A code times its block's scale, a power of two, is exact in bf16 (4 significant
// bits), so keys and values enter bf16 products as they are; the code's bits are moved into
// place and one multiplication by 2^120 * scale puts the exponent right (e4m3's small numbers
// included).  Where that factor would pass bf16's range the rest of it goes to the scores and
// the weights.  Weights are rounded to bf16 (off by at most 2^-8 of themselves, with a random
// sign; the result is rounded to 2^-8 once more), everything else is fp32.  They are
// taken relative to a reference that is raised when a score passes it by 2^KVA_RISE, and
// 2^-KVA_DOWN smaller, so that sums of values at the top of the range stay finite.
//
// Work: a unit is a tile of 128 keys of one (sequence, row tile, key head); setting one up counts
// as KVA_SETUP more.  The call's units in order are cut into equal stretches, one per CTA,
// whatever the lengths (which only the device knows).  What a CTA has of a row tile that
// others share goes to the workspace (reference, sum, unnormalised output), and
// kv_attn_join_kernel adds the parts up in order (no atomics).
//
// kv_attn_few_kernel: up to 16 rows.  Decoding is bound by reading the cache, and here it goes
// from global memory to registers to the product: a warp takes 16 keys at a time, loads them
// in the layout of mma.m16n8k16's operands (keys as M, rows as N: S^T = K Q^T, then O^T = V^T P^T),
// and no shared memory and no barrier lies between.  8 warps of a CTA take a tile's 16-key
// chunks in turn, each with references, sums and outputs of its own, joined once per row tile.
// A column of a product may come from any column of the head as long as both operands agree,
// so a lane loads 16 contiguous bytes of a key's row; for V^T, 16 bytes of four keys.
#pragma once
#include "kv_cache.cuh"

namespace ks {

constexpr int KVA_SETUP = 2;      // units that a row tile costs beyond its tiles
constexpr float KVA_RISE = 8.f;   // how far a score may pass its reference (base 2)
constexpr float KVA_DOWN = 24.f;  // weights are 2^-24: 2^(8 - 24) * 2^14 keys * 2^128 is finite
constexpr int KVF_WARPS = 8;

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
  int4* owner;            // [CTAs]: sequence, row tile, key head, parts (0: none to join)
  uint64_t budget_ns;
};

struct KvaFind {
  int64_t warp_sum[32];
  int64_t total, per;
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
  const int64_t pairs = (int64_t)p.c.B * p.row_tiles;
  const int64_t each = (pairs + threads - 1) / threads;
  const int64_t i0 = min(tid * each, pairs), i1 = min(i0 + each, pairs);
  int64_t sum = 0;
  for (int64_t i = i0; i < i1; ++i) {
    const int b = (int)(i / p.row_tiles), rt = (int)(i - (int64_t)b * p.row_tiles);
    sum += (int64_t)p.c.heads * (KVA_SETUP + kva_tiles(p, kv_len(p.c, b), kv_new(p.c, b), rt));
  }
  int64_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) f->warp_sum[warp] = incl;
  if (tid == 0) f->left = 0;
  __syncthreads();
  int64_t total = 0, before = 0;
  for (int w = 0; w < threads >> 5; ++w) {
    if (w < warp) before += f->warp_sum[w];
    total += f->warp_sum[w];
  }
  const int64_t per = (total + gridDim.x - 1) / gridDim.x, start = (int64_t)blockIdx.x * per;
  int64_t at = before + incl - sum;
  if (start >= at && start < at + sum) {
    for (int64_t i = i0; i < i1; ++i) {
      const int b = (int)(i / p.row_tiles), rt = (int)(i - (int64_t)b * p.row_tiles);
      const int cost = KVA_SETUP + kva_tiles(p, kv_len(p.c, b), kv_new(p.c, b), rt);
      if (start < at + (int64_t)p.c.heads * cost) {
        f->b = b;
        f->rt = rt;
        f->h = (int)((start - at) / cost);
        f->u = (int)((start - at) % cost);
        f->left = (int)min(per, total - start);
        break;
      }
      at += (int64_t)p.c.heads * cost;
    }
  }
  if (tid == 0) {
    f->total = total;
    f->per = per;
  }
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
  // parts of the row tile, seen from the CTA that has its first tile
  __device__ __forceinline__ int parts(int64_t per) const {
    return (int)((at + KVA_SETUP + nt - 1) / per) - (int)blockIdx.x + 1;
  }
};

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
// Bits of e4m3 codes in the high bytes of two halves to bf16 2^-120 times as large.
__device__ __forceinline__ uint32_t kva_place(uint32_t x) { return ((x >> 4) & 0x07F007F0u) | (x & 0x80008000u); }

__device__ __forceinline__ float kva_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
  if (has_sink) l += kva_ex2(sink_log2 - (m == -INFINITY ? 0.f : m) - KVA_DOWN);
  return l == 0.f ? 0.f : 1.f / l;  // (a NaN stays one)
}

// ------------------------------------------------------------------ few rows
__device__ __forceinline__ void kvf_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t kvf_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <int W>
__device__ __forceinline__ void kvf_load(uint32_t (&v)[W], const uint8_t* ptr) {
  if constexpr (W == 4)
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "l"(ptr));
  else
    asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "l"(ptr));
}

constexpr int KVF_HDR = 2048;
template <int NR>
struct KvfShared {
  KvaFind find;
  float m[KVF_WARPS][NR], l[KVF_WARPS][NR];  // of the warps
};
static_assert(sizeof(KvfShared<16>) <= KVF_HDR, "KvfShared exceeds its header");

// Where 16 keys lie.
struct KvfChunk {
  int64_t row;      // of the page pool's rows of heads
  uint32_t ks, vs;  // bits of the scales, 0: the page is not there
};

template <int D>
__device__ __forceinline__ int kvf_page(const KvAttnParams& p, int b, int pos, int keys) {
  const int pi = kva_div(pos, p.c.page, p.page_shift);
  return pos < keys ? __ldg(p.c.table + (int64_t)b * p.c.max_pages + pi) : 0;
}

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
  float* kvf_smem = reinterpret_cast<float*>(kvf_raw + KVF_HDR);  // [4][NR][D] outputs of four warps
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  kva_find(p, &find);
  KvaWalk w;
  w.start(p, &find);
  if (tid == 0) p.owner[blockIdx.x] = make_int4(0, 0, 0, 0);
  const int per_page = p.c.page / p.c.block;

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
    auto locate = [&](int pos, int pg, KvfChunk* k) {
      const int in = pos - kva_div(pos, p.c.page, p.page_shift) * p.c.page;
      const bool ok = pg >= 0 && pg < p.c.n_pages;
      if (!ok && lane == 0) report_bounds(p.c.status, w.b, (int)p.c.n_pages);
      const int64_t unit = (int64_t)(ok ? pg : 0) * p.c.heads + w.h;
      k->row = unit * p.c.page + in;
      const int64_t si = unit * per_page + kva_div(in, p.c.block, p.block_shift);
      k->ks = __float_as_uint(__ldg(p.c.k_scale + si));
      k->vs = __float_as_uint(__ldg(p.c.v_scale + si));
      if (!ok) k->ks = 0xFFFFFFFFu;
    };
    uint32_t kr[2][KJ][4], vr[4][VU][VW];
    auto load_k = [&](const KvfChunk& k) {
      const uint8_t* base = p.c.k8 + (k.row + r) * D + c * 16;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < KJ; ++j) kvf_load<4>(kr[i][j], base + i * 8 * D + j * 64);
    };
    auto load_v = [&](const KvfChunk& k) {
      const uint8_t* base = p.c.v8 + (k.row + 2 * c) * D + r * (4 * VW);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VU; ++j) kvf_load<VW>(vr[i][j], base + ((i & 1) + (i >> 1) * 8) * D + j * (32 * VW));
    };

    KvfChunk cur{}, nxt{};
    int pg1 = 0;
    if (ci < chunks) {
      const int pg0 = kvf_page<D>(p, w.b, ci * 16, w.keys);
      pg1 = kvf_page<D>(p, w.b, (ci + KVF_WARPS) * 16, chunks * 16);
      locate(ci * 16, pg0, &cur);
      load_k(cur);
      load_v(cur);
    }
    // queries as the second operand: word i of piece j holds columns 16 (c + 4 j) + 4 i ..
    uint32_t qf[NT][KJ * 4][2];
#pragma unroll
    for (int g = 0; g < NT; ++g) {
      const int row = r0 + g * 8 + r, t = row / p.G;
      const uint16_t* qp = p.q + (((int64_t)w.b * p.c.T + t) * p.H + w.h * p.G + (row - t * p.G)) * D;
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (row < p.rows) {
          a = __ldg(reinterpret_cast<const uint4*>(qp + 16 * (c + 4 * j)));
          b = __ldg(reinterpret_cast<const uint4*>(qp + 16 * (c + 4 * j) + 8));
        }
        const uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // codes 0 and 2 of a word go together, and 1 and 3
          qf[g][j * 4 + i][0] = __byte_perm(x[2 * i], x[2 * i + 1], 0x5410);
          qf[g][j * 4 + i][1] = __byte_perm(x[2 * i], x[2 * i + 1], 0x7632);
        }
      }
    }
    float m[NT][2], mu[NT][2], l[NT][2], o[NT][D / 16][4];
    uint32_t nanv[NT][2];  // columns of the lane's outputs that are NaN
#pragma unroll
    for (int g = 0; g < NT; ++g) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[g][i] = -INFINITY;
        mu[g][i] = KVA_DOWN;
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
      // ---------------------------------------------------------- scores
      float s[NT][4];
#pragma unroll
      for (int g = 0; g < NT; ++g) s[g][0] = s[g][1] = s[g][2] = s[g][3] = 0.f;
      float rest_k, rest_v;
      const bool there = cur.ks != 0xFFFFFFFFu;
      const uint32_t fk = kva_factor(there ? cur.ks : 0u, &rest_k), fv = kva_factor(cur.vs, &rest_v);
      const bool marked = there && ((cur.ks | cur.vs) & 1u);
      uint32_t nan_k = 0;  // of the lane's two keys, bit 0 and 1
      if (marked) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < KJ; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) nan_k |= (kva_nan4(kr[i][j][x]) ? 1u : 0u) << i;
        nan_k |= __shfl_xor_sync(0xFFFFFFFFu, nan_k, 1);
        nan_k |= __shfl_xor_sync(0xFFFFFFFFu, nan_k, 2);
      }
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x0 = kr[0][j][i], x1 = kr[1][j][i];
          const uint32_t a[4] = {mul_bf16x2(kva_place(x0 << 8), fk), mul_bf16x2(kva_place(x1 << 8), fk),
                                 mul_bf16x2(kva_place(x0), fk), mul_bf16x2(kva_place(x1), fk)};
#pragma unroll
          for (int g = 0; g < NT; ++g) kvf_mma(s[g], a, qf[g][j * 4 + i][0], qf[g][j * 4 + i][1]);
        }
      // ---------------------------------------------------------- the next keys
      const bool more = ci + KVF_WARPS < chunks;
      if (more) {
        locate(pos + KVF_WARPS * 16, pg1, &nxt);
        load_k(nxt);
        pg1 = kvf_page<D>(p, w.b, pos + 2 * KVF_WARPS * 16, chunks * 16);
      }
      // ---------------------------------------------------------- weights
      // lane: keys r and r + 8, columns 2 c and 2 c + 1 of each group
      const float sc = p.scale_log2 * rest_k;
      bool rise = false;
      const bool open = there && !marked && pos + 16 <= clear;
#pragma unroll
      for (int g = 0; g < NT; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[g][i] *= sc;
          if (!open) {
            const int row = r0 + g * 8 + 2 * c + (i & 1);
            if ((nan_k >> (i >> 1)) & 1u) s[g][i] = __uint_as_float(0x7FC00000u);
            if (!there || !kva_sees(p, w.b, w.len, w.n, row / p.G, pos + r + (i >> 1) * 8)) s[g][i] = -INFINITY;
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
            const float f = now == -INFINITY ? 1.f : kva_ex2(m[g][i] - now);
            m[g][i] = now;
            mu[g][i] = (now == -INFINITY ? 0.f : now) + KVA_DOWN;
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
          e[i] = kva_ex2(s[g][i] - mu[g][i & 1]);
          l[g][i & 1] += e[i];
          e[i] *= rest_v;
        }
        pb[g][0] = kvf_trans(cvt_bf16x2(e[0], e[1]));
        pb[g][1] = kvf_trans(cvt_bf16x2(e[2], e[3]));
      }
      // ---------------------------------------------------------- outputs
      if (marked) {
        // codes that are NaN count as zero in the product; the rows that see them get NaN
        uint32_t bits[4];  // of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9, by the lane's columns
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
            const int at = pos + 2 * y + (i & 1) + (i >> 1) * 8;
            if (of) {
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
            const uint32_t sel0 = h ? 0x6020u : 0x4000u, sel1 = h ? 0x7030u : 0x5010u;
            const uint32_t a[4] = {mul_bf16x2(kva_place(__byte_perm(vr[0][j][x], vr[1][j][x], sel0)), fv),
                                   mul_bf16x2(kva_place(__byte_perm(vr[0][j][x], vr[1][j][x], sel1)), fv),
                                   mul_bf16x2(kva_place(__byte_perm(vr[2][j][x], vr[3][j][x], sel0)), fv),
                                   mul_bf16x2(kva_place(__byte_perm(vr[2][j][x], vr[3][j][x], sel1)), fv)};
#pragma unroll
            for (int g = 0; g < NT; ++g) kvf_mma(o[g][(j * VW + x) * 2 + h], a, pb[g][0], pb[g][1]);
          }
      if (more) {
        load_v(nxt);
        cur = nxt;
      }
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
          sm_l[warp][g * 8 + 2 * c + i] = l[g][i];
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
        const float f = top == -INFINITY ? 1.f : kva_ex2(m[g][i] - top);
#pragma unroll
        for (int y = 0; y < D / 16; ++y) {
          o[g][y][i] *= f;
          o[g][y][i + 2] *= f;
          // bits y * 2 and y * 2 + 1: the tile's columns, in the order of the lane's codes
          if ((nanv[g][i] >> (2 * y)) & 1u) o[g][y][i] = __uint_as_float(0x7FC00000u);
          if ((nanv[g][i] >> (2 * y + 1)) & 1u) o[g][y][i + 2] = __uint_as_float(0x7FC00000u);
        }
      }
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
        sum += top == -INFINITY ? sm_l[x][row] : sm_l[x][row] * kva_ex2(sm_m[x][row] - top);
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
    if (tid == 0 && !whole && w.t0 == 0) p.owner[blockIdx.x] = make_int4(w.b, w.rt, w.h, w.parts(find.per));
    __syncthreads();
  }
}

// Parts of a row tile that several CTAs share, added up in order.  Block (c, y): rows y, y +
// gridDim.y, .. of the row tile whose first tile CTA c has.
__global__ void __launch_bounds__(256) kv_attn_join_kernel(const __grid_constant__ KvAttnParams p) {
  const int4 own = p.owner[blockIdx.x];
  if (own.w == 0) return;
  const int b = own.x, r0 = own.y * p.nr, h = own.z, parts = own.w, d = p.c.d, per_row = d >> 2;
  const int n = kv_new(p.c, b);
  const int lane_row = threadIdx.x / per_row, rows = blockDim.x / per_row;  // rows of the block at once
  for (int row = blockIdx.y * rows + lane_row; row - lane_row < p.nr; row += gridDim.y * rows) {
    if (lane_row >= rows || row >= p.nr || r0 + row >= p.rows) continue;
    const int t = (r0 + row) / p.G, g = (r0 + row) - t * p.G, col = (threadIdx.x - lane_row * per_row) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, sum = 0.f;
    for (int i = 0; i < parts; ++i) {
      const int64_t slot = i ? 2 * ((int64_t)blockIdx.x + i) : 2 * (int64_t)blockIdx.x + 1;
      top = fmaxf(top, __ldg(&p.part_ml[slot * p.nr + row]).x);
    }
    for (int i = 0; i < parts; ++i) {
      const int64_t slot = i ? 2 * ((int64_t)blockIdx.x + i) : 2 * (int64_t)blockIdx.x + 1;
      const float2 ml = __ldg(&p.part_ml[slot * p.nr + row]);
      const float4 y = __ldg(reinterpret_cast<const float4*>(p.part_o + (slot * p.nr + row) * d + col));
      const float f = top == -INFINITY ? 1.f : kva_ex2(ml.x - top);
      sum += f * ml.y;
      v.x += f * y.x; v.y += f * y.y; v.z += f * y.z; v.w += f * y.w;
    }
    const float f = kva_norm(top, sum, p.sink ? __ldg(p.sink + h * p.G + g) * 1.4426950408889634f : 0.f, p.sink);
    *reinterpret_cast<uint2*>(p.out + (((int64_t)b * p.c.T + t) * p.H + h * p.G + g) * d + col) =
        t < n ? make_uint2(cvt_bf16x2(v.x * f, v.y * f), cvt_bf16x2(v.z * f, v.w * f)) : make_uint2(0, 0);
  }
}

}  // namespace ks
