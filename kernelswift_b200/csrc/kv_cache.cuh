// A paged cache of keys and values per head (grouped queries) in e4m3, with one power-of-two
// scale for each block of tokens and head: appending to it, with the position rotation.
//
// k8, v8 [pages, heads, page, D], k_scale, v_scale [pages, heads, page / block].  Position i of
// a sequence is row i % page of page table[i / page]; a block is `block` rows in order, so a
// head's rows of a page lie together and a block's are one stretch of block * D bytes.
//
//   x    = the new row, its last rd columns rotated as pairs (2 i, 2 i + 1) by freqs[position],
//          in fp32 and not rounded before it is quantised (values: not rotated)
//   s    = the smallest power of two >= max(max |x|, 1e-4) / 448 over the block's new rows, at most
//          2^119; where the block holds rows of the sequence already, not less than before
//   code = e4m3(x / s), nearest even.  Where s grew, the rows that were there are rounded again
//          to the new scale, from their codes: exact but for what falls below e4m3's range.
//
// Marking: an element that is NaN or infinite becomes e4m3's NaN, and the lowest bit of its
// block's scale is set (2^e (1 + 2^-23)), so a reader tests a bit per block instead of every
// code.  A block that begins anew forgets what the page held.
//
// One CTA per (sequence, block that the call touches, head, keys or values): it alone reads and
// writes the block, so there are no races and no atomics; every row is read once and kept in
// registers between the maximum and the conversion.  Further CTAs rotate the queries.
// Bound by memory, for few rows by launch latency.  Measured (one B200): two prompts of 16384 tokens,
// 32 query and 8 key heads of 128, all columns rotated, blocks of 16: 165 to 168 us (755 MB, 4.5 TB/s,
// 0.70 of a copy's rate; issue slots 80 %, so the rotation and the conversion count: with values held
// in bf16 between maximum and conversion, and rotated twice, 238 us; cos and sin, 512 bytes a token, are
// read again for every head); blocks of 64 231 us (more registers a thread, fewer CTAs an SM); one
// token of 8 sequences 5.5 us on the device.
#pragma once
#include <cuda_fp16.h>

#include "quant_fp8.cuh"

namespace ks {

constexpr int KV_MAX_BLOCK = 128;
constexpr int KV_Q_PIECES = 4;  // 8-column pieces of queries per thread

struct KvCache {
  uint8_t* k8;
  float* k_scale;
  uint8_t* v8;
  float* v_scale;
  int64_t n_pages, max_pages;
  const int32_t* table;  // [B, max_pages]
  const int32_t* lens;   // [B]: tokens that are cached before the call's
  const int32_t* n_new;  // [B] or null: tokens of the call that are there (else T)
  int32_t heads, page, block, d;
  int32_t B, T;
  int* status;
};

__device__ __forceinline__ int kv_len(const KvCache& c, int b) { return max(0, __ldg(c.lens + b)); }
__device__ __forceinline__ int kv_new(const KvCache& c, int b) {
  return c.n_new ? min(max(0, __ldg(c.n_new + b)), c.T) : c.T;
}

struct KvAppendParams {
  KvCache c;
  const uint16_t* k;     // bf16 [B, T, heads, D], rows of a token together
  const uint16_t* v;
  const uint16_t* q;     // bf16 [B, T, q_heads, D] or null
  uint16_t* q_out;       // contiguous
  int64_t k_bs, k_ts, v_bs, v_ts, q_bs, q_ts;  // elements from sequence to sequence, token to token
  const float* freqs;    // [n_freqs, rd / 2, 2] or null
  const int32_t* pos;    // [B, T] or null: positions of the rotation
  int32_t n_freqs;
  int32_t page_shift, block_shift, row_shift;  // of page, block and D / 8; -1: not a power of two
  int32_t rd, q_heads;
  int32_t nb;            // blocks that T tokens may touch
  int64_t kv_ctas;
  int64_t q_pieces;      // of all queries
};

// The smallest power of two >= max(amax, 1e-4) / 448, at most 2^119 (448 * 2^119 is finite).
__device__ __forceinline__ float kv_power(float amax) {
  const float f = __fdiv_rn(fmaxf(amax, 1e-4f), 448.f);
  const uint32_t u = __float_as_uint(f);
  return fminf((u & 0x007FFFFFu) ? __uint_as_float((u & 0x7F800000u) + 0x00800000u) : f,
               __uint_as_float((119u + 127u) << 23));
}

// Eight columns from column c0 on, in fp32, rotated where they are among the last rd.  Each
// product and sum is rounded on its own, so results do not depend on how they are fused.
__device__ __forceinline__ void kv_rotate8(const uint4& raw, float (&y)[8], const float* freqs, int row, int rd, int c0) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = bf16lo_f32(w[i]);
    y[2 * i + 1] = bf16hi_f32(w[i]);
  }
  if (c0 >= 0 && freqs) {  // c0: column among the rotated ones
    const float4* f = reinterpret_cast<const float4*>(freqs + (int64_t)row * rd + c0);
    const float4 f0 = __ldg(f), f1 = __ldg(f + 1);
    const float cs[4] = {f0.x, f0.z, f1.x, f1.z}, sn[4] = {f0.y, f0.w, f1.y, f1.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = y[2 * i], b = y[2 * i + 1];
      y[2 * i] = __fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(b, sn[i]));
      y[2 * i + 1] = __fadd_rn(__fmul_rn(a, sn[i]), __fmul_rn(b, cs[i]));
    }
  }
}

// Row of freqs for token t of sequence b, at position `at`; false where there is none.
__device__ __forceinline__ bool kv_freq_row(const KvAppendParams& p, int b, int t, int at, int* row) {
  const int r = p.pos ? __ldg(p.pos + (int64_t)b * p.c.T + t) : at;
  *row = min(max(r, 0), p.n_freqs - 1);
  return r == *row;
}
__device__ __forceinline__ uint32_t kv_div(uint32_t x, int d, int shift) { return shift >= 0 ? x >> shift : x / (uint32_t)d; }

__device__ __forceinline__ float e4m3_f32(uint32_t code) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
  return __half2float(__ushort_as_half((unsigned short)h));
}

// NP: 8-column pieces of the block per thread (block * D / 8 <= NP * THREADS).
template <int NP, int THREADS>
__global__ void __launch_bounds__(THREADS, NP <= 2 ? 1280 / THREADS : 1) kv_append_kernel(const __grid_constant__ KvAppendParams p) {
  const KvCache& c = p.c;
  constexpr int threads = THREADS;
  const int per_row = c.d >> 3, tid = threadIdx.x;
  if (blockIdx.x >= p.kv_ctas) {
    // ------------------------------------------------------------ queries
    // (pieces of all queries are below 2^32)
    const uint32_t first = (uint32_t)(blockIdx.x - p.kv_ctas) * (threads * KV_Q_PIECES) + tid;
    const uint32_t per_token = (uint32_t)(p.q_heads * per_row), pieces = (uint32_t)p.q_pieces;
    uint32_t token = first / per_token, at = first - token * per_token;
    int b = (int)(token / (uint32_t)c.T), t = (int)(token - (uint32_t)b * (uint32_t)c.T);
    uint4 raw[KV_Q_PIECES];
    int frow[KV_Q_PIECES];
    int col[KV_Q_PIECES];
#pragma unroll
    for (int i = 0; i < KV_Q_PIECES; ++i) {
      raw[i] = make_uint4(0, 0, 0, 0);
      frow[i] = 0;
      col[i] = -1;
      if (first + i * threads < pieces) {
        raw[i] = __ldcs(reinterpret_cast<const uint4*>(p.q + b * p.q_bs + t * p.q_ts + (int64_t)at * 8));
        col[i] = (int)(at - kv_div(at, per_row, p.row_shift) * per_row) * 8 - (c.d - p.rd);
        if (col[i] >= 0) kv_freq_row(p, b, t, kv_len(c, b) + t, &frow[i]);
      }
      at += threads;
      while (at >= per_token) {
        at -= per_token;
        if (++t == c.T) {
          t = 0;
          ++b;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < KV_Q_PIECES; ++i) {
      const uint32_t e = first + i * threads;
      if (e >= pieces) break;
      float y[8];
      kv_rotate8(raw[i], y, p.freqs, frow[i], p.rd, col[i]);
      reinterpret_cast<uint4*>(p.q_out)[e] =
          col[i] < 0 ? raw[i]
                     : make_uint4(cvt_bf16x2(y[0], y[1]), cvt_bf16x2(y[2], y[3]), cvt_bf16x2(y[4], y[5]),
                                  cvt_bf16x2(y[6], y[7]));
    }
    return;
  }
  // -------------------------------------------------------------- keys and values
  // head fastest, so that neighbouring CTAs read neighbouring columns of the same tokens
  const uint32_t id = blockIdx.x;
  const int part = (int)(id % (uint32_t)(2 * c.heads));
  const uint32_t rest = id / (uint32_t)(2 * c.heads);
  const int ib = (int)(rest % (uint32_t)p.nb), b = (int)(rest / (uint32_t)p.nb);
  const bool is_k = part < c.heads;
  const int head = is_k ? part : part - c.heads;
  const int len = kv_len(c, b), n = kv_new(c, b);
  // the block's first position, and the rows of it that the call writes
  const int64_t start = ((int64_t)(len / c.block) + ib) * c.block;
  const int lo = (int)max((int64_t)0, len - start);
  const int hi = (int)min((int64_t)c.block, (int64_t)len + n - start);
  if (hi <= lo) return;
  // the rows are on their way while the page is looked up
  const uint16_t* x = is_k ? p.k + b * p.k_bs : p.v + b * p.v_bs;
  const int64_t ts = is_k ? p.k_ts : p.v_ts;
  const float* freqs = is_k ? p.freqs : nullptr;

  uint4 raw[NP];
  int row[NP], col[NP];  // of the piece in the block; -1: not the call's
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int e = tid + i * threads;
    row[i] = (int)kv_div(e, per_row, p.row_shift);
    col[i] = (e - row[i] * per_row) * 8;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (row[i] >= lo && row[i] < hi)
      raw[i] = __ldcs(reinterpret_cast<const uint4*>(x + (start + row[i] - len) * ts + (int64_t)head * c.d + col[i]));
    else
      row[i] = -1;
  }
  const uint32_t pi = kv_div((uint32_t)min(start, (int64_t)0x7FFFFFFF), c.page, p.page_shift);
  const int32_t pg = pi < c.max_pages ? __ldg(c.table + (int64_t)b * c.max_pages + pi) : -1;
  if (pg < 0 || pg >= c.n_pages) {
    if (tid == 0 && head == 0)
      report_bounds(c.status, b, (int)min(pi < c.max_pages ? c.n_pages : c.max_pages, (int64_t)0x7FFFFFFF));
    return;
  }
  const int64_t unit = (int64_t)pg * c.heads + head;
  const int in_page = (int)(start - (int64_t)pi * c.page), in_block = (int)kv_div(in_page, c.block, p.block_shift);
  uint8_t* codes = (is_k ? c.k8 : c.v8) + (unit * c.page + in_page) * c.d;
  float* scale = (is_k ? c.k_scale : c.v_scale) + unit * kv_div(c.page, c.block, p.block_shift) + in_block;
  const float old_raw = lo > 0 ? *scale : 0.f;
  float y[NP][8], amax = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    int fr = 0;
    const int rc = row[i] < 0 || !freqs ? -1 : col[i] - (c.d - p.rd);
    if (rc >= 0 && !kv_freq_row(p, b, (int)(start + row[i] - len), (int)start + row[i], &fr))
      report_bounds(c.status, b, p.n_freqs);
    kv_rotate8(raw[i], y[i], freqs, fr, p.rd, rc);  // (zeros where the row is not the call's)
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(y[i][j]));
  }
  __shared__ float red[2][THREADS / 32];
  const auto largest = [&](float (&r)[THREADS / 32], float a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xFFFFFFFFu, a, o));
    if ((tid & 31) == 0) r[tid >> 5] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) a = max_nan(a, r[w]);
    return a;
  };
  amax = largest(red[0], amax);
  bool bad = !(amax < INFINITY);
  if (bad) {  // (the whole block) the finite ones' largest; the others become NaN
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (fabsf(y[i][j]) < INFINITY) amax = fmaxf(amax, fabsf(y[i][j]));
        else y[i][j] = __uint_as_float(0x7FC00000u);
      }
    amax = largest(red[1], amax);
  }
  const uint32_t old_bits = __float_as_uint(old_raw);
  bad |= (old_bits & 1u) != 0;
  const float old = __uint_as_float(old_bits & ~1u);
  const float s = fmaxf(kv_power(amax), old);
  const float inv = __uint_as_float((254u << 23) - (__float_as_uint(s) & 0x7F800000u));  // 1 / s
  if (lo > 0 && s > old) {
    const float ratio = old * inv;
    for (int e = tid; e < lo * per_row; e += threads) {
      uint2* at = reinterpret_cast<uint2*>(codes + (int64_t)e * 8);
      const uint2 w = *at;
      uint32_t o[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t u = h ? w.y : w.x;
        o[h] = cvt_e4m3x2(e4m3_f32(u & 255) * ratio, e4m3_f32((u >> 8) & 255) * ratio) |
               (uint32_t)cvt_e4m3x2(e4m3_f32((u >> 16) & 255) * ratio, e4m3_f32(u >> 24) * ratio) << 16;
      }
      *at = make_uint2(o[0], o[1]);
    }
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (row[i] < 0) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[i][j] *= inv;
    const uint32_t a = cvt_e4m3x2(y[i][0], y[i][1]) | (uint32_t)cvt_e4m3x2(y[i][2], y[i][3]) << 16;
    const uint32_t d = cvt_e4m3x2(y[i][4], y[i][5]) | (uint32_t)cvt_e4m3x2(y[i][6], y[i][7]) << 16;
    *reinterpret_cast<uint2*>(codes + row[i] * c.d + col[i]) = make_uint2(a, d);
  }
  if (tid == 0) *scale = __uint_as_float(__float_as_uint(s) | (bad ? 1u : 0u));
}

}  // namespace ks
