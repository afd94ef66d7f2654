// Attention of drafted tokens over the quantised latent cache.
//
//   s[k] = scale * q . c_k,  o = sum_k exp(s_k - m) v_k / (sum_k exp(s_k - m) + exp(sink - m))
//
// with c_k the cached row of position k (latent_cache.cuh), v_k its first dv columns.
// A drafted token of sequence b sees the lens[b] cached positions and, among the T
// drafted rows that follow them in the cache, those its row of the mask allows (without
// a mask: itself and the ones before it).
//
// One CTA per (sequence, token, 8 heads); each warp takes every 8th key, lanes share
// its columns, and the running maximum, sum and output of a softmax per head live in
// registers.  The warps' parts meet in shared memory.
#pragma once
#include "latent_cache.cuh"

namespace ks {

constexpr int TA_WARPS = 8;
constexpr int TA_HEADS = 8;
constexpr int TA_MAX_CHUNKS = 9;  // 64-column chunks of a row

struct TreeAttnParams {
  const uint16_t* q;      // bf16 [B, T, H, D]
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
  float scale_log2;
  int* status;
};

__global__ void __launch_bounds__(TA_WARPS * 32) tree_attn_simple_kernel(TreeAttnParams p) {
  __shared__ float sq[TA_HEADS][TA_MAX_CHUNKS * 64];
  __shared__ float sm[TA_WARPS][TA_HEADS], sl[TA_WARPS][TA_HEADS];
  const int D = p.dq + p.dr, nq = p.dq / 64, nc = D / 64, nv = p.dv / 64;
  const int hg = (p.H + TA_HEADS - 1) / TA_HEADS;
  const int64_t bt = blockIdx.x / hg;
  const int h0 = (int)(blockIdx.x % hg) * TA_HEADS;
  const int64_t b = bt / p.T;
  const int t = (int)(bt - b * p.T);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < TA_HEADS * D; i += blockDim.x) {
    const int h = i / D, c = i % D;
    sq[h][c] = h0 + h < p.H ? __uint_as_float((uint32_t)p.q[(bt * p.H + h0 + h) * D + c] << 16) : 0.f;
  }
  __syncthreads();
  const int len = max(0, __ldg(p.lens + b));
  float m[TA_HEADS], l[TA_HEADS], o[TA_HEADS][2 * (TA_MAX_CHUNKS - 1)];
#pragma unroll
  for (int h = 0; h < TA_HEADS; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * (TA_MAX_CHUNKS - 1); ++i) o[h][i] = 0.f;
  }
  for (int k = warp; k < len + p.T; k += TA_WARPS) {
    if (k >= len) {
      const int j = k - len;
      if (p.mask ? p.mask[(bt * p.T) + j] == 0 : j > t) continue;
    }
    const int64_t r = cache_row(p.table, p.max_pages, p.n_pages, p.page, b, k, p.status);
    if (r < 0) continue;
    const float s = __ldg(p.scale + r);
    float c[2 * TA_MAX_CHUNKS];
#pragma unroll
    for (int i = 0; i < TA_MAX_CHUNKS; ++i) {
      uint32_t v = 0;
      if (i < nq) v = e4m3x2_scaled_bf16x2(*reinterpret_cast<const uint16_t*>(p.kv8 + r * p.dq + i * 64 + lane * 2), s);
      else if (i < nc) v = *reinterpret_cast<const uint32_t*>(p.tail + r * p.dr + (i - nq) * 64 + lane * 2);
      c[2 * i] = bf16lo_f32(v);
      c[2 * i + 1] = bf16hi_f32(v);
    }
#pragma unroll
    for (int h = 0; h < TA_HEADS; ++h) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < TA_MAX_CHUNKS; ++i)
        if (i < nc) x += c[2 * i] * sq[h][i * 64 + lane * 2] + c[2 * i + 1] * sq[h][i * 64 + lane * 2 + 1];
#pragma unroll
      for (int a = 16; a > 0; a >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, a);
      x *= p.scale_log2;
      const float mn = fmaxf(m[h], x);
      const float mu = mn == -INFINITY ? 0.f : mn;  // a NaN score stays one
      const float f = exp2f(m[h] - mu), e = exp2f(x - mu);
      m[h] = mn;
      l[h] = l[h] * f + e;
#pragma unroll
      for (int i = 0; i < 2 * (TA_MAX_CHUNKS - 1); ++i) o[h][i] = o[h][i] * f + e * c[i];
    }
  }
  // the warps' parts meet
  if (lane == 0)
    for (int h = 0; h < TA_HEADS; ++h) {
      sm[warp][h] = m[h];
      sl[warp][h] = l[h];
    }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < TA_HEADS; ++h) {
    float* acc = sq[h];  // the queries have been read
    const bool sunk = p.sink && h0 + h < p.H;
    const float snk = sunk ? __ldg(p.sink + h0 + h) * 1.4426950408889634f : -INFINITY;
    float M = snk;
    for (int w = 0; w < TA_WARPS; ++w) M = fmaxf(M, sm[w][h]);
    if (M == -INFINITY) M = 0.f;
    float den = exp2f(snk - M);
    for (int w = 0; w < TA_WARPS; ++w) den += sl[w][h] * exp2f(sm[w][h] - M);
    const float f = exp2f(m[h] - M);
    for (int w = 0; w < TA_WARPS; ++w) {
      if (w == warp)
#pragma unroll
        for (int i = 0; i < TA_MAX_CHUNKS - 1; ++i)
          if (i < nv)
            for (int z = 0; z < 2; ++z) {
              const float add = o[h][2 * i + z] * f;
              float* at = acc + i * 64 + lane * 2 + z;
              *at = w == 0 ? add : *at + add;
            }
      __syncthreads();
    }
    if (h0 + h < p.H)
      for (int c = threadIdx.x; c < p.dv; c += blockDim.x)
        p.out[(bt * p.H + h0 + h) * p.dv + c] =
            __bfloat16_as_ushort(__float2bfloat16_rn(den > 0.f || den != den ? acc[c] / den : 0.f));
  }
}

}  // namespace ks
