// The quantised latent cache: rows quantised as they are written, and read back.
//
// A cached row holds D = dq + dr columns: dq in e4m3 with one power-of-two scale
// (the row scale of quant_fp8.cuh), dr (the rotary part) in bf16.  Rows live in
// pages: slot s is row s % page of page s / page, and a sequence's position i is
// row i % page of page table[i / page].
//
//   amax = max(max_i |x_i|, 1e-4), scale = the smallest power of two >= amax / 448
//   (at most 2^119)
//   c_i  = e4m3(x_i / scale), nearest even, saturating;      read: bf16(c_i * scale) -- exact,
//   4 significant bits times a power of two fit bf16's 8.
//
// A row that holds a NaN or an infinity (in either part) is marked by scale = NaN and
// zero codes, so one test per row tells every reader and no code is ever e4m3's NaN.  It
// reads back as NaN in every column.
//
// Both kernels move bytes and are bound by memory (launch latency for a few rows): LANES
// threads share a row, and each loads all its pieces before it works on the first.  The
// bf16 side goes in 32-byte accesses, a whole sector, where rows are aligned to that.
// Measured (device time, one B200): 65536 rows of 576 columns written in 23.6 us (118 MB:
// 5.0 TB/s, 0.77 of a copy's rate; 32.8 us with one 16-byte piece at a time), 4 x 16379 rows
// read back in 19.5 us (116 MB: 6.0 TB/s, 0.92); 8 rows in 2.4 us, which is a launch.
#pragma once
#include <cuda_fp16.h>

#include "quant_fp8.cuh"

namespace ks {

constexpr int LC_THREADS = 256;
constexpr int LC_MAX_DQ = 1024;

struct CacheWriteParams {
  const uint16_t* kv;   // bf16 rows, kv_stride elements apart
  int64_t kv_stride;
  const void* slots;    // int32 or int64 [R]; negative: the row is not stored
  int32_t slots_i64;
  int64_t R, n_slots;
  uint8_t* kv8;         // [n_slots, dq]
  float* scale;         // [n_slots]
  uint16_t* tail;       // [n_slots, dr]
  int32_t dq, dr;
  int32_t wide;         // rows of kv start on 32-byte boundaries
  int* status;
};

// 32 bytes (a whole sector), zeros where not `pred`; `wide`: 32-byte aligned.
__device__ __forceinline__ void ld32_or_zero(uint32_t (&v)[8], const void* ptr, bool pred, bool wide) {
  if (wide) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %9, 0;"
        " mov.b32 %0, 0; mov.b32 %1, 0; mov.b32 %2, 0; mov.b32 %3, 0;"
        " mov.b32 %4, 0; mov.b32 %5, 0; mov.b32 %6, 0; mov.b32 %7, 0;"
        " @p ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8]; }"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
        : "l"(ptr), "r"((int)pred));
  } else {
    const uint4 a = ldcg_or_zero(ptr, pred), b = ldcg_or_zero(static_cast<const uint8_t*>(ptr) + 16, pred);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}
__device__ __forceinline__ void st32(void* ptr, const uint32_t (&v)[8], bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(ptr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    static_cast<uint4*>(ptr)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    static_cast<uint4*>(ptr)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// Exponent field all ones in either half (a NaN or an infinity).
__device__ __forceinline__ bool bf16x2_nonfinite(uint32_t v) {
  return (v & 0x7F800000u) == 0x7F800000u || (v & 0x00007F80u) == 0x00007F80u;
}

// LANES threads per row; NV = the most 16-column pieces of the e4m3 part that one of them
// holds in registers between the maximum and the conversion (one pass over kv).
template <int LANES, int NV>
__global__ void __launch_bounds__(LC_THREADS) cache_write_kernel(CacheWriteParams p) {
  const int64_t row = ((int64_t)blockIdx.x * LC_THREADS + threadIdx.x) / LANES;
  const int lane = threadIdx.x % LANES;
  const bool live = row < p.R, wide = p.wide;
  const int nt = p.dr >> 3;
  const uint16_t* x = p.kv + (live ? row : 0) * p.kv_stride;
  uint32_t v[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    ld32_or_zero(v[i], x + (lane + i * LANES) * 16, live && (lane + i * LANES) * 16 < p.dq, wide);
  // the first LANES pieces of the tail stay in registers too; more are copied below
  const uint4 t = ldcg_or_zero(x + p.dq + lane * 8, live && lane < nt);
  int64_t slot = -1;
  if (live) {
    slot = p.slots_i64 ? static_cast<const int64_t*>(p.slots)[row]
                       : (int64_t)static_cast<const int32_t*>(p.slots)[row];
    if (slot >= p.n_slots) {
      if (lane == 0) report_bounds(p.status, (int)row, (int)min(p.n_slots, (int64_t)0x7FFFFFFF));
      slot = -1;
    }
  }
  float amax = 0.f;
  bool bad = bf16x2_nonfinite(t.x) || bf16x2_nonfinite(t.y) || bf16x2_nonfinite(t.z) || bf16x2_nonfinite(t.w);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bad |= bf16x2_nonfinite(v[i][j]);
      amax = fmaxf(amax, fmaxf(fabsf(bf16lo_f32(v[i][j])), fabsf(bf16hi_f32(v[i][j]))));
    }
  for (int j = lane + LANES; live && j < nt; j += LANES) {
    const uint4 e = *reinterpret_cast<const uint4*>(x + p.dq + j * 8);
    bad |= bf16x2_nonfinite(e.x) || bf16x2_nonfinite(e.y) || bf16x2_nonfinite(e.z) || bf16x2_nonfinite(e.w);
  }
  if (bad) amax = INFINITY;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
  if (slot < 0) return;
  bad = amax == INFINITY;
  // smallest power of two >= amax / 448 (a positive normal number)
  const float f = __fdiv_rn(fmaxf(bad ? 0.f : amax, 1e-4f), 448.f);
  const uint32_t fb = __float_as_uint(f);
  // (at most 2^119: 448 * 2^119 is finite, so no finite row reads back as an infinity)
  const float s = fminf((fb & 0x007FFFFFu) ? __uint_as_float((fb & 0x7F800000u) + 0x00800000u) : f,
                        __uint_as_float((119u + 127u) << 23));
  const float inv = bad ? 0.f : __frcp_rn(s);  // exact: s is a power of two
  uint8_t* c8 = p.kv8 + slot * p.dq;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + i * LANES) * 16;
    if (c >= p.dq) break;
    uint32_t h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      h[k] = bad ? 0u : cvt_e4m3x2(bf16lo_f32(v[i][k]) * inv, bf16hi_f32(v[i][k]) * inv);
    *reinterpret_cast<uint4*>(c8 + c) =
        make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
  }
  uint16_t* ct = p.tail + slot * p.dr;
  if (lane < nt) *reinterpret_cast<uint4*>(ct + lane * 8) = t;
  for (int j = lane + LANES; j < nt; j += LANES)
    *reinterpret_cast<uint4*>(ct + j * 8) = *reinterpret_cast<const uint4*>(x + p.dq + j * 8);
  if (lane == 0) p.scale[slot] = bad ? __uint_as_float(0x7FC00000u) : s;
}

struct CacheReadParams {
  const uint8_t* kv8;
  const float* scale;
  const uint16_t* tail;
  int64_t n_pages;
  int32_t page, dq, dr;
  const int32_t* table;  // [B, max_pages]
  int64_t max_pages;
  const int32_t* lens;   // [B]
  int32_t n, start;      // start + n < 2^31
  uint16_t* out;         // [B, n, dq + dr]
  int32_t wide;          // rows of out start on 32-byte boundaries
  int* status;
};

// Row of position `pos` in sequence b, or -1 (reported) when the table cannot name it.
__device__ __forceinline__ int64_t cache_row(const int32_t* table, int64_t max_pages, int64_t n_pages,
                                             int32_t page, int64_t b, int32_t pos, int* status) {
  const int32_t pi = pos / page;
  if (pi >= max_pages) {
    report_bounds(status, (int)b, (int)max_pages);
    return -1;
  }
  const int32_t pg = __ldg(table + b * max_pages + pi);
  if (pg < 0 || pg >= n_pages) {
    report_bounds(status, (int)b, (int)n_pages);
    return -1;
  }
  return (int64_t)pg * page + (pos - pi * page);
}

// Two e4m3 codes to bf16 with the row's scale (exact).
__device__ __forceinline__ uint32_t e4m3x2_scaled_bf16x2(uint16_t c, float s) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return cvt_bf16x2(f.x * s, f.y * s);
}

// One sequence per blockIdx.y, LANES threads per row; a thread first loads all its pieces of
// the row (at most NV of 16 codes and NT of 8 bf16 columns), then converts and stores.
template <int LANES, int NV, int NT>
__global__ void __launch_bounds__(LC_THREADS) cache_read_kernel(CacheReadParams p) {
  const int32_t i = (int32_t)(blockIdx.x * (LC_THREADS / LANES) + threadIdx.x / LANES);
  const int lane = threadIdx.x % LANES;
  if (i >= p.n) return;
  const int64_t b = blockIdx.y, row = b * p.n + i;
  const int32_t pos = p.start + i;
  int64_t src = -1;
  if (pos < __ldg(p.lens + b))
    src = cache_row(p.table, p.max_pages, p.n_pages, p.page, b, pos, p.status);
  const bool ok = src >= 0;
  if (!ok) src = 0;
  const uint8_t* c8 = p.kv8 + src * p.dq + lane * 16;
  const uint16_t* ct = p.tail + src * p.dr + lane * 8;
  uint4 v[NV], t[NT];
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = ldcg_or_zero(c8 + k * LANES * 16, ok && (lane + k * LANES) * 16 < p.dq);
#pragma unroll
  for (int k = 0; k < NT; ++k) t[k] = ldcg_or_zero(ct + k * LANES * 8, ok && (lane + k * LANES) * 8 < p.dr);
  const float s = ok ? __ldg(p.scale + src) : 0.f;
  // (zero codes times NaN are NaN; the tail of a marked row is what was written)
  const bool marked = s != s;
  uint16_t* o = p.out + row * (p.dq + p.dr);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (lane + k * LANES) * 16;
    if (c >= p.dq) break;
    const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
    uint32_t h[8];
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      h[2 * z] = e4m3x2_scaled_bf16x2((uint16_t)w[z], s);
      h[2 * z + 1] = e4m3x2_scaled_bf16x2((uint16_t)(w[z] >> 16), s);
    }
    st32(o + c, h, p.wide);
  }
  const uint4 nan = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    const int c = (lane + k * LANES) * 8;
    if (c < p.dr) *reinterpret_cast<uint4*>(o + p.dq + c) = marked ? nan : t[k];
  }
  // a tail wider than that
  for (int c = (lane + NT * LANES) * 8; c < p.dr; c += LANES * 8)
    *reinterpret_cast<uint4*>(o + p.dq + c) = marked ? nan : ldcg_or_zero(p.tail + src * p.dr + c, ok);
}

}  // namespace ks
