// Log probabilities of given tokens, the entropy of their distributions and the likeliest
// alternatives, from logits.
//
//   m = max_i x_i, S = sum_i e^(x_i - m)
//   logp    = x_token - m - ln S
//   entropy = ln S + sum_i e^(x_i - m) (m - x_i) / S      (no term is negative: nothing cancels)
//   top     = the k largest x_i (k <= 32), the lowest index first among equal ones
//
// One pass over the logits.  A cluster of CTAs takes a row, each CTA a slice of it that stays
// in registers (64 values in bf16, 32 in fp32 per thread; longer slices go in passes): maximum,
// sums and the search for the largest all work on the registers, so a logit is read once.
// The largest k of a slice: the 64 groups of 8 threads have a maximum each, and the k-th
// largest of these bounds the k-th largest value from below, so only the few values that reach
// it are collected (about k for shuffled logits) and ranked by counting.  Where more than
// LP_LIST reach it (many equal values, NaN), k rounds look for the next largest key instead:
// exact for any input.  Keys order values as floats with -0 = 0 and NaN (positive) above all,
// then by index.
// Sums are in fp32 relative to the warp's maximum, merged by the usual rescaling.
//
// Bound by reading the logits; per value about 8 instructions and one exponential.
#pragma once
#include "ks_device.cuh"

namespace ks {

constexpr int LP_THREADS = 512;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_PIECES = 8;     // 16-byte pieces a thread holds
constexpr int LP_MAX_TOP = 32;
constexpr int LP_GROUPS = 64;    // of threads, with a maximum each (>= LP_MAX_TOP)
constexpr int LP_LIST = 1024;    // collected values
constexpr int LP_MAX_CLUSTER = 8;

struct LogprobsParams {
  const void* x;        // [N, V], ld elements apart
  int64_t ld;
  const void* tokens;   // int32 / int64 [N]; negative: none
  int32_t tok_i64;
  int64_t N;
  int32_t V, top;
  int32_t per;          // values of a CTA's slice
  float* logp;          // [N]
  float* entropy;       // [N]
  float* top_logp;      // [N, top]
  void* top_ids;        // [N, top], type of tokens
  int* status;
};

struct LpShared {
  float wm[LP_WARPS], ws[LP_WARPS], wt[LP_WARPS];
  float group[LP_GROUPS];
  float bound;
  int count;
  uint64_t best;                          // of a round
  uint64_t warp_best[LP_WARPS];
  uint64_t list[LP_LIST + LP_MAX_TOP];    // candidates; the first ones are the pass before's
  uint64_t top[LP_MAX_TOP];
  // of the cluster's first CTA, written by the others
  float cm[LP_MAX_CLUSTER], cs[LP_MAX_CLUSTER], ct[LP_MAX_CLUSTER];
  uint64_t ctop[LP_MAX_CLUSTER * LP_MAX_TOP];
};

// Value and index as one number that orders by value, the lower index first; 0: nothing.
__device__ __forceinline__ uint64_t lp_key(float x, int i) {
  uint32_t u = __float_as_uint(x);
  if (u == 0x80000000u) u = 0;
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) u = 0x7FFFFFFFu;
  const uint32_t o = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (uint64_t)o << 32 | (0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ int lp_index(uint64_t key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

// (m, s, t): maximum, sum of e^(x - m), sum of e^(x - m) (x - m) log2 e.
__device__ __forceinline__ void lp_merge(float& m, float& s, float& t, float m2, float s2, float t2) {
  const float M = fmaxf(m, m2);
  if (M == -INFINITY) return;
  const float d1 = (m - M) * 1.4426950408889634f, d2 = (m2 - M) * 1.4426950408889634f;
  const float f1 = exp2f(d1), f2 = exp2f(d2);
  t = (f1 > 0.f ? f1 * (t + s * d1) : 0.f) + (f2 > 0.f ? f2 * (t2 + s2 * d2) : 0.f);
  s = f1 * s + f2 * s2;
  m = M;
}

__device__ __forceinline__ float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 lp_add2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 lp_mul2(float2 a, float2 b) {
  float2 r;
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 lp_fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{ .reg .b64 w, x, y, z; mov.b64 w, {%2, %3}; mov.b64 x, {%4, %5}; mov.b64 y, {%6, %7};"
      " fma.rn.f32x2 z, w, x, y; mov.b64 {%0, %1}, z; }"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
// The larger, a NaN where a is one.
__device__ __forceinline__ float lp_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t lp_max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <bool BF16>
struct LpPiece {
  static constexpr int E = BF16 ? 8 : 4;
  uint4 w;
  __device__ __forceinline__ float at(int i) const {
    const uint32_t u = BF16 ? (i < 2 ? w.x : i < 4 ? w.y : i < 6 ? w.z : w.w)
                            : (i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w);
    if constexpr (BF16) return (i & 1) ? bf16hi_f32(u) : bf16lo_f32(u);
    else return __uint_as_float(u);
  }
  // the largest value, NaN passed over (-inf where all are)
  __device__ __forceinline__ float max() const {
    if constexpr (BF16) {
      const uint32_t a = lp_max_bf16x2(lp_max_bf16x2(w.x, w.y), lp_max_bf16x2(w.z, w.w));
      return fmaxf(fmaxf(bf16lo_f32(a), bf16hi_f32(a)), -INFINITY);
    } else {
      return fmaxf(fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3))), -INFINITY);
    }
  }
};

template <bool BF16>
__device__ __forceinline__ float lp_load(const uint8_t* base, int64_t i) {
  if constexpr (BF16) return __uint_as_float((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(base) + i) << 16);
  else return __ldg(reinterpret_cast<const float*>(base) + i);
}

// The 16 bytes from value `first` on, -inf where it is outside [at, stop).
template <bool BF16>
__device__ __noinline__ uint4 lp_cut(const uint8_t* base, int first, int at, int stop) {
  uint64_t lo = 0, hi = 0;
  constexpr int E = BF16 ? 8 : 4, BITS = BF16 ? 16 : 32;
#pragma unroll 1
  for (int j = E - 1; j >= 0; --j) {
    const int e = first + j;
    uint64_t x = BF16 ? 0xFF80u : 0xFF800000u;
    if (e >= at && e < stop)
      x = BF16 ? (uint64_t)reinterpret_cast<const uint16_t*>(base)[e] : (uint64_t)reinterpret_cast<const uint32_t*>(base)[e];
    hi = hi << BITS | lo >> (64 - BITS);
    lo = lo << BITS | x;
  }
  return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

template <bool BF16>
__global__ void __launch_bounds__(LP_THREADS, 2) token_logprobs_kernel(LogprobsParams p) {
  using P = LpPiece<BF16>;
  constexpr int E = P::E;
  constexpr int PASS = LP_THREADS * LP_PIECES * E;
  __shared__ LpShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t rank, size;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  // (waited for below: a CTA's shared memory is written to only when it has begun)
  if (size > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int64_t row = blockIdx.x / size;
  const int begin = (int)min((int64_t)rank * p.per, (int64_t)p.V), end = (int)min((int64_t)begin + p.per, (int64_t)p.V);
  const uint8_t* base = static_cast<const uint8_t*>(p.x) + row * p.ld * (BF16 ? 2 : 4);
  // pieces start on 16-byte boundaries: piece j holds values E j - shift ..
  const int shift = (int)((reinterpret_cast<uintptr_t>(base) & 15) / (BF16 ? 2 : 4));
  const int k = p.top;

  // the given token's logit, long before it is needed
  int64_t token = -1;
  float xt = 0.f;
  if (rank == 0 && tid == 0) {
    token = p.tok_i64 ? static_cast<const int64_t*>(p.tokens)[row]
                      : (int64_t)static_cast<const int32_t*>(p.tokens)[row];
    if (token >= p.V) report_bounds(p.status, (int)min(row, (int64_t)0x7FFFFFFF), p.V);
    else if (token >= 0)
      xt = lp_load<BF16>(base, token);
  }

  float M = -INFINITY, S = 0.f, Tt = 0.f;  // of the warp, all passes
  int kept = 0;                            // values of the passes before, in sh.top
  for (int at = begin, stop; at < end; at = stop) {
    // ------------------------------------------------------------ load
    P v[LP_PIECES];
    const int j0 = (at + shift) / E;
    const int mine = (j0 + tid) * E - shift;  // index of the thread's first value
    stop = min(j0 * E - shift + PASS, end);
    const auto first = [&](int i) { return mine + i * LP_THREADS * E; };
    const auto whole = [&](int i) { return first(i) >= at && first(i) + E <= stop; };
#pragma unroll
    for (int i = 0; i < LP_PIECES; ++i)
      if (whole(i)) v[i].w = __ldcs(reinterpret_cast<const uint4*>(base + (int64_t)first(i) * (BF16 ? 2 : 4)));
    // pieces that the slice cuts, value by value; values beyond it count as -inf and get no key
#pragma unroll
    for (int i = 0; i < LP_PIECES; ++i)
      if (!whole(i)) v[i].w = lp_cut<BF16>(base, first(i), at, stop);
    // ------------------------------------------------------------ maximum
    float pm[LP_PIECES], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < LP_PIECES; ++i) {
      pm[i] = v[i].max();
      m = fmaxf(m, pm[i]);
    }
    float wm = m, gm = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      wm = fmaxf(wm, __shfl_xor_sync(0xFFFFFFFFu, wm, o));
      if (o == 4) gm = wm;
    }
    if (k && (lane & 7) == 0) sh.group[warp * 4 + (lane >> 3)] = gm;
    if (tid == 0) sh.count = 0;
    // ------------------------------------------------------------ sums
    float2 s2 = make_float2(0.f, 0.f), t2 = s2;
    if (wm > -INFINITY) {
      const float2 minus = make_float2(-wm, -wm), log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
      for (int i = 0; i < LP_PIECES; ++i)
#pragma unroll
        for (int j = 0; j < E; j += 2) {
          // far below the maximum, and at -inf: e = 0 and 0 * y = 0
          float2 y = lp_mul2(lp_add2(make_float2(v[i].at(j), v[i].at(j + 1)), minus), log2e);
          y = make_float2(lp_max_nan(y.x, -200.f), lp_max_nan(y.y, -200.f));
          const float2 e = make_float2(lp_ex2(y.x), lp_ex2(y.y));
          s2 = lp_add2(s2, e);
          t2 = lp_fma2(e, y, t2);
        }
    } else {  // nothing but -inf, or a NaN among it
#pragma unroll
      for (int i = 0; i < LP_PIECES; ++i)
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (v[i].at(j) != v[i].at(j)) s2.x = v[i].at(j);
    }
    float s = s2.x + s2.y, t = t2.x + t2.y;
    // a NaN (or two infinities) anywhere makes the row's sums NaN
    const bool any_nan = __syncthreads_or(s != s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
      t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    }
    lp_merge(M, S, Tt, wm, s, t);
    if (any_nan) S = __uint_as_float(0x7FC00000u);
    // ------------------------------------------------------------ the largest k
    if (k) {
      if (tid < LP_GROUPS) {
        const float g = sh.group[tid];
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < LP_GROUPS; ++i) {
          const float o = sh.group[i];
          above += o > g || (o == g && i < tid);
        }
        if (above == k - 1) sh.bound = g;
      }
      if (tid < kept) sh.list[tid] = sh.top[tid];
      __syncthreads();
      const float bound = sh.bound;
#pragma unroll
      for (int i = 0; i < LP_PIECES; ++i) {
        if (pm[i] >= bound) {
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const float x = v[i].at(j);
            const int e = first(i) + j;
            if (x >= bound && e >= at && e < stop) {
              const int n = atomicAdd(&sh.count, 1);
              if (n < LP_LIST) sh.list[kept + n] = lp_key(x, e);
            }
          }
        }
      }
      __syncthreads();
      int n = sh.count;
      if (n > LP_LIST || any_nan) {
        // too many to rank: the next largest key, k times
        uint64_t below = ~0ull;
        n = 0;
        for (int r = 0; r < min(k, stop - at); ++r) {
          uint64_t best = 0;
          for (int e = at + tid; e < stop; e += LP_THREADS) {
            const uint64_t key = lp_key(lp_load<BF16>(base, e), e);
            if (key < below && key > best) best = key;
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor_sync(0xFFFFFFFFu, best, o);
            best = other > best ? other : best;
          }
          if (lane == 0) sh.warp_best[warp] = best;
          __syncthreads();
          if (tid == 0) {
            uint64_t b = 0;
            for (int w = 0; w < LP_WARPS; ++w) b = sh.warp_best[w] > b ? sh.warp_best[w] : b;
            sh.best = b;
            sh.list[kept + r] = b;
          }
          __syncthreads();
          below = sh.best;
          ++n;
        }
      }
      n += kept;
      for (int i = tid; i < n; i += LP_THREADS) {
        const uint64_t key = sh.list[i];
        int above = 0;
        for (int j = 0; j < n && above < k; ++j) above += sh.list[j] > key;
        if (above < k) sh.top[above] = key;
      }
      kept = min(n, k);
      __syncthreads();
    }
  }
  // -------------------------------------------------------------- the CTA's sums, then the row's
  if (lane == 0) {
    sh.wm[warp] = M;
    sh.ws[warp] = S;
    sh.wt[warp] = Tt;
  }
  __syncthreads();
  if (warp == 0) {
    M = lane < LP_WARPS ? sh.wm[lane] : -INFINITY;
    S = lane < LP_WARPS ? sh.ws[lane] : 0.f;
    Tt = lane < LP_WARPS ? sh.wt[lane] : 0.f;
    const bool bad = __any_sync(0xFFFFFFFFu, S != S);
#pragma unroll
    for (int o = LP_WARPS / 2; o > 0; o >>= 1)
      lp_merge(M, S, Tt, __shfl_xor_sync(0xFFFFFFFFu, M, o), __shfl_xor_sync(0xFFFFFFFFu, S, o),
               __shfl_xor_sync(0xFFFFFFFFu, Tt, o));
    if (bad) S = __uint_as_float(0x7FC00000u);
  }
  if (size > 1) {
    // into the first CTA's shared memory
    const auto remote = [&](const void* a) {
      uint32_t r;
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(a)));
      return r;
    };
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid == 0) {
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(&sh.cm[rank])), "f"(M) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(&sh.cs[rank])), "f"(S) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(&sh.ct[rank])), "f"(Tt) : "memory");
    }
    if (tid < k)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(&sh.ctop[rank * k + tid])),
                   "l"(tid < kept ? sh.top[tid] : 0ull)
                   : "memory");
    cluster_sync();
    if (rank) return;
    if (tid == 0) {
      M = sh.cm[0]; S = sh.cs[0]; Tt = sh.ct[0];
      bool bad = S != S;
      for (uint32_t i = 1; i < size; ++i) {
        bad |= sh.cs[i] != sh.cs[i];
        lp_merge(M, S, Tt, sh.cm[i], sh.cs[i], sh.ct[i]);
      }
      if (bad) S = __uint_as_float(0x7FC00000u);
    }
    if (k) {
      const int n = (int)size * k;
      if (tid < n) {
        const uint64_t key = sh.ctop[tid];
        int above = 0;
        for (int j = 0; j < n && above < k; ++j) above += sh.ctop[j] > key;
        if (key && above < k) sh.top[above] = key;
      }
    }
  }
  if (tid == 0) {
    // without a finite maximum nothing is defined
    const float none = __uint_as_float(0x7FC00000u);
    const bool fine = S == S && fabsf(M) < INFINITY;
    const float ln = logf(S);
    sh.wm[0] = M;
    sh.ws[0] = fine ? ln : none;
    p.logp[row] = token < 0 ? 0.f : token >= p.V || !fine ? none : (xt - M) - ln;
    p.entropy[row] = fine ? fmaxf(ln - 0.6931471805599453f * (Tt / S), 0.f) : none;
  }
  if (k) {
    __syncthreads();
    if (tid < k) {
      const uint64_t key = sh.top[tid];
      p.top_logp[row * k + tid] = (lp_value(key) - sh.wm[0]) - sh.ws[0];
      if (p.tok_i64) static_cast<int64_t*>(p.top_ids)[row * k + tid] = lp_index(key);
      else static_cast<int32_t*>(p.top_ids)[row * k + tid] = lp_index(key);
    }
  }
}

}  // namespace ks
