// Log probabilities of given tokens, the entropy of their distributions and the likeliest
// alternatives, from logits.
//
//   m = max_i x_i, S = sum_i e^(x_i - m)
//   logp    = x_token - m - ln S
//   entropy = ln S + sum_i e^(x_i - m) (m - x_i) / S      (no term is negative: nothing cancels)
//   top     = the k largest x_i (k <= 32), the lowest index first among equal ones
//
// One pass over the logits: every thread of a CTA (of a cluster, where there are few rows) goes
// through its 16-byte pieces of the row, 64 values (bf16; 32 in fp32) at a time, with a maximum
// and sums of its own, raised batch by batch; nothing meets but at the end.  It leaves the
// maximum of each of its batches in shared memory.
// The largest k: the cluster's threads form 64 groups with a maximum each, and the k-th largest
// of these bounds the row's k-th largest value from below, so few values reach it (24 of 20 for
// shuffled logits); only batches whose maximum does are read again.  Every CTA hands its values
// to the first one, which ranks them by counting.  Values equal to the bound are kept apart:
// where there are many (masked or constant logits) the first CTA looks for the lowest of them
// from the row's beginning on and stops when it has enough.  A row with a NaN, or with more than
// LP_LIST larger ones (sorted logits, one stretch of some 600 allowed tokens), is searched k times for
// the next largest key by one CTA: 8 such rows of 129280 bf16 values 0.81 ms with 20 alternatives
// (shuffled 12 us), 2048 rows 6.6 ms (0.11).  Keys order values as floats with -0 = 0 and NaN above
// all, then by index.
// Sums are in fp32 relative to the thread's maximum, merged by the usual rescaling.
//
// Bound by reading the logits; per value about 5 instructions, one of them an exponential (16 a
// cycle and SM).  Measured (one B200): 2048 rows of 129280 bf16 values with 20 alternatives 113
// to 118 us (530 MB: 4.5 TB/s, 0.69 of a copy's rate), without 100; 4096 rows of 32003 fp32 values
// 88 to 91 us (5.9 TB/s); 8 rows of 129280 values with 5 alternatives 9 us on the device.  Forms that held
// a slice of the row per CTA in registers and met in barriers before and after the search took 342
// us (a bound per slice, so k values of each to rank) and 406 us (a bound per row) with 20
// alternatives; each thread reading its own batches again, 164 us.
#pragma once
#include "ks_device.cuh"

namespace ks {

constexpr int LP_THREADS = 256;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_PIECES = 8;     // 16-byte pieces a thread holds
constexpr int LP_MAX_TOP = 32;
constexpr int LP_GROUPS = 64;    // of four threads, with a maximum each (>= LP_MAX_TOP)
constexpr int LP_LIST = 512;     // collected values above the bound, and equal to it
constexpr int LP_MAX_CLUSTER = 8;
constexpr int LP_HITS = 256;
constexpr int LP_MAXIMA = 16;    // per thread, of one or more batches each

struct LogprobsParams {
  const void* x;        // [N, V], ld elements apart
  int64_t ld;
  const void* tokens;   // int32 / int64 [N]; negative: none
  int32_t tok_i64;
  int64_t N;
  int32_t V, top;
  int32_t per;          // values of a CTA's slice
  int32_t together;     // batches that share a maximum
  float* logp;          // [N]
  float* entropy;       // [N]
  float* top_logp;      // [N, top]
  void* top_ids;        // [N, top], type of tokens
  int* status;
};

struct LpShared {
  float wm[LP_WARPS], ws[LP_WARPS], wt[LP_WARPS];
  float group[LP_GROUPS];                 // of the cluster
  float bound;
  volatile int full[2];                   // a list has no room: no more is counted
  uint64_t best;                          // of a round
  uint64_t warp_best[LP_WARPS];
  int warp_count[LP_WARPS];
  // of the cluster's first CTA, written by the others
  int above, equal, nan;                  // values collected; a NaN was met
  float cm[LP_MAX_CLUSTER], cs[LP_MAX_CLUSTER], ct[LP_MAX_CLUSTER];
  uint64_t list[2 * LP_LIST];             // above the bound, equal to it
  float maxima[LP_MAXIMA][LP_THREADS];
  int n_hits;
  int2 hits[LP_HITS];                     // (thread, batch) with a value that reaches the bound
  uint64_t top[LP_MAX_TOP];
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

__device__ __forceinline__ uint32_t lp_max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
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
  __device__ __forceinline__ uint32_t max2() const {  // of the even and of the odd values
    return lp_max_bf16x2(lp_max_bf16x2(w.x, w.y), lp_max_bf16x2(w.z, w.w));
  }
  // the largest value, NaN passed over (-inf where all are)
  __device__ __forceinline__ float max() const {
    if constexpr (BF16) {
      const uint32_t a = max2();
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

// Address of this CTA's shared object in CTA `cta` of the cluster.
__device__ __forceinline__ uint32_t lp_remote(const void* p, uint32_t cta) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(cta));
  return r;
}
__device__ __forceinline__ void lp_put(float* p, uint32_t cta, float x) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(lp_remote(p, cta)), "f"(x) : "memory");
}
__device__ __forceinline__ int lp_count(int* p) {  // of the first CTA
  int n;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(n) : "r"(lp_remote(p, 0)) : "memory");
  return n;
}

// A value that reaches the bound, to the first CTA's list.
__device__ __noinline__ void lp_hand_over(LpShared& sh, float x, int e, int tie) {
  if (sh.full[tie]) return;
  const int n = lp_count(tie ? &sh.equal : &sh.above);
  if (n < LP_LIST)
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(lp_remote(&sh.list[tie * LP_LIST + n], 0)), "l"(lp_key(x, e))
                 : "memory");
  else
    sh.full[tie] = 1;
}

// The k-th largest (k from 0) of 64 values, two per lane: a bitonic sort in one warp.
__device__ __forceinline__ float lp_kth(float a, float b, int k, int lane) {
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      if (stride == 32) {  // descending: a has the lower places
        const float hi = fmaxf(a, b), lo = fminf(a, b);
        a = hi;
        b = lo;
      } else {
        const float oa = __shfl_xor_sync(0xFFFFFFFFu, a, stride), ob = __shfl_xor_sync(0xFFFFFFFFu, b, stride);
        const bool low = (lane & stride) == 0;
        const bool da = (lane & size) == 0, db = ((lane + 32) & size) == 0;  // descending there
        a = low == da ? fmaxf(a, oa) : fminf(a, oa);
        b = low == db ? fmaxf(b, ob) : fminf(b, ob);
      }
    }
  const float x = __shfl_sync(0xFFFFFFFFu, a, k & 31), y = __shfl_sync(0xFFFFFFFFu, b, k & 31);
  return k < 32 ? x : y;
}

// Ranks n keys (all different) by counting; the first `keep` of them in order to top.
__device__ __forceinline__ void lp_rank(const uint64_t* keys, int n, int keep, uint64_t* top) {
  for (int i = threadIdx.x; i < n; i += LP_THREADS) {
    const uint64_t key = keys[i];
    int above = 0;
    for (int j = 0; j < n && above < keep; ++j) above += keys[j] > key;
    if (above < keep) top[above] = key;
  }
}

template <bool BF16>
__global__ void __launch_bounds__(LP_THREADS, 4) token_logprobs_kernel(LogprobsParams p) {
  using P = LpPiece<BF16>;
  constexpr int E = P::E, BATCH = LP_THREADS * LP_PIECES * E;
  constexpr float C = 1.4426950408889634f;
  __shared__ LpShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t cta, size;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int64_t row = blockIdx.x / size;
  const uint8_t* base = static_cast<const uint8_t*>(p.x) + row * p.ld * (BF16 ? 2 : 4);
  // pieces start on 16-byte boundaries: piece j holds values E j - shift ..
  const int shift = (int)((reinterpret_cast<uintptr_t>(base) & 15) / (BF16 ? 2 : 4));
  const int k = p.top;
  if (tid == 0) sh.above = sh.equal = sh.nan = sh.full[0] = sh.full[1] = sh.n_hits = 0;
  // (waited for below: a CTA's shared memory is written to only when it has begun)
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

  // the given token's logit, long before it is needed
  int64_t token = -1;
  float xt = 0.f;
  if (cta == 0 && tid == 0) {
    token = p.tok_i64 ? static_cast<const int64_t*>(p.tokens)[row]
                      : (int64_t)static_cast<const int32_t*>(p.tokens)[row];
    if (token >= p.V) report_bounds(p.status, (int)min(row, (int64_t)0x7FFFFFFF), p.V);
    else if (token >= 0) xt = lp_load<BF16>(base, token);
  }

  const int at = (int)min((int64_t)cta * p.per, (int64_t)p.V), stop = (int)min((int64_t)at + p.per, (int64_t)p.V);
  const int start = (at + shift) / E * E - shift;  // of the first piece
  const int batches = stop > at ? (stop - start + BATCH - 1) / BATCH : 0;
  const auto first = [&](int b, int i) { return start + b * BATCH + (i * LP_THREADS + tid) * E; };
  const auto piece = [&](int e) { return reinterpret_cast<const uint4*>(base + (int64_t)e * (BF16 ? 2 : 4)); };
  // a piece that the slice may cut; values beyond it read as -inf
  const auto guarded = [&](int e) {
    constexpr uint32_t none = BF16 ? 0xFF80FF80u : 0xFF800000u;
    if (e >= at && e + E <= stop) return __ldg(piece(e));
    if (e < stop && e + E > at) return lp_cut<BF16>(base, e, at, stop);
    return make_uint4(none, none, none, none);
  };

  float M = -INFINITY, S = 0.f, Tt = 0.f;  // of the thread
  float held = -INFINITY;                  // maximum of the batches that share one
  for (int b = 0; b < batches; ++b) {
    P v[LP_PIECES];
    if (start + b * BATCH >= at && start + (b + 1) * BATCH <= stop) {
#pragma unroll
      for (int i = 0; i < LP_PIECES; ++i) v[i].w = __ldcs(piece(first(b, i)));
    } else {
#pragma unroll
      for (int i = 0; i < LP_PIECES; ++i) v[i].w = guarded(first(b, i));
    }
    float m;
    if constexpr (BF16) {
      uint32_t a = v[0].max2();
#pragma unroll
      for (int i = 1; i < LP_PIECES; ++i) a = lp_max_bf16x2(a, v[i].max2());
      m = fmaxf(fmaxf(bf16lo_f32(a), bf16hi_f32(a)), -INFINITY);
    } else {
      m = -INFINITY;
#pragma unroll
      for (int i = 0; i < LP_PIECES; ++i) m = fmaxf(m, v[i].max());
    }
    if (k) {
      held = fmaxf(held, m);
      if ((b + 1) % p.together == 0 || b + 1 == batches) {
        sh.maxima[b / p.together][tid] = held;
        held = -INFINITY;
      }
    }
    m = fmaxf(m, M);
    // y = (x - m) log2 e as one rounding of x c - h, h = m c rounded; what h is off by is common to
    // the batch's values and put right in its sums
    const float h = m * C, err = fmaf(m, C, -h);
    float2 s2 = make_float2(0.f, 0.f), t2 = s2;
    // (at most 0.1 below 10^6; larger maxima, of masked stretches say, go the plain way)
    const bool near = fabsf(m) < 1e6f;
    if (near) {
      const float2 minus = make_float2(-h, -h), log2e = make_float2(C, C);
      const auto add = [&](float a, float c) {
        const float2 y = fma2(make_float2(a, c), log2e, minus);
        const float2 e = make_float2(ex2f(y.x), ex2f(y.y));
        s2 = add2(s2, e);
        t2 = fma2(e, y, t2);
      };
      // (values below -1e37, -inf among them, count as that: e = 0 and e y = 0; NaN stays)
#pragma unroll
      for (int i = 0; i < LP_PIECES; ++i) {
        if constexpr (BF16) {
          const uint32_t u[4] = {v[i].w.x, v[i].w.y, v[i].w.z, v[i].w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t c = lp_max_nan_bf16x2(u[j], 0xFCF1FCF1u);
            add(bf16lo_f32(c), bf16hi_f32(c));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; j += 2) add(max_nan(v[i].at(j), -1e37f), max_nan(v[i].at(j + 1), -1e37f));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < LP_PIECES; ++i)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float x = v[i].at(j);
          // nothing but -inf: 0, and NaN where it is one
          const float y = m == -INFINITY ? x - x : max_nan((x - m) * C, -200.f);
          const float z = m == -INFINITY ? (x != x ? x : 0.f) : ex2f(y);
          s2.x += z;
          if (m > -INFINITY) t2.x = fmaf(z, y, t2.x);
        }
    }
    float s = s2.x + s2.y, t = t2.x + t2.y;
    if (near) {
      const float f = ex2f(-err);
      t = f * (t - err * s);
      s *= f;
    }
    // raise what is there to the new maximum
    const float d = M == m ? 0.f : (M - m) * C, f = ex2f(d);
    Tt = (f > 0.f ? f * (Tt + S * d) : 0.f) + t;
    S = S * f + s;
    M = m;
  }
  const bool bad = S != S;
  // -------------------------------------------------------------- the warp's, the CTA's, the row's
  float wm = M, gm = M;
  const int lanes = 4 * (int)size;  // of a group: 64 groups in the cluster
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    wm = fmaxf(wm, __shfl_xor_sync(0xFFFFFFFFu, wm, o));
    if (2 * o == lanes) gm = wm;
  }
  const bool nan = __any_sync(0xFFFFFFFFu, bad);
  {
    const float d = M == wm ? 0.f : (M - wm) * C, f = ex2f(d);
    Tt = f > 0.f ? f * (Tt + S * d) : 0.f;
    S *= f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      S += __shfl_xor_sync(0xFFFFFFFFu, S, o);
      Tt += __shfl_xor_sync(0xFFFFFFFFu, Tt, o);
    }
    if (nan) S = __uint_as_float(0x7FC00000u);
  }
  if (lane == 0) {
    sh.wm[warp] = wm;
    sh.ws[warp] = S;
    sh.wt[warp] = Tt;
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (k) {
    // every group's maximum to every CTA
    if ((lane & (lanes - 1)) == 0)
      for (uint32_t c = 0; c < size; ++c) lp_put(&sh.group[(cta * LP_THREADS + tid) / lanes], c, gm);
    if (nan && lane == 0) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(lp_remote(&sh.nan, 0)), "r"(1) : "memory");
    if (size > 1) cluster_sync();
  }
  __syncthreads();
  if (warp == 0 && k) {
    const float kth = lp_kth(sh.group[lane], sh.group[lane + 32], k - 1, lane);
    if (lane == 0) sh.bound = kth;
  }
  if (warp == 1) {
    M = lane < LP_WARPS ? sh.wm[lane] : -INFINITY;
    S = lane < LP_WARPS ? sh.ws[lane] : 0.f;
    Tt = lane < LP_WARPS ? sh.wt[lane] : 0.f;
    const bool any_bad = __any_sync(0xFFFFFFFFu, S != S);
#pragma unroll
    for (int o = LP_WARPS / 2; o > 0; o >>= 1)
      lp_merge(M, S, Tt, __shfl_xor_sync(0xFFFFFFFFu, M, o), __shfl_xor_sync(0xFFFFFFFFu, S, o),
               __shfl_xor_sync(0xFFFFFFFFu, Tt, o));
    if (any_bad) S = __uint_as_float(0x7FC00000u);
    if (lane == 0) {
      lp_put(&sh.cm[cta], 0, M);
      lp_put(&sh.cs[cta], 0, S);
      lp_put(&sh.ct[cta], 0, Tt);
    }
  }
  if (k) {
    __syncthreads();
    const float bound = sh.bound;
    // which batches to read again ..
    if (gm >= bound)
      for (int j = 0; j * p.together < batches; ++j)
        if (sh.maxima[j][tid] >= bound)
          for (int b = j * p.together; b < min((j + 1) * p.together, batches); ++b) {
            const int n = atomicAdd(&sh.n_hits, 1);
            if (n < LP_HITS) sh.hits[n] = make_int2(tid, b);
          }
    __syncthreads();
    const int n_hits = sh.n_hits;
    const auto scan = [&](const uint4& w, int e0) {
      P v;
      v.w = w;
      if (!(v.max() >= bound)) return;
#pragma unroll
      for (int q = 0; q < E; ++q) {
        const float x = v.at(q);
        if (x >= bound && e0 + q >= at && e0 + q < stop) lp_hand_over(sh, x, e0 + q, x == bound);
      }
    };
    if (n_hits <= LP_HITS) {
      // .. shared out: eight threads a batch, a piece each
      static_assert(LP_PIECES == 8, "eight threads");
      for (int i = tid >> 3; i < n_hits; i += LP_THREADS / 8) {
        const int e0 = start + sh.hits[i].y * BATCH + ((tid & 7) * LP_THREADS + sh.hits[i].x) * E;
        scan(guarded(e0), e0);
      }
    } else if (gm >= bound) {
      for (int b = 0; b < batches; ++b)
        if (sh.maxima[b / p.together][tid] >= bound && !(sh.full[0] && sh.full[1]))
#pragma unroll 1
          for (int i = 0; i < LP_PIECES; ++i) scan(guarded(first(b, i)), first(b, i));
    }
  }
  if (size > 1) {
    cluster_sync();
    if (cta) return;
  } else {
    __syncthreads();
  }
  // -------------------------------------------------------------- the first CTA
  if (tid == 0) {
    M = sh.cm[0]; S = sh.cs[0]; Tt = sh.ct[0];
    bool none = S != S;
    for (uint32_t i = 1; i < size; ++i) {
      none |= sh.cs[i] != sh.cs[i];
      lp_merge(M, S, Tt, sh.cm[i], sh.cs[i], sh.ct[i]);
    }
    // without a finite maximum nothing is defined
    const bool fine = !none && fabsf(M) < INFINITY;
    const float undefined = __uint_as_float(0x7FC00000u), ln = logf(S);
    sh.wm[0] = M;
    sh.ws[0] = fine ? ln : undefined;
    p.logp[row] = token < 0 ? 0.f : token >= p.V || !fine ? undefined : (xt - M) - ln;
    p.entropy[row] = fine ? fmaxf(ln - 0.6931471805599453f * (Tt / S), 0.f) : undefined;
  }
  if (k == 0) return;
  const int above = sh.above, equal = sh.equal;
  int n = 0;
  if (sh.nan || above > LP_LIST) {
    // the next largest key, k times
    uint64_t below = ~0ull;
    for (; n < k; ++n) {
      uint64_t best = 0;
      for (int64_t e = tid; e < p.V; e += LP_THREADS) {
        const uint64_t key = lp_key(lp_load<BF16>(base, e), (int)e);
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
        sh.list[n] = b;
      }
      __syncthreads();
      below = sh.best;
    }
  } else {
    // the list is made one stretch: those above the bound, then those equal to it
    n = above;
    uint64_t key = 0, key2 = 0;
    if (equal <= LP_LIST) {
      if (tid < equal) key = sh.list[LP_LIST + tid];
      if (tid + LP_THREADS < equal) key2 = sh.list[LP_LIST + tid + LP_THREADS];
      __syncthreads();
      if (key) sh.list[n + tid] = key;
      if (key2) sh.list[n + tid + LP_THREADS] = key2;
      n += equal;
    } else {
      // the lowest of those equal to the bound, in the order of their places
      const float bound = sh.bound;
      const int want = max(k - above, 0);
      int found = 0;
      for (int64_t e0 = 0; e0 < p.V && found < want; e0 += LP_THREADS) {
        const int64_t e = e0 + tid;
        const bool hit = e < p.V && lp_load<BF16>(base, e) == bound;
        const uint32_t hits = __ballot_sync(0xFFFFFFFFu, hit);
        __syncthreads();
        if (lane == 0) sh.warp_count[warp] = __popc(hits);
        __syncthreads();
        int place = found + __popc(hits & ((1u << lane) - 1u)), all = 0;
        for (int w = 0; w < LP_WARPS; ++w) {
          if (w < warp) place += sh.warp_count[w];
          all += sh.warp_count[w];
        }
        if (hit && place < want) sh.list[n + place] = lp_key(bound, (int)e);
        found = min(found + all, want);
      }
      n += found;
    }
  }
  static_assert(LP_LIST <= 2 * LP_THREADS, "two keys a thread are moved");
  __syncthreads();
  lp_rank(sh.list, n, k, sh.top);
  __syncthreads();
  if (tid < k) {
    const uint64_t key = sh.top[tid];
    p.top_logp[row * k + tid] = (lp_value(key) - sh.wm[0]) - sh.ws[0];
    if (p.tok_i64) static_cast<int64_t*>(p.top_ids)[row * k + tid] = lp_index(key);
    else static_cast<int32_t*>(p.top_ids)[row * k + tid] = lp_index(key);
  }
}

}  // namespace ks
