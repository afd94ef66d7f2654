// Verification of drafted tokens against the target's probabilities, from given
// random numbers.
//
// p [B, T + 1, V]: row 0 is the target's distribution after the last accepted token,
// row i + 1 the one after drafted token i.  u [B, T + 1] in [0, 1) decides at each row,
// noise [B, V] (exponential) samples the next token.
//
//  * Sampled chain (q [B, T, V], the draft's distributions): token i stands if
//    u_i q_i(x_i) < p_i(x_i) and every token before it stands.  n of them stand; the
//    next token is drawn from w = max(p_n - q_n, 0), or from p_T when all stand.
//  * Fixed candidates (parents [B, T], -1 = the root; a tree, or a chain when null):
//    the children of a row split [0, 1) into stretches of length p_row(token), in index
//    order, and u_row falls into one child's (taken, the walk goes on there) or into
//    none (the next token is drawn from p_row without the children's tokens).  A
//    sibling that repeats an older one's token has no stretch.
//
// Drawing: argmax_x w(x) / noise(x), ties to the lowest x.  With exponential noise
// this picks x with probability w(x) / sum w, needs no sum, and does not depend on
// the order of the work: every operation is one correctly rounded fp32 operation per
// entry, and the stretches are summed in fp64 in one order.  If w is zero everywhere, p's
// row takes its place.
//
// One cluster of CTAs per sequence.  Every CTA walks the draft itself (a few dependent
// loads), then takes its slice of the one vocabulary row that matters; the slices'
// maxima meet through distributed shared memory.  Bound by reading that row of p, q and
// the noise (8 or 12 bytes per entry), for few sequences by the chain of load latencies
// (token -> probability -> row).  Divisions are left to the few entries that may
// beat the warp's best so far.
// Measured (device time, one B200): 64 chains over 129280 entries 22.9 us (99 MB: 4.3 TB/s;
// 39.4 us with a division per entry), 16 trees of 40 candidates 13.0 us, of which the walk
// and the launch are most, one chain over 32003 entries 6.9 us.  With the noise prefetched to
// L2 before the walk: 38.1, 19.6 and 7.1 us.
#pragma once
#include "ks_device.cuh"

namespace ks {

constexpr int VD_THREADS = 512;
constexpr int VD_MAX_T = 1024;
constexpr int VD_MAX_CLUSTER = 8;
constexpr int VD_BITS = 1 << 17;  // of the map of children's tokens: with the walk's arrays it fits 48 KB

struct VerifyParams {
  const float* p;       // [B, T + 1, V]
  const float* q;       // [B, T, V] or null
  const void* tokens;   // int32 / int64 [B, T]
  int32_t tok_i64;
  const int32_t* parents;  // [B, T] or null (chain)
  const float* u;       // [B, T + 1]
  const float* noise;   // [B, V]
  void* out;            // [B, T + 1], type of tokens
  int32_t* n_acc;       // [B]
  int32_t* path;        // [B, T]
  int64_t B;
  int32_t T, V;
  int32_t vec4;         // rows and pointers are 16-byte aligned
  int32_t per;          // entries of a slice (a multiple of 32)
  int32_t words;        // of the map of children's tokens: a bit per entry, or VD_BITS shared ones
  int* status;
};

struct VdBest {
  float val;
  int32_t idx;
  int32_t any;  // some w > 0
};

__device__ __forceinline__ void vd_take(VdBest& a, float val, int32_t idx) {
  if (val > a.val || (val == a.val && idx < a.idx)) {
    a.val = val;
    a.idx = idx;
  }
}

__device__ __forceinline__ int64_t vd_token(const VerifyParams& p, int64_t i) {
  return p.tok_i64 ? static_cast<const int64_t*>(p.tokens)[i]
                   : (int64_t)static_cast<const int32_t*>(p.tokens)[i];
}

// WRAP: the slice has more entries than the map has bits (an instance of its own: with the
// choice made inside, 64 chains over 129280 entries take 25.6 instead of 22.9 us).
template <bool WRAP>
__global__ void __launch_bounds__(VD_THREADS) verify_draft_kernel(VerifyParams p) {
  extern __shared__ __align__(16) uint8_t vd_smem[];
  // px [T] double, ux, tok, par [T], next [T + 1], path [T], then the map of children's tokens
  double* px = reinterpret_cast<double*>(vd_smem);
  float* ux = reinterpret_cast<float*>(px + p.T);
  int32_t* tok = reinterpret_cast<int32_t*>(ux + p.T);
  int32_t* par = tok + p.T;
  int32_t* next = par + p.T;
  int32_t* path = next + p.T + 1;
  uint32_t* gone = reinterpret_cast<uint32_t*>(path + p.T);
  __shared__ int s_n, s_end;
  __shared__ VdBest s_warp[VD_THREADS / 32];
  __shared__ VdBest s_cta[VD_MAX_CLUSTER];
  uint32_t rank, nranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nranks));
  const int64_t b = blockIdx.x / nranks;
  const int T = p.T, V = p.V, tid = threadIdx.x, lane = tid & 31;
  const float* pb = p.p + b * (T + 1) * (int64_t)V;
  const float* ub = p.u + b * (T + 1);

  // The cluster's CTAs have all started before one writes into another's memory: arrive
  // here, wait there.
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // ------------------------------------------------------------------ the walk
  if (tid == 0) {
    s_n = T;
    s_end = 0;
  }
  auto word = [&](int x) { return WRAP ? (x >> 5) & (VD_BITS / 32 - 1) : x >> 5; };  // of entry x of the slice
  if (!p.q)
    for (int i = tid; i < p.words; i += VD_THREADS) gone[i] = 0;
  for (int i = tid; i <= T; i += VD_THREADS) next[i] = -1;
  __syncthreads();
  for (int i = tid; i < T; i += VD_THREADS) {
    const int64_t x = vd_token(p, b * T + i);
    const int32_t pa = p.parents ? p.parents[b * T + i] : i - 1;
    const bool in = x >= 0 && x < V && pa >= -1 && pa < i;
    if (!in && rank == 0) report_bounds(p.status, (int)b, V);
    tok[i] = in ? (int32_t)x : -1;
    par[i] = in ? pa : -2;
    const float pv = in ? pb[(int64_t)(pa + 1) * V + x] : 0.f;
    if (p.q) {
      const float qv = in ? p.q[(b * T + i) * (int64_t)V + x] : 0.f;
      if (!(__fmul_rn(ub[i], qv) < pv)) atomicMin(&s_n, i);
    } else {
      px[i] = (double)pv;
      ux[i] = in ? ub[pa + 1] : 0.f;
    }
  }
  __syncthreads();
  if (p.q) {
    if (tid == 0) s_end = s_n;
    for (int i = tid; i < T; i += VD_THREADS) path[i] = i;
  } else {
    // A warp per candidate, lanes over the older ones.  First: a sibling that repeats an
    // older one's token gives up its stretch.
    for (int i = tid >> 5; i < T; i += VD_THREADS / 32) {
      bool dup = false;
      for (int j = lane; j < i; j += 32) dup |= par[j] == par[i] && tok[j] == tok[i];
      if (__any_sync(0xFFFFFFFFu, dup) && lane == 0) px[i] = 0.0;
    }
    __syncthreads();
    for (int i = tid >> 5; i < T; i += VD_THREADS / 32) {
      // Where its stretch begins, and where it ends: the sum that the next sibling begins
      // at, of the same terms in the same order, so that rounding leaves no gap and no overlap.
      double at = 0.0;
      for (int j = lane; j < i; j += 32)
        if (par[j] == par[i]) at += px[j];
      double to = lane == (i & 31) ? at + px[i] : at;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        at += __shfl_xor_sync(0xFFFFFFFFu, at, o);
        to += __shfl_xor_sync(0xFFFFFFFFu, to, o);
      }
      const double uu = (double)ux[i];
      if (lane == 0 && par[i] >= -1 && at <= uu && uu < to) next[par[i] + 1] = i;
    }
    __syncthreads();
    if (tid == 0) {
      int n = 0, row = 0;
      while (n < T && next[row] >= 0) {  // ends: a child's index is above its parent's
        path[n++] = next[row];
        row = next[row] + 1;
      }
      s_n = n;
      s_end = row;
    }
    __syncthreads();
    const int lo = (int)rank * p.per;
    for (int i = tid; i < T; i += VD_THREADS)
      if (par[i] == s_end - 1 && tok[i] >= lo && tok[i] < lo + p.per)
        atomicOr(&gone[word(tok[i] - lo)], 1u << ((tok[i] - lo) & 31));
  }
  __syncthreads();
  const int n = s_n, end = s_end;

  // ------------------------------------------------------------------ the next token
  const float* row = pb + (int64_t)end * V;
  const float* qrow = p.q && n < T ? p.q + (b * T + n) * (int64_t)V : nullptr;
  const float* e = p.noise + b * (int64_t)V;
  const int lo = (int)rank * p.per, hi = min(V, lo + p.per);
  // Whether x is a child's token, given that its bit is set: where entries share bits the
  // children are gone through (T / VD_BITS of the entries at most).
  auto child = [&](int x) {
    bool is = !WRAP;
    if constexpr (WRAP)
      for (int i = 0; i < T && !is; ++i) is = tok[i] == x && par[i] == end - 1;
    return is;
  };
  VdBest best;
  for (int pass = 0; pass < 2; ++pass) {  // the second only where w is zero everywhere
    best = {-1.f, 0x7FFFFFFF, 0};
    const bool cut = pass == 0;
    // A ratio below 1 - 2^-20 of the best so far cannot win whatever its rounding, and one
    // product shows that; the correctly rounded division is left to the few that may.  The
    // best so far is the warp's (a lane's own let most steps of a warp divide).
    float bar = 0.f;
    auto one = [&](int x, float pv, float qv, float nv, bool out) {
      float w = pv;
      if (cut) {
        if (qrow) w = fmaxf(__fsub_rn(pv, qv), 0.f);
        if (out && child(x)) w = 0.f;
      }
      best.any |= w > 0.f;
      if (w >= bar * nv) vd_take(best, __fdiv_rn(w, nv), x);
    };
    auto share = [&] {  // non-negative floats are in order as integers
      const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(fmaxf(best.val, 0.f)));
      bar = __uint_as_float(top) * (1.f - 0x1p-20f);
    };
    if (p.vec4) {
#pragma unroll 2
      for (int x0 = lo; x0 < hi; x0 += VD_THREADS * 4) {
        const int x = x0 + tid * 4;
        if (x < hi) {
          const float4 pv = __ldg(reinterpret_cast<const float4*>(row + x));
          const float4 nv = __ldg(reinterpret_cast<const float4*>(e + x));
          float4 qv = make_float4(0.f, 0.f, 0.f, 0.f);
          if (qrow) qv = __ldg(reinterpret_cast<const float4*>(qrow + x));
          uint32_t g = 0;
          if (!p.q) g = gone[word(x - lo)] >> ((x - lo) & 31);
          one(x, pv.x, qv.x, nv.x, g & 1);
          one(x + 1, pv.y, qv.y, nv.y, g & 2);
          one(x + 2, pv.z, qv.z, nv.z, g & 4);
          one(x + 3, pv.w, qv.w, nv.w, g & 8);
        }
        share();
      }
    } else {
#pragma unroll 4
      for (int x0 = lo; x0 < hi; x0 += VD_THREADS) {
        const int x = x0 + tid;
        if (x < hi) {
          const uint32_t g = p.q ? 0u : gone[word(x - lo)] >> ((x - lo) & 31);
          one(x, __ldg(row + x), qrow ? __ldg(qrow + x) : 0.f, __ldg(e + x), g & 1);
        }
        share();
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float v = __shfl_xor_sync(0xFFFFFFFFu, best.val, o);
      const int32_t i = __shfl_xor_sync(0xFFFFFFFFu, best.idx, o);
      best.any |= __shfl_xor_sync(0xFFFFFFFFu, best.any, o);
      vd_take(best, v, i);
    }
    if (lane == 0) s_warp[tid >> 5] = best;
    if (pass == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    __syncthreads();
    if (tid < (int)nranks) {  // this CTA's best into slot `rank` of CTA `tid`
      for (int i = 0; i < VD_THREADS / 32; ++i) {
        best.any |= s_warp[i].any;
        vd_take(best, s_warp[i].val, s_warp[i].idx);
      }
      uint32_t at;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&s_cta[rank])), "r"(tid));
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(best.val) : "memory");
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at + 4), "r"(best.idx) : "memory");
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at + 8), "r"(best.any) : "memory");
    }
    cluster_sync();
    best = s_cta[0];
    for (int i = 1; i < (int)nranks; ++i) {
      best.any |= s_cta[i].any;
      vd_take(best, s_cta[i].val, s_cta[i].idx);
    }
    if (best.any || pass == 1) break;
    cluster_sync();  // every CTA has read the slots before they are written again
  }
  if (rank != 0) return;
  const int32_t x = best.idx < V ? best.idx : 0;
  for (int i = tid; i <= T; i += VD_THREADS) {
    const int64_t v = i < n ? (int64_t)tok[path[i]] : i == n ? (int64_t)x : -1;
    if (p.tok_i64) static_cast<int64_t*>(p.out)[b * (T + 1) + i] = v;
    else static_cast<int32_t*>(p.out)[b * (T + 1) + i] = (int32_t)v;
    if (i < T) p.path[b * T + i] = i < n ? path[i] : -1;
  }
  if (tid == 0) p.n_acc[b] = n;
}

}  // namespace ks
