// spb_logprobs.cu -- log probabilities of given tokens from rows of logits, with the row's
// log-sum-exp, entropy and largest entries.
//
//   lse = m + log(sum e^(x - m)),  logprob = x[token] - lse,  entropy = log(sum e) - sum e (x - m) / sum e
// with m the row's maximum. -inf entries are masked tokens and weigh nothing. A row without a
// finite or +inf entry has lse -inf and entropy 0; a row that holds NaN or +inf has no
// distribution: lse, entropy, its tokens' logprobs and its alternatives' are NaN, the ids -1.
//
// One pass over the logits, so memory bounds it: 1000 rows x 151936 take 110 to 114 us, 81 to 85 % of the
// measured copy rate; 64 rows x 262144 16.4 us (62 %; 256 CTAs on 148 SMs make up 1.6 of the 6.2 us above the
// copy), 19.8 with one alternative and 23.1 with 20: every CTA ranks its own best, then they are joined. A row
// is cut into up to 16 parts of at least 16384 entries; a CTA's thread takes every 512th group of four
// neighbours of a part, a warp joins its threads' sums, and a part its sixteen warps'. A cluster of C CTAs
// shares the parts of a row; C follows from the rows of the call (few rows: a row over many CTAs), but what is
// summed in which order follows from the vocabulary's size alone, so a row's bytes depend neither on the other
// rows nor on its alignment.
//
// A thread sums e^(x - m) = 2^((x - m) L), L = log2(e) in f32, and the same weighted by the exponents, with m
// the largest entry it has met: so the row's largest entry counts 1 exactly, sum e >= 1, and neither log(sum e) nor
// x - m holds digits that the other has to cancel (a reference below the maximum costs a likely token's log
// probability and a peaked row's entropy 1e-6).
// The difference comes first: in x L - m L the rounding of m L grows with m (0.5 at 1e7, 2^99 at 1e37) and would
// stand in the exponent. The exponential is ex2.approx, which is low on the whole by less than its 2 units in the
// last place: entropies of 5 nats come out 4e-7 low (2e-8 with a double's exponential; exp2f, 133 us for the 1000
// rows, and log2(e) in two parts, 118, are as low).
//
// The largest entries: the top'th largest of the threads' maxima bounds the top'th largest entry from below,
// and only the threads that reach it can hold larger ones: their groups are read again (from L2) and what
// reaches the bound is ranked by counting. Rows whose large entries crowd into few threads' groups, or are
// equal in great number, can overflow that list: they find one entry after the other.
#include <cooperative_groups.h>
#include <cstdlib>
#include <mutex>

#include "spb_exact.cuh"
#include "spb_logprob_plan.h"
#include "spb_tree.cuh"

namespace cg = cooperative_groups;

namespace spb {

namespace {

constexpr int LT = 512, LW = LT / 32;
constexpr int LCAND = 2048;        // entries at or above the bound that are ranked by counting
constexpr int LBATCH = 4;          // groups of four in flight per thread
constexpr float LOG2E_F = 1.44269504f;
constexpr float LOG2E_LO = 1.92596299e-8f;   // log2(e) - LOG2E_F
constexpr float LN2_F = 0.693147182f;
constexpr float FLOOR2 = -200.0f;  // exponents of two below this are zero in f32

// larger value first, equal values lowest id first (-0 and +0 are equal); every entry above -inf is above 0
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long top_key(float v, int id) {
  return v > -INFINITY ? ((unsigned long long)ordered(v) << 32) | (uint32_t)~id : 0ull;
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Running {
  float m, s, t;   // largest entry, sum of 2^((x - m) L), the same weighted by its exponent
};

// e^d, d <= 0 the distance of two references (at least one above -inf; else 0), and its exponent of two a. A
// reference stands for many entries at once: the rounding of a and log2(e)'s rest are made good.
__device__ __forceinline__ float rescale(float d, float &a) {
  d = fmaxf(d, -140.0f);   // (e^-140 is zero in f32, and NaN, of equal infinities, becomes that)
  a = __fmul_rn(d, LOG2E_F);
  const float f = exp2_fast(a), rest = __fmaf_rn(d, LOG2E_LO, __fmaf_rn(d, LOG2E_F, -a));
  return __fmaf_rn(f, __fmul_rn(rest, LN2_F), f);
}

// part [p0, p1) of a row that starts SH floats behind a 16-byte boundary
template <int SH, bool ENT>
__device__ __forceinline__ void part(const float *x, int p0, int p1, int vocab, Running &r) {
  const int lane = threadIdx.x & 31, b1 = (p1 + 3) >> 2;
  const float4 *xa = reinterpret_cast<const float4 *>(x - SH);   // group b is entries 4 b .. of xa, SH on
#pragma unroll 1
  for (int b0 = (p0 >> 2) + (int)threadIdx.x - lane; b0 < b1; b0 += LBATCH * LT) {   // (warp-uniform)
    float v[LBATCH][4];
    const int last = b0 + (LBATCH - 1) * LT + 31;   // the batch's last group
    if (last < b1 && 4 * last + (SH ? 8 : 4) <= vocab && (SH == 0 || b0 > 0)) {
#pragma unroll
      for (int u = 0; u < LBATCH; u++) {
        const int b = b0 + u * LT + lane;
        const float4 c = xa[b];
        v[u][0] = c.x; v[u][1] = c.y; v[u][2] = c.z; v[u][3] = c.w;
        if (SH) {   // (the rest of the group: the neighbour's line, from L1)
          const float4 d = xa[b + 1];
          const float w[8] = {c.x, c.y, c.z, c.w, d.x, d.y, d.z, d.w};
#pragma unroll
          for (int i = 0; i < 4; i++) v[u][i] = w[SH + i];
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < LBATCH; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int e = 4 * (b0 + u * LT + lane) + i;
          v[u][i] = e < p1 ? x[e] : -INFINITY;
        }
    }
    float bm = v[0][0];
#pragma unroll
    for (int u = 0; u < LBATCH; u++)
#pragma unroll
      for (int i = 0; i < 4; i++) bm = fmaxf(bm, v[u][i]);
    if (bm > r.m) {
      float a;
      const float f = rescale(__fsub_rn(r.m, bm), a);
      r.t = __fmul_rn(f, __fmaf_rn(r.s, a, r.t));
      r.s = __fmul_rn(r.s, f);
      r.m = bm;
    }
    const float m = r.m == -INFINITY ? 0.0f : r.m;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int u = 0; u < LBATCH; u++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float a = max_nan(__fmul_rn(__fsub_rn(v[u][i], m), LOG2E_F), FLOOR2), e = exp2_fast(a);
        s = __fadd_rn(s, e);
        if (ENT) t = __fmaf_rn(e, a, t);
      }
    r.s = __fadd_rn(r.s, s);
    r.t = __fadd_rn(r.t, t);
  }
}

__device__ __forceinline__ unsigned long long warp_max_u64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// (m, s, t) of two disjoint sets of entries as one, s and t being sums relative to m
__device__ __forceinline__ void join(float &m, float &s, float &t, float m2, float s2, float t2) {
  const float mm = fmaxf(m, m2);
  float a, b;
  const float f = rescale(__fsub_rn(m, mm), a), g = rescale(__fsub_rn(m2, mm), b);
  t = __fadd_rn(__fmul_rn(f, __fmaf_rn(s, a, t)), __fmul_rn(g, __fmaf_rn(s2, b, t2)));
  s = __fadd_rn(__fmul_rn(s, f), __fmul_rn(s2, g));
  m = mm;
}
// over W neighbouring lanes (a power of two); every one of them gets the result
template <int W>
__device__ __forceinline__ void join_lanes(float &m, float &s, float &t) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    const float t2 = __shfl_xor_sync(0xffffffffu, t, o);
    // (the same operands in the same order on both sides of the pair)
    if ((threadIdx.x & o) == 0) join(m, s, t, m2, s2, t2);
    else {
      float mm = m2, ss = s2, tt = t2;
      join(mm, ss, tt, m, s, t);
      m = mm; s = ss; t = tt;
    }
  }
}

template <bool ENT>
__global__ void __launch_bounds__(LT, 3) k_logprobs(LogprobArgs a, int C, int P, int per) {
  __shared__ float um[LPARTS][LW], us[LPARTS][LW], ut[LPARTS][LW];   // this CTA's parts, warp by warp
  __shared__ float pm[LPARTS], ps[LPARTS], pt[LPARTS];               // the row's parts, pushed by their ranks
  __shared__ uint32_t list[LT], bound_sh, redv[LW];
  __shared__ unsigned long long redk[LW], best[LOGPROB_TOP], cand[LCAND];
  __shared__ unsigned long long in_best[16][LOGPROB_TOP];            // every rank's best, on rank 0
  __shared__ int count, n_cand, n_win;
  __shared__ uint16_t winner[LT];
  __shared__ float m_sh, ls_sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = C > 1 ? (int)cluster.block_rank() : 0, row = blockIdx.x / C;
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) { count = n_cand = n_win = 0; bound_sh = 1u; }
  if (tid < LOGPROB_TOP) best[tid] = 0ull;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float *x = a.x + (size_t)row * a.ld;
  // ---- the rank's parts: part p of every C
  const int sh = (int)(((uintptr_t)x >> 2) & 3);
  float largest = -INFINITY;   // this thread's
#pragma unroll 1
  for (int p = rank, i = 0; p < P; p += C, i++) {
    const int p0 = p * per, p1 = min(p0 + per, a.vocab);
    Running r{-INFINITY, 0.0f, 0.0f};
    switch (sh) {
      case 0: part<0, ENT>(x, p0, p1, a.vocab, r); break;
      case 1: part<1, ENT>(x, p0, p1, a.vocab, r); break;
      case 2: part<2, ENT>(x, p0, p1, a.vocab, r); break;
      default: part<3, ENT>(x, p0, p1, a.vocab, r); break;
    }
    largest = fmaxf(largest, r.m);
    float m = r.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float shift;
    const float f = rescale(__fsub_rn(r.m, m), shift);
    float s = __fmul_rn(r.s, f), t = __fmul_rn(f, __fmaf_rn(r.s, shift, r.t));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, o));
      t = __fadd_rn(t, __shfl_xor_sync(0xffffffffu, t, o));
    }
    if (lane == 0) { um[i][warp] = m; us[i][warp] = s; ut[i][warp] = t; }
  }
  // with alternatives: the ceil(top / 16)'th largest of the warp's maxima (top <= 32: one of the first two)
  uint32_t key = 0u;
  if (a.top > 0) {
    key = largest > -INFINITY ? ordered(largest) : 0u;
    uint32_t k1 = __reduce_max_sync(0xffffffffu, key);
    if (a.top > LW) {
      const int l = __ffs(__ballot_sync(0xffffffffu, key == k1)) - 1;
      k1 = __reduce_max_sync(0xffffffffu, lane == l ? 0u : key);
    }
    if (lane == 0) redv[warp] = k1;
  }
  __syncthreads();
  if (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // every rank has started
  // warp i joins part i's warps and hands the part to every rank
  if (rank + warp * C < P) {
    float m = um[warp][lane & (LW - 1)], s = us[warp][lane & (LW - 1)], t = ut[warp][lane & (LW - 1)];
    join_lanes<LW>(m, s, t);
    const int p = rank + warp * C;
    if (lane < C) {
      if (C > 1) {
        *cluster.map_shared_rank(&pm[p], lane) = m;
        *cluster.map_shared_rank(&ps[p], lane) = s;
        *cluster.map_shared_rank(&pt[p], lane) = t;
      } else {
        pm[p] = m; ps[p] = s; pt[p] = t;
      }
    }
  }
  if (a.top > 0) {
    // at least `top` threads' maxima reach this: those go into a list, its top'th is the bound (fewer than
    // `top` threads hold any entry above -inf: the bound is 1, every such entry counts)
    uint32_t loose = redv[0];
#pragma unroll
    for (int w = 1; w < LW; w++) loose = min(loose, redv[w]);
    if (key >= loose && key != 0u) list[atomicAdd(&count, 1)] = key;
    __syncthreads();
    const int n = count;
    if (tid < n) {
      const uint32_t k = list[tid];
      int above = 0;
#pragma unroll 8
      for (int i = 0; i < n; i++) above += list[i] > k || (list[i] == k && i < tid);
      if (above == a.top - 1) bound_sh = k;
    }
    __syncthreads();
    const uint32_t bound = bound_sh;
    // the threads that reach the bound (`top` of them, more only where maxima are equal): their groups, an
    // entry per thread
    if (key >= bound && key != 0u) winner[atomicAdd(&n_win, 1)] = (uint16_t)tid;
    __syncthreads();
    const int steps = (per + 4 * LT - 1) / (4 * LT), mine = (P - rank + C - 1) / C, each = 4 * steps * mine;
    const int entries = n_win * each;
#pragma unroll 1
    for (int i0 = tid; i0 < entries; i0 += 4 * LT) {
      float v[4];
      int id[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int i = i0 + u * LT, w = i / each, j = i - w * each;
        const int st = (j >> 2) % steps, p = rank + (j >> 2) / steps * C;
        id[u] = i < entries ? p * per + 4 * (winner[w] + st * LT) + (j & 3) : a.vocab;
        const bool in = i < entries && id[u] < min((p + 1) * per, a.vocab);
        v[u] = in ? x[id[u]] : -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const unsigned long long k = top_key(v[u], id[u]);
        if ((uint32_t)(k >> 32) >= bound) {
          const int at = atomicAdd(&n_cand, 1);
          if (at < LCAND) cand[at] = k;
        }
      }
    }
    __syncthreads();
    const int nc = n_cand;
    if (nc <= LCAND) {
      for (int c = tid; c < nc; c += LT) {
        const unsigned long long k = cand[c];
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < nc; i++) above += cand[i] > k;
        if (above < a.top) best[above] = k;
      }
    } else {   // one entry after the other
      unsigned long long last = ~0ull;
      for (int i = 0; i < a.top; i++) {
        unsigned long long b = 0ull;
        for (int p = rank; p < P; p += C)
          for (int e = p * per + tid; e < min((p + 1) * per, a.vocab); e += LT) {
            const unsigned long long k = top_key(x[e], e);
            if (k < last && k > b) b = k;
          }
        b = warp_max_u64(b);
        if (lane == 0) redk[warp] = b;
        __syncthreads();
        for (int w = 0; w < LW; w++) b = max(b, redk[w]);
        __syncthreads();
        last = b;
        if (tid == 0) best[i] = b;
      }
    }
    __syncthreads();
    if (tid < a.top) {
      if (C > 1) *cluster.map_shared_rank(&in_best[rank][tid], 0) = best[tid];
      else in_best[0][tid] = best[tid];
    }
  }
  if (C > 1) cluster.sync();   // the last cluster access
  else __syncthreads();
  // ---- every rank: the row's statistics
  if (warp == 0) {
    float m = -INFINITY, s = 0.0f, t = 0.0f;
    if (lane < P) { m = pm[lane]; s = ps[lane]; t = pt[lane]; }
    join_lanes<32>(m, s, t);
    // (a row without entries above -inf: s 0)
    const bool none = !(s == s) || m == INFINITY;
    const float ls = none ? NAN : logf(s);
    if (lane == 0) {
      m_sh = m;
      ls_sh = ls;
      if (rank == 0) {
        if (a.lse) a.lse[row] = none ? NAN : s > 0.0f ? __fadd_rn(m, ls) : -INFINITY;
        if (a.entropy) a.entropy[row] = none ? NAN : s > 0.0f ? __fsub_rn(ls, __fmul_rn(LN2_F, __fdiv_rn(t, s))) : 0.0f;
      }
    }
  }
  __syncthreads();
  // x - lse as (x - m) - log(s), m the row's maximum: likely tokens keep the digits that lse has lost to m
  const float m0 = m_sh, ls = ls_sh;
  auto logprob = [&](float x) { return ls != ls ? NAN : x == -INFINITY ? -INFINITY : __fsub_rn(__fsub_rn(x, m0), ls); };
  // ---- this row's tokens: without tok_row token `row`, else every row's CTAs look through the list (row 0's
  // cluster also reports the rows that are out of range)
  const int t1 = a.tok_row ? a.n_tok : min(a.n_tok, row + 1);
  for (int i = (a.tok_row ? rank * LT : rank == 0 ? row : a.n_tok) + tid; i < t1; i += C * LT) {
    const int tr = a.tok_row ? a.tok_row[i] : row;
    if (tr < 0 || tr >= a.rows) {
      if (row == 0) { raise_err(a.err, ERR_TOKEN); a.logprob[i] = NAN; }
      continue;
    }
    if (tr != row) continue;
    const int tok = a.tok[i];
    float v = NAN;
    if (tok >= 0 && tok < a.vocab) v = logprob(x[tok]);
    else if (tok != -1) raise_err(a.err, ERR_TOKEN);
    a.logprob[i] = v;
  }
  // ---- rank 0: the alternatives of all ranks
  if (rank == 0 && a.top > 0) {
    if (C > 1) {   // lists in descending order, joined two by two, a pair by a warp
      unsigned long long *to = cand;
      for (int n = C; n > 1; n = (n + 1) / 2) {
        if (2 * warp < n) {
          unsigned long long k = 0ull, o = 0ull;
          const int l = 2 * warp, rev = 31 - lane;
          if (n == C) {
            if (lane < a.top) k = in_best[l][lane];
            if (l + 1 < n && rev < a.top) o = in_best[l + 1][rev];
          } else {
            const unsigned long long *from = cand + (to == cand ? 256 : 0);
            k = from[l * 32 + lane];
            if (l + 1 < n) o = from[(l + 1) * 32 + rev];
          }
          k = max(k, o);   // the larger half of the two, as a bitonic sequence
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) {
            const unsigned long long p = __shfl_xor_sync(0xffffffffu, k, d);
            k = (lane & d) ? min(k, p) : max(k, p);
          }
          if (n > 2) to[warp * 32 + lane] = k;
          else if (lane < a.top) best[lane] = k;
        }
        to = to == cand ? cand + 256 : cand;
        __syncthreads();
      }
    }
    __syncthreads();
    if (tid < a.top) {
      const unsigned long long k = best[tid];
      a.ids[(size_t)row * a.top + tid] = k == 0ull || ls != ls ? -1 : (int)~(uint32_t)k;
      a.best[(size_t)row * a.top + tid] = logprob(k == 0ull ? -INFINITY : key_value(k));
    }
  }
}

// which clusters run, asked once per device (a capture never sees a failed launch)
struct Room {
  std::mutex mu;
  bool asked = false;                 // (a call that could not ask leaves it to the next)
  bool fits[2][3][LPARTS + 1] = {};   // [entropy][pad][CTAs]
};

template <bool ENT>
cudaError_t ask(bool (&fits)[3][LPARTS + 1]) {
  cudaError_t e = cudaFuncSetAttribute(k_logprobs<ENT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k_logprobs<ENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, LPADS[2]);
  if (e != cudaSuccess) return e;
  for (int p = 0; p < 3; p++)
    for (int c = 2; c <= LPARTS; c++) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)c);
      cfg.blockDim = dim3(LT);
      cfg.dynamicSmemBytes = LPADS[p];
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = c;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      fits[p][c] = cudaOccupancyMaxActiveClusters(&n, k_logprobs<ENT>, &cfg) == cudaSuccess && n > 0;
    }
  (void)cudaGetLastError();
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_logprobs(const LogprobArgs &a, cudaStream_t st) {
  if (a.rows <= 0) return cudaSuccess;
  static Room rooms[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  Room &room = rooms[dev & 63];
  {
    std::lock_guard<std::mutex> lk(room.mu);
    if (!room.asked) {
      e = ask<false>(room.fits[0]);
      if (e == cudaSuccess) e = ask<true>(room.fits[1]);
      if (e != cudaSuccess) return e;
      room.asked = true;
    }
  }
  const auto &fits = room.fits[a.entropy ? 1 : 0];
  const LogprobPlan plan = plan_logprobs(a.rows, a.vocab, [&](int c, int pad) { return fits[pad == 0 ? 0 : pad == LPADS[1] ? 1 : 2][c]; });
  const int C = plan.ctas, P = plan.parts, per = plan.per;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(C * a.rows));
  cfg.blockDim = dim3(LT);
  cfg.dynamicSmemBytes = plan.pad;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int na = 0;
  static const bool pdl = [] {
    const char *v = getenv("SPB_PDL");
    return !(v && v[0] == '0');
  }();
  if (pdl) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    na++;
  }
  if (C > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = C;
    attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
    na++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  return a.entropy ? cudaLaunchKernelEx(&cfg, k_logprobs<true>, a, C, P, per) : cudaLaunchKernelEx(&cfg, k_logprobs<false>, a, C, P, per);
}

}  // namespace spb
