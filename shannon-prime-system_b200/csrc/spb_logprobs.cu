// spb_logprobs.cu -- log probabilities of given tokens from rows of logits, with the row's
// log-sum-exp, entropy and largest entries.
//
//   lse = m + log(sum e^(x - m)),  logprob = x[token] - lse,  entropy = log(sum e) - sum e (x - m) / sum e
// with m the row's maximum. -inf entries are masked tokens and weigh nothing. A row without a
// finite or +inf entry has lse -inf and entropy 0; a row that holds NaN or +inf has no
// distribution: lse, entropy, its tokens' logprobs and its alternatives' are NaN, the ids -1.
#include "spb_exact.cuh"
#include "spb_tree.cuh"

namespace spb {

namespace {

constexpr int LT = 256;

// larger value first, equal values lowest id first (-0 and +0 are equal); 0 is below every entry
__device__ __forceinline__ unsigned long long top_key(float v, int id) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)o << 32) | (uint32_t)~id;
}

__device__ float block_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (int i = 0; i < LT / 32; i++) s += red[i];
  return s;
}

__device__ unsigned long long block_max_u64(unsigned long long v, unsigned long long *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long m = 0;
  for (int i = 0; i < LT / 32; i++) m = max(m, red[i]);
  return m;
}

// One CTA per row, one pass per quantity.
__global__ void __launch_bounds__(LT) k_logprobs(LogprobArgs a) {
  __shared__ float red[LT / 32];
  __shared__ unsigned long long redk[LT / 32];
  const int r = blockIdx.x, tid = threadIdx.x;
  const float *x = a.x + (size_t)r * a.ld;
  float m = -INFINITY;
  bool bad = false;
  for (int j = tid; j < a.vocab; j += LT) {
    const float v = x[j];
    bad |= !(v < INFINITY);
    m = fmaxf(m, v);
  }
  bad = __syncthreads_or(bad);
  unsigned long long k = block_max_u64(top_key(m, 0), redk);
  {
    const uint32_t o = (uint32_t)(k >> 32);
    m = __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
  }
  float s = 0.0f, t = 0.0f;
  for (int j = tid; j < a.vocab; j += LT) {
    const float d = x[j] - m, e = expf(d);
    if (x[j] > -INFINITY) { s += e; t += e * d; }
  }
  s = block_sum(s, red);
  t = block_sum(t, red);
  float lse = m + logf(s), ent = logf(s) - t / s;
  if (m == -INFINITY) { lse = -INFINITY; ent = 0.0f; }
  if (bad) lse = ent = NAN;
  if (tid == 0) {
    if (a.lse) a.lse[r] = lse;
    if (a.entropy) a.entropy[r] = ent;
  }
  for (int i = tid; i < a.n_tok; i += LT) {
    const int tr = a.tok_row ? a.tok_row[i] : i;
    if (tr < 0 || tr >= a.rows) {
      if (r == 0) { raise_err(a.err, ERR_TOKEN); a.logprob[i] = NAN; }
      continue;
    }
    if (tr != r) continue;
    const int tok = a.tok[i];
    float v = NAN;
    if (tok >= 0 && tok < a.vocab) v = bad ? NAN : x[tok] == -INFINITY ? -INFINITY : x[tok] - lse;
    else if (tok != -1) raise_err(a.err, ERR_TOKEN);
    a.logprob[i] = v;
  }
  unsigned long long last = ~0ull;
  for (int i = 0; i < a.top; i++) {
    unsigned long long b = 0;
    for (int j = tid; j < a.vocab; j += LT) {
      const unsigned long long key = top_key(x[j], j);
      if (x[j] > -INFINITY && key < last && key > b) b = key;
    }
    b = block_max_u64(b, redk);
    last = b;
    if (tid == 0) {
      const int id = b && !bad ? (int)~(uint32_t)b : -1;
      a.ids[(size_t)r * a.top + i] = id;
      a.best[(size_t)r * a.top + i] = bad ? NAN : id < 0 ? -INFINITY : x[id] - lse;
    }
    if (!b) last = 0;
  }
}

}  // namespace

cudaError_t launch_logprobs(const LogprobArgs &a, cudaStream_t st) {
  if (a.rows <= 0) return cudaSuccess;
  k_logprobs<<<a.rows, LT, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace spb
