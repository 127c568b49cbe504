// spb_tree.cu -- verifying a tree of drafted tokens over a cache: the exact attention of its
// nodes, and the move of an accepted path's K and V rows behind the context.
//
// Node i of a sequence whose cache holds ctx positions is cached in slot ctx + i and stands at
// position ctx + depth(i). It sees the context and its own ancestors, inside its layer's window.
// Scores, exponentials and V-sums are the integers of the decode attention (k_attn): the same
// bytes as decoding each path of the tree token by token (sp_session.c:327-347, 429-442).
#include "spb_device.cuh"
#include "spb_exact.cuh"
#include "spb_tree.cuh"

#include <cstdlib>

namespace spb {

namespace {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Sequence s of the cache; false when its rows, context or slots are out of range.
__device__ bool tree_seq(const TreeCache &c, int s, int max_ctx, TreeSeq &q) {
  if (c.seqs) {
    q = c.seqs[s];
  } else {
    const size_t elems = (size_t)c.NL * c.NKV * c.page * c.HD;
    q.kv.k = c.ptab ? c.k : c.k + (size_t)s * elems;
    q.kv.v = c.ptab ? c.v : c.v + (size_t)s * elems;
    q.kv.ptab = c.ptab ? c.ptab + (size_t)s * c.ptab_ld : nullptr;
    q.kv.pg = c.page;
    q.ctx = c.ctx[s];
    q.row0 = c.row0[s];
    q.n = (int)max(-1ll, min((long long)c.row0[s + 1] - q.row0, (long long)TREE_NODES + 1));
    q.cap = c.ptab ? (int)min((long long)c.page * c.ptab_ld, 0x7fffffffll) : c.page;
  }
  return q.row0 >= 0 && q.n >= 0 && q.n <= TREE_NODES && q.row0 <= c.rows - q.n && q.ctx >= 0 && q.ctx <= max_ctx &&
         q.ctx <= q.cap - q.n;
}

// element offset of a slot's row in K or V; an entry outside the pool reads as page 0
__device__ __forceinline__ size_t tree_row(const TreeCache &c, const KvPages &kv, int layer, int g, int slot, uint32_t *err) {
  const int j = slot / kv.pg;
  int page = kv.ptab ? kv.ptab[j] : 0;
  if (kv.ptab && !c.seqs && (unsigned)page >= (unsigned)c.n_pages) {
    raise_err(err, ERR_TREE);
    page = 0;
  }
  return ((((size_t)page * c.NL + layer) * c.NKV + g) * kv.pg + (size_t)(slot - j * kv.pg)) * c.HD;
}

constexpr int TT = 256;

// One CTA per (row, head): the window's scores for their maximum, then again in runs of 256 slots
// for the exponentials and the V-sums.
__global__ void __launch_bounds__(TT) k_tree_attn(TreeAttnArgs a) {
  __shared__ int seq_sh;
  __shared__ int32_t par[TREE_NODES];
  __shared__ unsigned long long anc[TREE_NODES];
  __shared__ int32_t qs[256];
  __shared__ int32_t es[TT];
  __shared__ int32_t mx;
  __shared__ unsigned long long ssum;
  const int row = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int HD = a.c.HD, g = h / (a.NH / a.c.NKV);
  pdl_trigger();
  pdl_wait();
  if (tid == 0) { seq_sh = -1; mx = INT32_MIN; ssum = 0ull; }
  __syncthreads();
  TreeSeq q;
  for (int s = tid; s < a.c.n_seq; s += TT)
    if (tree_seq(a.c, s, a.max_ctx, q)) { if (row >= q.row0 && row < q.row0 + q.n) seq_sh = s; }
    else raise_err(a.err, ERR_TREE);
  __syncthreads();
  if (seq_sh < 0) return;
  tree_seq(a.c, seq_sh, a.max_ctx, q);
  const int node = row - q.row0;
  bool bad = false;
  if (tid < q.n) {
    const int p = a.parent[q.row0 + tid];
    bad = p < -1 || p >= tid;
    par[tid] = p;
  }
  for (int i = tid; i < HD; i += TT) qs[i] = a.q[((size_t)row * a.NH + h) * HD + i];
  if (__syncthreads_or(bad)) {
    if (tid == 0) raise_err(a.err, ERR_TREE);
    return;
  }
  if (tid < q.n) {
    unsigned long long m = 0;
    for (int p = tid; p >= 0; p = par[p]) m |= 1ull << p;
    anc[tid] = m;
  }
  __syncthreads();
  const int depth = __popcll(anc[node]) - 1;
  const int first = a.win < 0 ? 0 : max(0, q.ctx + depth - a.win + 1);
  const int end = q.ctx + q.n;
  auto sees = [&](int slot) {
    if (slot < q.ctx) return slot >= first;
    const int i = slot - q.ctx;
    return ((anc[node] >> i) & 1ull) != 0 && q.ctx + __popcll(anc[i]) - 1 >= first;
  };
  auto score = [&](int slot) -> int32_t {   // by one warp
    const int32_t *kr = q.kv.k + tree_row(a.c, q.kv, a.layer, g, slot, a.err);
    int64_t s = 0;
    for (int i = lane; i < HD; i += 32) s += (int64_t)qs[i] * kr[i];
    s = warp_sum_i64(s);
    float z = __fmul_rn(__double2float_rn(__dmul_rn(__ll2double_rn(s), 0x1p-32)), a.ascale);
    if (!(fabsf(z) < 131072.0f)) { raise_err(a.err, ERR_SCORE_RANGE); z = 0.0f; }
    return (int32_t)llround_d((double)z * 16384.0);
  };
  const int u0 = min(first, q.ctx);
  for (int j = u0 + warp; j < end; j += TT / 32)
    if (sees(j)) {
      const int32_t zi = score(j);
      if (lane == 0) atomicMax(&mx, zi);
    }
  __syncthreads();
  acc128 acc{0ull, 0ll};
  for (int j0 = u0; j0 < end; j0 += TT) {
    for (int j = warp; j < TT; j += TT / 32) {
      int64_t e = 0;
      if (j0 + j < end && sees(j0 + j)) e = exp_fixed((((int64_t)score(j0 + j) - (int64_t)mx) * ONE) >> 14);
      if (lane == 0) {
        es[j] = (int32_t)e;
        atomicAdd(&ssum, (unsigned long long)e);
      }
    }
    __syncthreads();
    if (tid < HD)
      for (int j = 0; j < min(TT, end - j0); j++)
        if (es[j]) acc128_add(acc, (int64_t)es[j] * q.kv.v[tree_row(a.c, q.kv, a.layer, g, j0 + j, a.err) + tid]);
    __syncthreads();
  }
  if (tid < HD) {
    const int64_t hi = (int64_t)(((uint64_t)acc.hi << 16) | (acc.lo >> 48));
    const int64_t qd = floordiv_s128(hi, acc.lo << 16, ssum);
    const float o = __double2float_rn(__dmul_rn(__ll2double_rn(qd), 0x1p-32));
    a.out[((size_t)row * a.NH + h) * HD + tid] = o;
    if (a.ao_max) atomicMax(a.ao_max + row, __float_as_uint(fabsf(o)));
  }
}

// ---- the accepted path's rows: slot ctx + path[i] -> slot ctx + i, ascending
//
// A thread owns one 16-byte column of one (K or V, layer, KV head) row set and walks the path, so
// no two threads touch the same bytes. path is strictly ascending, path[i] >= i: a batch loads its
// rows before it stores any, and what earlier batches stored lies below every later source.
constexpr int MOVE = 8;   // rows in flight per thread

__global__ void __launch_bounds__(256) k_kv_compact(KvCompactArgs a) {
  __shared__ int path[TREE_NODES];
  __shared__ size_t src[TREE_NODES], dst[TREE_NODES];   // element offsets of (layer 0, KV head 0)
  const int tid = threadIdx.x, s = blockIdx.y;
  pdl_trigger();
  pdl_wait();
  TreeSeq seq;   // (the path's length in the rows' place; the slots it reaches are checked below)
  if (!tree_seq(a.c, s, 0x7fffffff, seq)) {
    if (tid == 0) raise_err(a.err, ERR_TREE);
    return;
  }
  const int n = seq.n;
  if (tid < n) path[tid] = a.path[seq.row0 + tid];
  __syncthreads();
  bool bad = false;
  if (tid < n) {
    const int p = path[tid];
    bad = p < 0 || p >= TREE_NODES || (tid > 0 && p <= path[tid - 1]) || seq.ctx > seq.cap - 1 - p;
    if (!bad) {
      auto at = [&](int slot) { return tree_row(a.c, seq.kv, 0, 0, slot, a.err); };
      const int j0 = (seq.ctx + p) / seq.kv.pg, j1 = (seq.ctx + tid) / seq.kv.pg;
      if (seq.kv.ptab && !a.c.seqs)
        bad = (unsigned)seq.kv.ptab[j0] >= (unsigned)a.c.n_pages || (unsigned)seq.kv.ptab[j1] >= (unsigned)a.c.n_pages;
      if (!bad) { src[tid] = at(seq.ctx + p); dst[tid] = at(seq.ctx + tid); }
    }
  }
  if (__syncthreads_or(bad)) {   // nothing of this sequence moves
    if (tid == 0) raise_err(a.err, ERR_TREE);
    return;
  }
  int keep = 0;   // a first run that is in place already
  while (keep < n && path[keep] == keep) keep++;
  const int per = a.c.HD / 4;                          // 16-byte columns of a row
  const long long cols = 2ll * a.c.NL * a.c.NKV * per;
  const long long x = (long long)blockIdx.x * 256 + tid;
  if (x >= cols) return;
  const int col = (int)(x % per);
  const long long r = x / per;                        // (K or V, layer, KV head)
  const long long lh = r % ((long long)a.c.NL * a.c.NKV);
  int32_t *base = (r >= (long long)a.c.NL * a.c.NKV ? seq.kv.v : seq.kv.k) + (size_t)lh * seq.kv.pg * a.c.HD + 4 * col;
  for (int i0 = keep; i0 < n; i0 += MOVE) {
    int4 b[MOVE];
#pragma unroll
    for (int u = 0; u < MOVE; u++)
      if (i0 + u < n) b[u] = *reinterpret_cast<const int4 *>(base + src[i0 + u]);
#pragma unroll
    for (int u = 0; u < MOVE; u++)
      if (i0 + u < n) *reinterpret_cast<int4 *>(base + dst[i0 + u]) = b[u];
  }
}

bool tree_pdl() {
  static const bool on = [] {
    const char *e = getenv("SPB_PDL");
    return !(e && e[0] == '0');
  }();
  return on;
}

template <typename A>
cudaError_t launch(void (*kern)(A), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t st, const A &a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (tree_pdl()) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    na++;
  }
  if (cluster > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = cluster;
    attr[na].val.clusterDim.y = 1;
    attr[na].val.clusterDim.z = 1;
    na++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace

cudaError_t launch_tree_attn(const TreeAttnArgs &a, cudaStream_t st) {
  if (a.c.rows <= 0) return cudaSuccess;
  return launch(k_tree_attn, dim3(a.NH, a.c.rows), dim3(TT), 0, 1, st, a);
}

cudaError_t launch_kv_compact(const KvCompactArgs &a, cudaStream_t st) {
  if (a.c.rows <= 0) return cudaSuccess;
  const long long cols = 2ll * a.c.NL * a.c.NKV * (a.c.HD / 4);
  return launch(k_kv_compact, dim3((unsigned)((cols + 255) / 256), a.c.n_seq), dim3(256), 0, 1, st, a);
}

}  // namespace spb
