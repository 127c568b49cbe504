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

#include <cooperative_groups.h>
#include <cstdlib>

namespace cg = cooperative_groups;

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

// ---- exact products on the matrix units
//
// An int32 x is four balanced base-256 digits, x = sum_i d_i 256^i with d_i in [-128, 127]: adding
// 0x80808080 makes every digit u_i = d_i + 128 an unsigned byte (the carries are the balancing).
// <q, k> = sum_ij 256^(i+j) <digit i of q, digit j of k>, each an int8 matrix product into int32;
// products of the same i + j share one accumulator (a class). The queries' digits are signed, the
// cache's lower three stay biased, and the bias comes off once per sum:
//   <q, k> = sum_i sum_{j<3} 256^(i+j) <d_i(q), u_j(k)> + (fourth digits of k) - BIAS sum q.
// The exponentials e in [0, 2^30] are four unsigned bytes, so the V-sums' bias is BIAS sum e. A fourth
// digit that is zero throughout an operand (|x| < 127.5 2^16 on the grid) adds nothing and is skipped.
// Classes: 3 * 128 * 255 * 256 < 2^25 for a score, (3 * 255 + 128) * 255 per slot of a V-sum.
constexpr int64_t BIAS = 128 * (1 + 256 + 65536);

// byte planes of four int32 values x + 0x80808080: byte i of out[p] is biased digit p of the i-th value
__device__ __forceinline__ void digits(int x0, int x1, int x2, int x3, uint32_t (&out)[4]) {
  const uint32_t w0 = (uint32_t)x0 + 0x80808080u, w1 = (uint32_t)x1 + 0x80808080u;
  const uint32_t w2 = (uint32_t)x2 + 0x80808080u, w3 = (uint32_t)x3 + 0x80808080u;
  const uint32_t a = __byte_perm(w0, w1, 0x5140), b = __byte_perm(w2, w3, 0x5140);
  const uint32_t c = __byte_perm(w0, w1, 0x7362), d = __byte_perm(w2, w3, 0x7362);
  out[0] = __byte_perm(a, b, 0x5410);
  out[1] = __byte_perm(a, b, 0x7632);
  out[2] = __byte_perm(c, d, 0x5410);
  out[3] = __byte_perm(c, d, 0x7632) ^ 0x80808080u;   // signed
}
__device__ __forceinline__ uint4 bytes4(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
  const uint32_t a = __byte_perm(w0, w1, 0x5140), b = __byte_perm(w2, w3, 0x5140);
  const uint32_t c = __byte_perm(w0, w1, 0x7362), d = __byte_perm(w2, w3, 0x7362);
  return make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x5410),
                    __byte_perm(c, d, 0x7632));
}

__device__ __forceinline__ void mma_ss(int32_t (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_su(int32_t (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_us(int32_t (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_uu(int32_t (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// 32 bytes of a row in one load: a quad of lanes takes a whole 128-byte line
__device__ __forceinline__ void ld_kv8(int4 &a, int4 &b, const int32_t *p) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p));
}
__device__ __forceinline__ void ld_kv2(int32_t (&v)[2], const int32_t *p) {
  asm volatile("ld.global.v2.b32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "l"(p));
}

constexpr int32_t UNSEEN = INT32_MIN;   // the score of a position that a node does not see

// exp_fixed of a score's distance below its maximum in 32-bit steps: far = max - z in units of 2^-14,
// g = ceil(far log2(e)) in 2^30, n = g >> 30 octaves and the rest; the island's polynomial in x = 2^30 -
// rest, each (acc x) >> 30 as the high word of acc * 4x (x < 2^30 here). 32 octaves (363408.75 steps) and
// more are the island's zero.
__device__ __forceinline__ uint32_t mad_hi(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("mad.hi.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t exp_grid(int32_t z, int32_t mx) {
  const uint32_t far = (uint32_t)mx - (uint32_t)z;
  const uint64_t g = (uint64_t)far * (uint32_t)K_LOG2E + 16383u;   // 2^44 per octave
  const uint32_t n = (uint32_t)(g >> 44), r4 = (uint32_t)(g >> 12) & ~3u, x4 = 0u - r4;
  uint32_t acc = mad_hi(165394u, x4, 1431680u);
  acc = mad_hi(acc, x4, 10327387u);
  acc = mad_hi(acc, x4, 59597083u);
  acc = mad_hi(acc, x4, 257941248u);
  acc = mad_hi(acc, x4, 744261118u);
  acc = mad_hi(acc, x4, 1073741824u) >> 1;
  acc = (r4 == 0u ? 1u << 30 : acc) >> (n & 31u);
  return z == UNSEEN || n >= 32u ? 0u : acc;
}

// f32 of floor(N 2^16 / S) 2^-32 (the decode attention's rounding), r = 2^16 / S in double: N r is off by
// at most 2^-50 of itself, so its floor is the quotient's unless a whole number lies that near; those, and
// quotients beyond 2^50, take the exact division.
__device__ __forceinline__ float finish(const acc128 &N, uint64_t S, double r) {
  const double nd = (int64_t)N.lo >> 63 == N.hi ? __ll2double_rn((int64_t)N.lo)
                                                : __dadd_rn(__dmul_rn(__ll2double_rn(N.hi), 0x1p64), __ull2double_rn(N.lo));
  const double x = __dmul_rn(nd, r), w = floor(x), f = __dsub_rn(x, w), eps = __dmul_rn(fabs(x), 0x1p-50);
  if (f > eps && f < __dsub_rn(1.0, eps) && fabs(x) < 0x1p50) return __double2float_rn(__dmul_rn(w, 0x1p-32));
  const int64_t hi = (int64_t)(((uint64_t)N.hi << 16) | (N.lo >> 48));   // |N| < 2^80
  return __double2float_rn(__dmul_rn(__ll2double_rn(floordiv_s128(hi, N.lo << 16, S)), 0x1p-32));
}

// One CTA: 16 query vectors (a sequence's nodes x the G query heads of one KV head) over a run
// of slots; a cluster of CL CTAs covers the sequence's slots and joins maxima, sums and V-sums,
// which are whole numbers, so no split changes a byte.
//   scores    a warp takes 8 slots at a time: their K rows go from global memory straight into the
//             column operand (a lane's 32 bytes are eight columns of one slot, so the digit planes
//             are a byte transpose in registers), the queries' planes wait in shared memory;
//             9 products, 33 cycles a slot at HD 256 (18 of them the matrix units', 6 the recombination
//             and scaling of its eight slots; without the K loads as long)
//   exps      in place over the scores, each four neighbours' bytes transposed into the planes of
//             the row operand; 7 cycles a slot
//   V-sums    a warp takes 16 head dims over the slots of the run, V rows again straight from global
//             memory (eight slots x two dims per lane and step); 12 products, 50 cycles a slot (24 the
//             matrix units'; 36 if the same bytes lay in 256-byte pieces: 64 bytes of a row at a time cost
//             the L1 its lookups, as much when every one of them hits)
// and 28000 cycles a CTA besides: finding the tile 2600, rows 2400, queries and parents 5500, the maxima's
// exchange 5000, the sums' 9500, the division 2600 (2080 slots; a cluster of 4).
// Measured and not kept (64 nodes at context 8192, 217 us): 32 query vectors per CTA (364: the sums
// spill, V comes in pieces of 32 bytes), 8 warps of twice the dims (241), V through shared memory for the
// whole CTA (260: a barrier per step) or in a ring per warp (229: 80 KB that the L1 misses while K comes
// in), a row's pieces fetched by neighbouring lanes and shuffled (214, small trees 2 to 4 % slower), whole lines
// of V by two neighbouring warps that hand each other their planes (290: a barrier per step), 16 slots per warp
// and step of K (262), K in runs of four steps, in two buffers (spills) or in one (217 both).
// 128 registers a thread at 16 warps hold all but 244 (width 256), 280 (128) and 312 bytes (64), which spill.
// MULTI (more slots per rank than scores are kept for): the maxima first, then scores again in runs of
// CS slots, each run's V-sums added up in shared memory: K is read twice (12B shape, 4 nodes: 222 us behind
// 33000 positions in one run, 476 behind 40000; 264 to 268 bytes spill, 216 at width 64).
template <int HD, bool MULTI>
struct TreeTile {
  static constexpr int QV = 16, KS = HD / 32;
  static constexpr int NW = 16, TT = 32 * NW;
  static constexpr int ND = 2;                                  // head dims of a lane's V rows: its 56 sums
  static constexpr int DG = HD / (8 * ND), PG = NW / DG;        // warps along the dims, groups along the slots
  // slots whose scores are kept, in blocks of 16 query vectors x 32 slots in the row operand's order:
  // [slot half][row half][lane][4 slots], and then the exponentials' planes, [plane][lane][4 registers]
  static constexpr int CS = MULTI ? 1056 : 2112;
  static constexpr size_t QF = (size_t)KS * 4 * 512;            // the queries' planes
  static constexpr size_t SUMS = (size_t)QV * HD * 16;          // V-sums of a tile
  static constexpr size_t HEAD = QF + (MULTI ? SUMS : 0);       // (MULTI: the running V-sums)
  static constexpr size_t SC = (size_t)QV * CS * 4;
  static constexpr size_t WORK = SC + CS * 4;
  // over the scores: every source's sums of this rank's dims (HD / CL of them, or up to one more: CL <= 16)
  static constexpr size_t POST = (SUMS + (size_t)16 * QV * 16) * (MULTI ? 1 : PG);
  static constexpr int BESIDE = MULTI ? 0 : (int)((SC - POST) / (QV * 4)) & ~31;   // slots that leave room for the sums
  static constexpr size_t SMEM = HEAD + (WORK > POST ? WORK : POST);
};

template <int HD, bool MULTI>
__global__ void __launch_bounds__(512, 1) k_tree_attn(TreeAttnArgs a, int CL) {
  using T = TreeTile<HD, MULTI>;
  constexpr int QV = T::QV, KS = T::KS, CS = T::CS, TT = T::TT, NW = T::NW, ND = T::ND;
  constexpr int KG = KS < 4 ? 1 : 2;                            // 32-column steps of K in one run of loads
  extern __shared__ __align__(128) uint8_t raw[];
  uint4 *qf = reinterpret_cast<uint4 *>(raw);                   // [KS][4][32]
  longlong2 *keep = reinterpret_cast<longlong2 *>(raw + T::QF); // MULTI: [QV][HD]
  int32_t *sc = reinterpret_cast<int32_t *>(raw + T::HEAD);     // [CS / 32][512]
  uint32_t *rows = reinterpret_cast<uint32_t *>(raw + T::HEAD + T::SC);  // [CS] the slots' rows in K and V
  longlong2 *sums = reinterpret_cast<longlong2 *>(raw + T::HEAD);        // [CL][PG][QV][HD / CL]
  __shared__ int32_t par[TREE_NODES];
  __shared__ unsigned long long anc[TREE_NODES];
  __shared__ int32_t first[QV];
  __shared__ unsigned long long seen[QV];
  __shared__ int32_t bounds[2];                                 // -1: bad parents; the tile's latest window start
  __shared__ int32_t mx[QV], mx_in[16][QV];
  __shared__ unsigned long long ssum[QV], s_in[16][QV], qsum[QV];
  __shared__ uint32_t omx[QV];
  __shared__ double rinv[QV];
  __shared__ int32_t out_at[QV], node_of[QV];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n8 = lane >> 2, c4 = lane & 3;
  const int rank = CL > 1 ? (int)cluster.block_rank() : 0, g = blockIdx.x / CL % a.c.NKV;   // heads of a tile side by side
  const int G = a.NH / a.c.NKV;
  pdl_trigger();
  if (tid < QV) { mx[tid] = UNSEEN; ssum[tid] = qsum[tid] = 0ull; omx[tid] = 0u; }
  pdl_wait();

  // ---- which sequence: tiles are counted over the sequences (every warp for itself), up to 32 of them the
  // longest contexts first: their CTAs run longest, and the short ones fill the gaps (8 sessions of 8 nodes,
  // contexts of 128 to 8192: 196 -> 150 us)
  TreeSeq q;
  int tile = -1;
  const int at = blockIdx.x / CL / a.c.NKV;
  for (int s0 = 0, before = 0; s0 < a.c.n_seq; s0 += 32) {
    int n = 0, ctx = -1;
    if (s0 + lane < a.c.n_seq) {
      if (tree_seq(a.c, s0 + lane, a.max_ctx, q)) {
        n = (q.n * G + QV - 1) / QV;
        ctx = q.ctx;
      } else if (warp == 0) {
        raise_err(a.err, ERR_TREE);
      }
    }
    int excl = 0, total = 0;   // tiles of this lane's predecessors, of all 32
    const bool sorted = a.c.n_seq <= 32;
    for (int o = 0; o < min(32, a.c.n_seq - s0); o++) {
      const int c = __shfl_sync(0xffffffffu, ctx, o), m = __shfl_sync(0xffffffffu, n, o);
      total += m;
      if (sorted ? c > ctx || (c == ctx && o < lane) : o < lane) excl += m;
    }
    const int z = at - before - excl;
    const uint32_t hit = __ballot_sync(0xffffffffu, z >= 0 && z < n);
    if (hit) {
      const int l = __ffs(hit) - 1;
      tile = __shfl_sync(0xffffffffu, z, l);
      tree_seq(a.c, s0 + l, a.max_ctx, q);
      break;
    }
    before += total;
  }
  if (tile < 0) return;   // (the whole cluster)
  const int x0 = tile * QV, nq = min(QV, q.n * G - x0);   // this tile's query vectors: x -> node x / G, head x % G

  // ---- this rank's slots [c0, c1): from where the window of a first token begins (deeper nodes' begin later)
  const int u0 = a.win < 0 ? 0 : max(0, q.ctx - a.win + 1), u1 = q.ctx + q.n;
  const int span = ((u1 - u0 + CL - 1) / CL + 31) & ~31;
  if (!MULTI && span > CS) {   // (the launch gave every rank CS slots at most: not reached)
    if (tid == 0) raise_err(a.err, ERR_TREE);
    return;
  }
  if (CL > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int c0 = min(u0 + rank * span, u1), c1 = min(c0 + span, u1);

  auto locate = [&](int cb, int len) {   // the rows of slots [cb, cb + len), the last one again up to a multiple of 32
    for (int i = tid; i < ((len + 31) & ~31); i += TT)
      rows[i] = (uint32_t)(tree_row(a.c, q.kv, a.layer, g, cb + min(i, len - 1), a.err) / HD);
    __syncthreads();
  };

  // K in runs of one or two steps of columns, two runs on their way in turn (a run waits as one: a warp has
  // six load counters, and more of them rolling would wait for each other)
  int4 kb[2][KG][2];
  auto load = [&](int4 (&b)[KG][2], const int32_t *p) {
#pragma unroll
    for (int i = 0; i < KG; i++) ld_kv8(b[i][0], b[i][1], p + i * 32);
  };
  auto row_of = [&](int t) { return q.kv.k + (size_t)rows[t * 8 + n8] * HD + 8 * c4; };
  auto kfirst = [&](int len) {
    if (warp < ((len + 31) & ~31) / 8) {
      load(kb[0], row_of(warp));
      load(kb[1], row_of(warp) + KG * 32);
    }
  };

  if (c0 < c1) locate(c0, min(CS, c1 - c0));
  kfirst(min(CS, c1 - c0));   // across the queries' and parents' loads

  // ---- warp 0: ancestors by doubling, then every query vector's window and tree slots
  bool bad = false;
  if (warp == 0) {
    int up[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int node = lane + 32 * i;
      up[i] = node < q.n ? a.parent[q.row0 + node] : -1;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int node = lane + 32 * i;
      if (up[i] < -1 || up[i] >= node) { bad = node < q.n; up[i] = -1; }
      par[node] = up[i];
      anc[node] = (1ull << node) | (up[i] >= 0 ? 1ull << up[i] : 0ull);
    }
    bad = __any_sync(0xffffffffu, bad);
    __syncwarp();
    for (int r = 1; r < q.n; r <<= 1) {
      unsigned long long m[2];
      int p[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        m[i] = up[i] >= 0 ? anc[up[i]] : 0ull;
        p[i] = up[i] >= 0 ? par[up[i]] : -1;
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 2; i++) {
        anc[lane + 32 * i] |= m[i];
        par[lane + 32 * i] = up[i] = p[i];
      }
      __syncwarp();
    }
    int f = q.ctx, hi = 0;
    unsigned long long m = 0;
    if (lane < nq) {
      m = anc[(x0 + lane) / G];
      const int depth = __popcll(m) - 1;
      f = a.win < 0 ? 0 : max(0, q.ctx + depth - a.win + 1);
      if (f > q.ctx)   // the window leaves ancestors out
        for (unsigned long long b = m; b; b &= b - 1) {
          const int j = __ffsll((long long)b) - 1;
          if (q.ctx + __popcll(anc[j]) - 1 < f) m &= ~(1ull << j);
        }
      hi = f;
    }
    if (lane < QV) {
      first[lane] = f;
      seen[lane] = m;
      node_of[lane] = (x0 + lane) / G - x0 / G;              // (a tile may begin inside a node's heads)
      out_at[lane] = (q.row0 + (x0 + lane) / G) * a.NH + g * G + (x0 + lane) % G;
    }
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) { bounds[0] = bad ? -1 : 0; bounds[1] = hi; }
  }
  // ---- the other warps: the queries' digit planes in the row operand's order, and their sums
  bool top = false;
  if (warp > 0)
    for (int i = tid - 32; i < KS * 32; i += TT - 32) {
      const int l = i & 31, ks = i >> 5;
      uint32_t pl[4][4];
#pragma unroll
      for (int u = 0; u < 4; u++) {   // (row, columns): the operand's four registers
        const int x = (l >> 2) + (u & 1) * 8, d = ks * 32 + (l & 3) * 8 + (u >> 1) * 4;
        int4 v = make_int4(0, 0, 0, 0);
        if (x < nq) {
          const int node = (x0 + x) / G, h = (x0 + x) % G;
          v = *reinterpret_cast<const int4 *>(a.q + ((size_t)(q.row0 + node) * a.NH + (size_t)g * G + h) * HD + d);
        }
        digits(v.x, v.y, v.z, v.w, pl[u]);
#pragma unroll
        for (int p = 0; p < 3; p++) pl[u][p] ^= 0x80808080u;
        top |= pl[u][3] != 0u;
        int64_t s = (int64_t)v.x + v.y + (int64_t)v.z + v.w;   // of the row's four lanes
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        if ((l & 3) == 0 && s != 0) atomicAdd(&qsum[x], (unsigned long long)s);
      }
#pragma unroll
      for (int p = 0; p < 4; p++) qf[(ks * 4 + p) * 32 + l] = make_uint4(pl[0][p], pl[1][p], pl[2][p], pl[3][p]);
    }
  const bool q3 = __syncthreads_or(top);   // some query has a fourth digit
  if (bounds[0] < 0) {   // the parents are out of range (for the whole cluster)
    if (tid == 0) raise_err(a.err, ERR_TREE);
    if (CL > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    return;
  }
  const int clear = bounds[1];

  // ---- scores of slots [cb, cb + len) into sc, the rows' maxima into mx (the first rows are on their way)
  auto scores = [&](int cb, int len, bool want_max) {
    const int nt = ((len + 31) & ~31) / 8;
    int32_t lmax[2] = {UNSEEN, UNSEEN};
    const float scale = __fmul_rn(a.ascale, 0x1p-18f);   // score on the 2^32 grid -> units of 2^-14
    const int32_t *kr = warp < nt ? row_of(warp) : q.kv.k;
#pragma unroll 1
    for (int t = warp; t < nt; t += NW) {
      const int32_t *kn = row_of(min(t + NW, nt - 1));
      int32_t acc[7][4];
#pragma unroll
      for (int c = 0; c < 7; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[c][i] = 0;
      uint32_t k3 = 0u;
#pragma unroll
      for (int k0 = 0; k0 < KS; k0 += KG) {
        int4(&kc)[KG][2] = kb[k0 / KG & 1];
#pragma unroll
        for (int i = 0; i < KG; i++) {
          uint32_t b0[4], b1[4];
          digits(kc[i][0].x, kc[i][0].y, kc[i][0].z, kc[i][0].w, b0);
          digits(kc[i][1].x, kc[i][1].y, kc[i][1].z, kc[i][1].w, b1);
          k3 |= b0[3] | b1[3];
#pragma unroll
          for (int p = 0; p < 3; p++) {
            const uint4 A = qf[((k0 + i) * 4 + p) * 32 + lane];
#pragma unroll
            for (int j = 0; j < 3; j++) mma_su(acc[p + j], A, b0[j], b1[j]);
          }
        }
        const int kx = k0 + 2 * KG;
        load(kc, kx < KS ? kr + kx * 32 : kn + (kx - KS) * 32);
      }
      if (__any_sync(0xffffffffu, k3 != 0u) || q3) {   // fourth digits: the rows once more (a vote per step costs 10 %)
#pragma unroll 1
        for (int ks = 0; ks < KS; ks++) {
          int4 v0, v1;
          ld_kv8(v0, v1, kr + ks * 32);
          uint32_t b0[4], b1[4];
          digits(v0.x, v0.y, v0.z, v0.w, b0);
          digits(v1.x, v1.y, v1.z, v1.w, b1);
#pragma unroll
          for (int p = 0; p < 4; p++) mma_ss(acc[p + 3], qf[(ks * 4 + p) * 32 + lane], b0[3], b1[3]);
          const uint4 A = qf[(ks * 4 + 3) * 32 + lane];
#pragma unroll
          for (int j = 0; j < 3; j++) mma_su(acc[3 + j], A, b0[j], b1[j]);
        }
      }
      kr = kn;
      const int slot = cb + t * 8 + 2 * c4;   // this lane's two slots
      const bool all = cb + t * 8 >= clear && cb + t * 8 + 8 <= min(q.ctx, c1);
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int x = n8 + h * 8;
          const int64_t off = -BIAS * (int64_t)qsum[x];
          int32_t z[2];
          bool see[2] = {true, true};
          if (!all) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int sl = slot + i;
              see[i] = (sl < q.ctx ? sl >= first[x] : ((seen[x] >> ((sl - q.ctx) & 63)) & 1ull) != 0) && sl < c1;
            }
          }
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int e = 2 * h + i;
            int64_t s = off + acc[0][e];
            s += (int64_t)acc[1][e] * 256;
            s += (int64_t)acc[2][e] * 65536;
            s += (int64_t)acc[3][e] * 16777216;
            s += (int64_t)((uint64_t)((uint32_t)acc[4][e] + (uint32_t)acc[5][e] * 256u + (uint32_t)acc[6][e] * 65536u) << 32);
            // f32 of the score (one rounding: below 2^53 wherever |z| < 2^17), then z 2^14 rounded half
            // away from zero: adding a half towards zero never crosses a whole number
            float v = __fmul_rn(__ll2float_rn(s), scale);
            if (!(fabsf(v) < 2147483648.0f)) {
              if (see[i]) raise_err(a.err, ERR_SCORE_RANGE);
              v = 0.0f;
            }
            z[i] = see[i] ? __float2int_rz(__fadd_rz(v, copysignf(0.5f, v))) : UNSEEN;
            lmax[h] = max(lmax[h], z[i]);
          }
          // slots 8 (t % 4) + 2 c4 .. of block t / 4: half (t % 4) / 2, lane 4 n8 + (2 (t % 2) + c4 / 2)
          int32_t *to = sc + (t >> 2) * 512 + ((t >> 1) & 1) * 256 + h * 128;
          *reinterpret_cast<int2 *>(to + (4 * n8 + 2 * (t & 1) + (c4 >> 1)) * 4 + 2 * (c4 & 1)) = make_int2(z[0], z[1]);
        }
    }
    if (want_max) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
          int32_t v = lmax[h];
          v = max(v, __shfl_xor_sync(0xffffffffu, v, 1));
          v = max(v, __shfl_xor_sync(0xffffffffu, v, 2));
          if (c4 == 0 && v != UNSEEN) atomicMax(&mx[n8 + h * 8], v);
      }
    }
    __syncthreads();
  };

  // ---- exponentials in place, a block of 16 x 32 by a warp: a lane's four quarters are its four registers
  // of the row operand, four neighbours' bytes each, and leave as planes
  auto exps = [&](int len) {
    int64_t sum[2] = {0, 0};
#pragma unroll 1
    for (int i = warp; i < (len + 31) / 32; i += NW) {
      const int32_t m0 = mx[n8], m1 = mx[n8 + 8];
      int4 *p = reinterpret_cast<int4 *>(sc + i * 512) + lane;
      uint4 r[4];
      int64_t s0 = 0, s1 = 0;
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int4 z = p[u * 32];
        const int32_t mm = u & 1 ? m1 : m0;
        const uint32_t e0 = exp_grid(z.x, mm), e1 = exp_grid(z.y, mm), e2 = exp_grid(z.z, mm), e3 = exp_grid(z.w, mm);
        const int64_t s = ((int64_t)e0 + e1) + ((int64_t)e2 + e3);
        if (u & 1) s1 += s;
        else s0 += s;
        r[u] = bytes4(e0, e1, e2, e3);
      }
      uint4 *o = reinterpret_cast<uint4 *>(p);
      o[0] = make_uint4(r[0].x, r[1].x, r[2].x, r[3].x);
      o[32] = make_uint4(r[0].y, r[1].y, r[2].y, r[3].y);
      o[64] = make_uint4(r[0].z, r[1].z, r[2].z, r[3].z);
      o[96] = make_uint4(r[0].w, r[1].w, r[2].w, r[3].w);
      sum[0] += s0;
      sum[1] += s1;
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      int64_t s = sum[h];
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if (c4 == 0 && s != 0) atomicAdd(&ssum[n8 + 8 * h], (unsigned long long)s);
    }
    __syncthreads();
  };

  // ---- V-sums: warp (dg, pg) takes dims 16 dg .. over every PG-th run of 32 slots
  const int dg = warp % T::DG, pg = warp / T::DG;
  int32_t acc[ND][7][4];
  int32_t va[2][4][ND], vb[2][4][ND];   // two runs' V rows, on their way while the run before is multiplied
  auto vload = [&](int32_t (&v)[2][4][ND], int st, int nst) {
    if (st >= nst) return;
    const int32_t *base = q.kv.v + dg * 8 * ND + ND * n8;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint4 r = *reinterpret_cast<const uint4 *>(rows + st * 32 + h * 16 + 4 * c4);
      ld_kv2(v[h][0], base + (size_t)r.x * HD);
      ld_kv2(v[h][1], base + (size_t)r.y * HD);
      ld_kv2(v[h][2], base + (size_t)r.z * HD);
      ld_kv2(v[h][3], base + (size_t)r.w * HD);
    }
  };
  auto vfirst = [&](int len) {
    if (len <= 0) return;
    vload(va, pg, (len + 31) / 32);
    vload(vb, pg + T::PG, (len + 31) / 32);
  };
  auto vsums = [&](int len) {   // (the first two runs' rows are on their way)
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int c = 0; c < 7; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[d][c][i] = 0;
    const int nst = (len + 31) / 32;
    auto step = [&](int32_t (&v)[2][4][ND], int st) {
      uint32_t b[ND][2][4], v3 = 0u;   // [dim][half][plane]
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          digits(v[h][0][d], v[h][1][d], v[h][2][d], v[h][3][d], b[d][h]);
          v3 |= b[d][h][3];
        }
      vload(v, st + 2 * T::PG, nst);
      const bool any3 = __any_sync(0xffffffffu, v3 != 0u);
      const uint4 *A = reinterpret_cast<const uint4 *>(sc + st * 512) + lane;
#pragma unroll
      for (int p = 0; p < 4; p++) {
        const uint4 e = A[p * 32];
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
          for (int j = 0; j < 3; j++) mma_uu(acc[d][p + j], e, b[d][0][j], b[d][1][j]);
      }
      if (any3) {
#pragma unroll
        for (int p = 0; p < 4; p++)
#pragma unroll
          for (int d = 0; d < ND; d++) mma_us(acc[d][p + 3], A[p * 32], b[d][0][3], b[d][1][3]);
      }
    };
#pragma unroll 1
    for (int st = pg; st < nst; st += 2 * T::PG) {
      step(va, st);
      if (st + T::PG < nst) step(vb, st + T::PG);
    }
  };
  // V-sum = lo + hi 2^32: four classes below 2^31 each fit lo with room for every rank's, three fit hi
  auto fold = [&](int d, int i) {
    const int32_t(&c)[7][4] = acc[d];
    longlong2 r;
    r.x = c[0][i] + (long long)c[1][i] * 256 + (long long)c[2][i] * 65536 + (long long)c[3][i] * 16777216;
    r.y = c[4][i] + (long long)c[5][i] * 256 + (long long)c[6][i] * 65536;
    return r;
  };
  auto each = [&](auto &&f) {   // (query vector, dim, V-sum) of this lane's accumulators
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) f(n8 + (i >> 1) * 8, dg * 8 * ND + ND * (2 * c4 + (i & 1)) + d, fold(d, i));
  };

  if (!MULTI) {   // (the launch gave every rank CS slots at most)
    scores(c0, c1 - c0, true);
    vfirst(c1 - c0);   // across the exchange and the exponentials
  } else {
    for (int cb = c0; cb < c1; cb += CS) {
      if (cb > c0) {
        locate(cb, min(CS, c1 - cb));
        kfirst(min(CS, c1 - cb));
      }
      scores(cb, min(CS, c1 - cb), true);
    }
  }
  if (CL > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // every rank has started
    for (int i = tid; i < CL * QV; i += TT) *cluster.map_shared_rank(&mx_in[rank][i % QV], i / QV) = mx[i % QV];
    cluster.sync();
    if (tid < QV) {
      int32_t m = UNSEEN;
      for (int r = 0; r < CL; r++) m = max(m, mx_in[r][tid]);
      mx[tid] = m;
    }
    __syncthreads();
  }
  if (MULTI) {
    for (int i = tid; i < QV * HD; i += TT) keep[i] = make_longlong2(0, 0);
    for (int cb = c0; cb < c1; cb += CS) {
      const int len = min(CS, c1 - cb);
      __syncthreads();
      locate(cb, len);
      kfirst(len);
      scores(cb, len, false);
      exps(len);
      vfirst(len);
      vsums(len);
      for (int r = 0; r < T::PG; r++) {   // (the slot groups add to the same sums in turn)
        if (pg == r)
          each([&](int x, int d, longlong2 v) {
            longlong2 &k = keep[x * HD + d];
            k.x += v.x;
            k.y += v.y;
          });
        if (T::PG > 1) __syncthreads();
      }
    }
  } else {
    exps(c1 - c0);
    vsums(c1 - c0);
  }
  // ---- join: dim d's sums go to rank d / DPR, straight from registers
  // (their memory: behind the scores, or over them once every rank is done with its own)
  const bool beside = !MULTI && span <= T::BESIDE;
  if (beside) sums = reinterpret_cast<longlong2 *>(raw + T::HEAD + (size_t)T::BESIDE * QV * 4);
  else if (CL > 1) cluster.sync();
  else __syncthreads();
  // (x / DPR as a product: x < 16 HD = 2^12 at most, and x times the reciprocal's excess stays below 2^22)
  const int DPR = (HD + CL - 1) / CL, src = MULTI ? 1 : T::PG;   // a rank's dims; sums per rank
  const uint32_t inv = ((1u << 22) + DPR - 1) / DPR;
  auto by_dpr = [&](int x) { return (int)((uint32_t)x * inv >> 22); };
  auto push = [&](int x, int d, longlong2 v) {
    if (x >= nq) return;
    const int o = by_dpr(d);
    longlong2 *to = sums + ((rank * src + (MULTI ? 0 : pg)) * QV + x) * DPR + (d - o * DPR);
    if (CL > 1) to = cluster.map_shared_rank(to, o);
    *to = v;
  };
  if (MULTI) {
    for (int i = tid; i < QV * HD; i += TT) push(i / HD, i % HD, keep[i]);
  } else {
    each(push);
  }
  if (CL > 1) {
    for (int i = tid; i < CL * QV; i += TT) *cluster.map_shared_rank(&s_in[rank][i % QV], i / QV) = ssum[i % QV];
    cluster.sync();   // the last cluster access
    if (tid < QV) {
      unsigned long long s = 0;
      for (int r = 0; r < CL; r++) s += s_in[r][tid];
      ssum[tid] = s;
    }
  }
  if (tid < QV) rinv[tid] = __ddiv_rn(65536.0, __ull2double_rn(ssum[tid]));
  __syncthreads();
#pragma unroll 2
  for (int i = tid; i < nq * DPR; i += TT) {
    const int x = by_dpr(i), d = i - x * DPR;
    if (rank * DPR + d >= HD) continue;   // (the last ranks' dims where HD / CL is no whole number)
    long long lo = 0, hi = 0;
    for (int r = 0; r < CL * src; r++) {
      const longlong2 v = sums[(r * QV + x) * DPR + d];
      lo += v.x;
      hi += v.y;
    }
    const long long S = (long long)ssum[x];
    acc128 N{0ull, 0ll};   // lo + hi 2^32 - BIAS sum e
    acc128_add(N, lo);
    acc128_add(N, acc128{(uint64_t)hi << 32, hi >> 32});
    acc128_add(N, acc128{(uint64_t)(-BIAS * S), __mul64hi(-BIAS, S)});
    const float o = finish(N, (uint64_t)S, rinv[x]);
    a.out[(size_t)out_at[x] * HD + rank * DPR + d] = o;
    if (a.ao_max) atomicMax(&omx[node_of[x]], __float_as_uint(fabsf(o)));
  }
  if (a.ao_max) {
    __syncthreads();
    if (tid < QV && omx[tid]) atomicMax(a.ao_max + q.row0 + x0 / G + tid, omx[tid]);
  }
}

// ---- the accepted path's rows: slot ctx + path[i] -> slot ctx + i, ascending
//
// A thread owns one 16-byte column of one (K or V, layer, KV head) row set and walks the path, so
// no two threads touch the same bytes. path is strictly ascending, path[i] >= i: a batch loads its
// rows before it stores any, and what earlier batches stored lies below every later source. The bytes
// moved bound it, and short of that the latency of one batch: 12 rows in each of 8 sessions (36 layers x 8
// heads x 128: 57 MB, 8.6 us at the measured copy rate) take 9.7 us a call, of which the host needs as much.
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

template <typename... K, typename... A>
cudaError_t launch(void (*kern)(K...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t st, const A &...a) {
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
  return cudaLaunchKernelEx(&cfg, kern, static_cast<K>(a)...);
}

}  // namespace

namespace {

// A CTA's fixed work (finding its tile, the queries, two cluster barriers, the join: 16000 to 20000 cycles) in
// slots of 80 cycles. 12B shape, 4 nodes: context 100 16.8 / 13.4 / 13.2 us with clusters of 1 / 4 / 8, context
// 2048 36 / 25 / 45 with 4 / 8 / 16 (8 clusters of 16 take two waves); 64 nodes at context 8192 216 / 300 with
// 4 / 8 (two waves and five).
constexpr int TREE_FIXED = 256;

template <int HD, bool MULTI>
cudaError_t tree_attn(const TreeAttnArgs &a, long long tiles, long long likely, int span, cudaStream_t st) {
  using T = TreeTile<HD, MULTI>;
  auto kern = k_tree_attn<HD, MULTI>;
  // CTAs that run at once, by cluster size (asked once per device, before any launch: a capture never
  // sees a failed launch)
  static int room[64][17];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  dev &= 63;
  if (room[dev][1] == 0) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)T::SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    for (int i = 16; i >= 1; i--) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(i);
      cfg.blockDim = dim3(T::TT);
      cfg.dynamicSmemBytes = T::SMEM;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = i;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) n = 0;
      room[dev][i] = n * i;
    }
    (void)cudaGetLastError();
    if (room[dev][1] <= 0) return cudaErrorLaunchOutOfResources;
  }
  // the cluster size whose waves of CTAs take the least slots one after the other
  int best = 0;
  long long cost = 0;
  for (int i = 1; i <= 16; i++) {
    const long long per = ((span + i - 1) / i + 31) & ~31;
    if (room[dev][i] <= 0 || (!MULTI && per > T::CS)) continue;
    const long long waves = (likely * a.c.NKV * i + room[dev][i] - 1) / room[dev][i];
    const long long c = waves * (per + TREE_FIXED);
    if (best == 0 || c < cost) { best = i; cost = c; }
  }
  if (best == 0) return cudaErrorNotSupported;
  if (tiles * a.c.NKV * best > 0x7fffffffll) return cudaErrorInvalidValue;
  return launch(kern, dim3((unsigned)(tiles * a.c.NKV * best)), dim3(T::TT), T::SMEM, best, st, a, best);
}

template <int HD>
cudaError_t tree_attn_hd(const TreeAttnArgs &a, cudaStream_t st) {
  const int G = a.NH / a.c.NKV;
  // more slots than a cluster of 16 keeps scores for go in runs
  const int span = (a.win >= 0 && a.win < a.max_ctx ? a.win : a.max_ctx) + TREE_NODES;
  // tiles: every sequence's last one may be partly filled
  constexpr int QV = TreeTile<HD, false>::QV;
  const long long most = (long long)a.c.n_seq * ((TREE_NODES * G + QV - 1) / QV);
  long long tiles = a.c.n_seq == 1 ? ((long long)a.c.rows * G + QV - 1) / QV : (long long)a.c.rows * G / QV + a.c.n_seq;
  if (tiles > most) tiles = most;
  // the tiles there are if the sequences are alike (the grid's others leave at once)
  const long long likely = a.c.n_seq * (((long long)a.c.rows * G + (long long)QV * a.c.n_seq - 1) / ((long long)QV * a.c.n_seq));
  if (span <= 16 * TreeTile<HD, false>::CS) {
    const cudaError_t e = tree_attn<HD, false>(a, tiles, likely, span, st);
    if (e != cudaErrorNotSupported) return e;   // (no room for a cluster that large)
  }
  return tree_attn<HD, true>(a, tiles, likely, span, st);
}

}  // namespace

cudaError_t launch_tree_attn(const TreeAttnArgs &a, cudaStream_t st) {
  if (a.c.rows <= 0) return cudaSuccess;
  switch (a.c.HD) {
    case 64: return tree_attn_hd<64>(a, st);
    case 128: return tree_attn_hd<128>(a, st);
    case 256: return tree_attn_hd<256>(a, st);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_kv_compact(const KvCompactArgs &a, cudaStream_t st) {
  if (a.c.rows <= 0) return cudaSuccess;
  const long long cols = 2ll * a.c.NL * a.c.NKV * (a.c.HD / 4);
  return launch(k_kv_compact, dim3((unsigned)((cols + 255) / 256), a.c.n_seq), dim3(256), 0, 1, st, a);
}

}  // namespace spb
