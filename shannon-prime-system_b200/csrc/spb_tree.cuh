// spb_tree.cuh -- launch interface of the kernels that verify a tree of drafted tokens: the
// attention of its nodes over a cache (spb_tree.cu), the move of an accepted path's K/V rows
// (spb_tree.cu) and log probabilities with entropy and alternatives (spb_logprobs.cu).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "spb_kernels.cuh"

namespace spb {

constexpr int TREE_NODES = 64;   // drafted tokens of one sequence: an ancestor set is one 64-bit word
constexpr int TREE_SPAN = 1 << 20; // slots a node may see: the V-sums' low words stay below 2^63

// One sequence: its cache, the positions it holds, its rows [row0, row0 + n) among the step's
// (node i cached in slot ctx + i) and the slots its page table reaches.
struct TreeSeq {
  KvPages kv;
  int32_t ctx, row0, n, cap;
};

// Where the sequences are: descriptors (the session path), or a pool with a page table per
// sequence and the arrays of an isolated call.
struct TreeCache {
  const TreeSeq *seqs;             // device [n_seq], or null:
  int32_t *k, *v;                  // pools [n_pages][NL][NKV][page][HD]
  const int32_t *ptab;             // device [n_seq][ptab_ld]; null: sequence s is page s
  const int32_t *ctx, *row0;       // device [n_seq], [n_seq + 1]
  int n_pages, page, ptab_ld;
  int n_seq, rows;                 // rows: of all sequences together
  int NL, NKV, HD;
};

struct TreeAttnArgs {
  TreeCache c;
  int layer, NH, win;              // win < 0: no window
  int max_ctx;                     // no sequence's context is longer
  const int32_t *parent;           // device [rows]: index of a node's parent in its sequence, -1 for a first token
  const int32_t *q;                // [rows][NH * HD] rotated queries on the 2^16 grid
  float *out;                      // [rows][NH * HD]
  float ascale;
  uint32_t *err;
  uint32_t *ao_max;                // nullable: per-row atomicMax of the f32 bits of max |out|
};
cudaError_t launch_tree_attn(const TreeAttnArgs &a, cudaStream_t st);

struct KvCompactArgs {
  TreeCache c;                     // c.row0: the bounds of each sequence's path in `path`, c.rows its length
  const int32_t *path;             // device: accepted nodes, ascending in each sequence
  uint32_t *err;
};
cudaError_t launch_kv_compact(const KvCompactArgs &a, cudaStream_t st);

constexpr int LOGPROB_TOP = 32;          // alternatives of a row at most
constexpr int LOGPROB_VOCAB = 1 << 22;   // entries of a row at most

struct LogprobArgs {
  const float *x;                  // [rows][ld]
  int rows, vocab;
  int64_t ld;
  const int32_t *tok_row, *tok;    // [n_tok] row (null: token t of row t) and token; -1: no token
  int n_tok;
  float *logprob;                  // [n_tok]
  float *lse, *entropy;            // [rows], nullable
  int top;
  int32_t *ids;                    // [rows][top]
  float *best;                     // [rows][top]
  uint32_t *err;
};
cudaError_t launch_logprobs(const LogprobArgs &a, cudaStream_t st);

}  // namespace spb
