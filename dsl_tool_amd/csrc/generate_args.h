// Arguments of the kernels that generate several continuations of a prompt:
// the cache's pages (pages.hip), rotary positions (rotary.hip) and the log
// probabilities of tokens (logprobs.hip).  Launchers assume arguments were
// validated.
#pragma once

#include "serve_args.h"

namespace dsl {

// The pages of a cache: k and v `bytes` each, scales [heads].
struct PageArgs {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  int64_t bytes;         // heads * page * dim
  int heads;
};

struct ForkArgs {
  const int32_t *lens, *table;                   // [seqs], [seqs][table_ld]
  int64_t table_ld;
  const int32_t *parents, *more;                 // [children]; new tokens [children] (nullptr: more_all each)
  int more_all;
  const int32_t *refs;                           // [pages]
  int seqs, width, children, pages, page;
  int32_t *out_lens, *out_table, *out_refs, *lacking;   // [children], [children][width], [pages], [1]
  int32_t *ws;
};
size_t fork_workspace_bytes(int seqs, int width, int children, int pages);
hipError_t launch_fork(const PageArgs &c, const ForkArgs &p, hipStream_t st);

struct CompactArgs {
  const int32_t *table;                          // [seqs][table_ld]
  int64_t table_ld;
  const int32_t *refs;
  int seqs, width, pages;
  int32_t *out_table, *out_refs, *moved, *live;  // [seqs][width], [pages], [pages], [1]
  int32_t *ws;
};
size_t compact_workspace_bytes(int pages);
hipError_t launch_compact(const PageArgs &c, const CompactArgs &p, hipStream_t st);

struct RotaryHeads {
  const void *x;         // [rows][heads][dim], unit stride in dim
  int64_t row, head;
  void *y;               // the same, may be x
  int64_t yrow, yhead;
  int heads;
};
struct RotaryArgs {
  RotaryHeads q, k;      // k.heads 0: none
  int rows, dim, half;   // half: pairs
  const void *positions; // [axes][pos_ld] int32 or int64
  bool pos64;
  int64_t pos_ld;
  int axes;
  const int32_t *axis_of;        // [half], nullptr: axis 0
  const double *freqs;           // [half]
  float magnitude;
  bool adjacent;         // pairs (2 i, 2 i + 1), else (i, i + half)
};
hipError_t launch_rotary(int src, const RotaryArgs &p, hipStream_t st);

struct LogprobArgs {
  const void *x;         // [rows][ld]
  int64_t ld;
  int rows, vocab;
  const int32_t *ids;    // [rows][ids_ld]
  int64_t ids_ld;
  int n_ids;
  float scale;
  int top;               // 0 .. kMaxTop, <= vocab
  float *logp, *entropy, *top_logp;              // [rows][n_ids], [rows], [rows][top]
  int32_t *top_ids;      // [rows][top]
  void *ws;
};
constexpr int kMaxTop = 32;
size_t logprob_workspace_bytes(int src, int rows, int vocab, int top);
hipError_t launch_logprobs(int src, const LogprobArgs &p, hipStream_t st);

}  // namespace dsl
