// extern "C" entry points, declared in include/dsl_gemm.h, of what generates
// several continuations of a prompt: the cache's pages between steps, rotary
// positions and the log probabilities of tokens.  As in capi.hip, everything is
// validated on the host before anything is enqueued, and nothing is allocated.
#include "capi_util.h"
#include "generate_args.h"

using namespace dsl::capi;

namespace {

constexpr int64_t kInts = (int64_t)1 << 31;

// The sizes of a cache, a table and its sequences.
int check_pool(const char *fn, int64_t pages, int64_t heads, int64_t page, int64_t dim, int64_t seqs, int64_t width) {
  if (pages < 0 || heads <= 0 || seqs < 0 || width < 0 || pages >= kInts)
    return fail(DSL_ERR_ARG, "%s: need 0 <= pages < 2^31, heads > 0, seqs, width >= 0", fn);
  if (dim != 64 && dim != 128 && dim != 256)
    return fail(DSL_ERR_UNSUPPORTED, "%s: head dim %lld must be 64, 128 or 256", fn, (long long)dim);
  if (page != 16 && page != 32 && page != 64 && page != 128 && page != 256)
    return fail(DSL_ERR_UNSUPPORTED, "%s: page size %lld must be 16, 32, 64, 128 or 256", fn, (long long)page);
  if (heads > 16384 || seqs > 65535)
    return fail(DSL_ERR_UNSUPPORTED, "%s: at most 16384 heads and 65535 sequences in a call", fn);
  if (width > (kInts - 65536) / page)
    return fail(DSL_ERR_ARG, "%s: page table rows span more than 2^31 - 65536 tokens", fn);
  return DSL_OK;
}

int check_pool_tensors(const char *fn, dsl::PageArgs *c, void *k, void *v, float *ks, float *vs, int64_t pages,
                       int64_t heads, int64_t page, int64_t dim, const int32_t *table, int64_t table_ld, int64_t seqs,
                       int64_t width) {
  if (table_ld < width)
    return fail(DSL_ERR_ARG, "%s: table_ld=%lld < width=%lld", fn, (long long)table_ld, (long long)width);
  int rc;
  if (pages > 0) {
    if ((rc = check_out(fn, k, "k_cache")) || (rc = check_out(fn, v, "v_cache"))) return rc;
    if (!ks || !vs || !aligned(ks, 4) || !aligned(vs, 4))
      return fail(DSL_ERR_ARG, "%s: cache scales are NULL or misaligned", fn);
  }
  if (seqs > 0 && width > 0 && (!table || !aligned(table, 4)))
    return fail(DSL_ERR_ARG, "%s: page table is NULL or misaligned", fn);
  *c = dsl::PageArgs{static_cast<uint8_t *>(k), static_cast<uint8_t *>(v), ks, vs, heads * page * dim, (int)heads};
  return DSL_OK;
}

// An int32 array of n values, 4-byte aligned.
int check_ints(const char *fn, const char *name, const void *x, int64_t n) {
  if (n > 0 && (!x || !aligned(x, 4))) return fail(DSL_ERR_ARG, "%s: %s is NULL or misaligned", fn, name);
  return DSL_OK;
}

int check_workspace(const char *fn, const void *ws, size_t have, size_t need) {
  if (need && (!ws || have < need || !aligned(ws, 16)))
    return fail(DSL_ERR_WORKSPACE, "%s: workspace of %zu bytes (16-B aligned) required", fn, need);
  return DSL_OK;
}

int check_rotary_heads(const char *fn, const char *name, const dsl::RotaryHeads &r, int64_t dim) {
  if (!r.x || !r.y || !aligned(r.x, 2) || !aligned(r.y, 2))
    return fail(DSL_ERR_ARG, "%s: %s or its result is NULL or misaligned", fn, name);
  if (r.row < 0 || r.head < 0 || r.yrow < 0 || r.yhead < 0 || (r.heads > 1 && (r.head < dim || r.yhead < dim)))
    return fail(DSL_ERR_ARG, "%s: strides of %s must be >= 0, heads at least dim apart", fn, name);
  if (r.x == r.y && (r.row != r.yrow || r.head != r.yhead))
    return fail(DSL_ERR_ARG, "%s: %s in place needs the same strides for its result", fn, name);
  return DSL_OK;
}

int logprob_sizes(const char *fn, int64_t rows, int64_t vocab, int64_t top, int x_dtype) {
  if (x_dtype != DSL_IN_BF16 && x_dtype != DSL_IN_F16 && x_dtype != DSL_IN_F32)
    return fail(DSL_ERR_ARG, "%s: unknown x_dtype %d", fn, x_dtype);
  if (rows < 0 || vocab <= 0 || vocab >= kInts)
    return fail(DSL_ERR_ARG, "%s: need rows >= 0 and 0 < vocab < 2^31 (got %lld, %lld)", fn, (long long)rows,
                (long long)vocab);
  if (rows >= 1 << 22) return fail(DSL_ERR_UNSUPPORTED, "%s: rows=%lld: at most 2^22 - 1 in a call", fn, (long long)rows);
  if (top < 0 || top > vocab) return fail(DSL_ERR_ARG, "%s: top=%lld must be 0 .. vocab", fn, (long long)top);
  if (top > dsl::kMaxTop) return fail(DSL_ERR_UNSUPPORTED, "%s: top=%lld > %d", fn, (long long)top, dsl::kMaxTop);
  return DSL_OK;
}
int logprob_src(int x_dtype) {
  return x_dtype == DSL_IN_BF16 ? dsl::SRC_BF16 : (x_dtype == DSL_IN_F16 ? dsl::SRC_F16 : dsl::SRC_F32);
}

}  // namespace

extern "C" {

size_t dsl_kv8_fork_workspace_bytes(int64_t seqs, int64_t width, int64_t children, int64_t pages) {
  if (seqs < 0 || seqs > 65535 || children < 0 || children > 65535 || width < 0 || width >= kInts || pages < 0 ||
      pages >= kInts)
    return 0;
  return dsl::fork_workspace_bytes((int)seqs, (int)width, (int)children, (int)pages);
}

int dsl_kv8_fork(void *k_cache, void *v_cache, float *k_scale, float *v_scale, int64_t pages, int64_t heads,
                 int64_t page, int64_t dim, const int32_t *table, int64_t table_ld, int64_t width,
                 const int32_t *seq_lens, int64_t seqs, const int32_t *parents, const int32_t *more, int64_t more_all,
                 int64_t children, const int32_t *refs, int32_t *out_lens, int32_t *out_table, int32_t *out_refs,
                 int32_t *lacking, void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "dsl_kv8_fork";
  dsl::PageArgs c{};
  int rc = check_pool(fn, pages, heads, page, dim, seqs, width);
  if (rc) return rc;
  if (children < 0) return fail(DSL_ERR_ARG, "%s: children must be >= 0", fn);
  if (children > 65535) return fail(DSL_ERR_UNSUPPORTED, "%s: at most 65535 children in a call", fn);
  if (more_all < 0 || more_all >= kInts) return fail(DSL_ERR_ARG, "%s: need 0 <= new tokens < 2^31", fn);
  if ((rc = check_pool_tensors(fn, &c, k_cache, v_cache, k_scale, v_scale, pages, heads, page, dim, table, table_ld,
                               seqs, width)) ||
      (rc = check_ints(fn, "seq_lens", seq_lens, seqs)) || (rc = check_ints(fn, "parents", parents, children)) ||
      (rc = check_ints(fn, "refs", refs, pages)) || (rc = check_ints(fn, "out_lens", out_lens, children)) ||
      (rc = check_ints(fn, "out_table", out_table, children * width)) ||
      (rc = check_ints(fn, "out_refs", out_refs, pages)) || (rc = check_ints(fn, "lacking", lacking, 1)))
    return rc;
  if (!aligned(more, 4)) return fail(DSL_ERR_ARG, "%s: new tokens are misaligned", fn);
  if (pages > 0 && (refs == out_refs || (seqs > 0 && width > 0 && table == out_table)))
    return fail(DSL_ERR_ARG, "%s: the new table and counts must not be the old ones", fn);
  if ((rc = check_workspace(fn, workspace, workspace_bytes, dsl_kv8_fork_workspace_bytes(seqs, width, children, pages))))
    return rc;
  if (seqs > 0 && children > 0 && seq_lens == out_lens)
    return fail(DSL_ERR_ARG, "%s: the new lengths must not be the old ones", fn);
  dsl::ForkArgs p{};
  p.lens = seq_lens;
  p.table = table;
  p.table_ld = table_ld;
  p.parents = parents;
  p.more = more;
  p.more_all = (int)more_all;
  p.refs = refs;
  p.seqs = (int)seqs;
  p.width = (int)width;
  p.children = (int)children;
  p.pages = (int)pages;
  p.page = (int)page;
  p.out_lens = out_lens;
  p.out_table = out_table;
  p.out_refs = out_refs;
  p.lacking = lacking;
  p.ws = static_cast<int32_t *>(workspace);
  return hip_status(dsl::launch_fork(c, p, static_cast<hipStream_t>(stream)), fn);
}

size_t dsl_kv8_compact_workspace_bytes(int64_t pages) {
  return pages < 0 || pages >= kInts ? 0 : dsl::compact_workspace_bytes((int)pages);
}

int dsl_kv8_compact(void *k_cache, void *v_cache, float *k_scale, float *v_scale, int64_t pages, int64_t heads,
                    int64_t page, int64_t dim, const int32_t *table, int64_t table_ld, int64_t width, int64_t seqs,
                    const int32_t *refs, int32_t *out_table, int32_t *out_refs, int32_t *moved, int32_t *live,
                    void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "dsl_kv8_compact";
  dsl::PageArgs c{};
  int rc = check_pool(fn, pages, heads, page, dim, seqs, width);
  if (rc) return rc;
  if ((rc = check_pool_tensors(fn, &c, k_cache, v_cache, k_scale, v_scale, pages, heads, page, dim, table, table_ld,
                               seqs, width)) ||
      (rc = check_ints(fn, "refs", refs, pages)) || (rc = check_ints(fn, "out_table", out_table, seqs * width)) ||
      (rc = check_ints(fn, "out_refs", out_refs, pages)) || (rc = check_ints(fn, "moved", moved, pages)) ||
      (rc = check_ints(fn, "live", live, 1)))
    return rc;
  if (pages > 0 && refs == out_refs) return fail(DSL_ERR_ARG, "%s: the new counts must not be the old ones", fn);
  if (table == out_table && table_ld != width && seqs > 1 && width > 0)
    return fail(DSL_ERR_ARG, "%s: the table in place needs table_ld = width", fn);
  if ((rc = check_workspace(fn, workspace, workspace_bytes, dsl_kv8_compact_workspace_bytes(pages)))) return rc;
  dsl::CompactArgs p{};
  p.table = table;
  p.table_ld = table_ld;
  p.refs = refs;
  p.seqs = (int)seqs;
  p.width = (int)width;
  p.pages = (int)pages;
  p.out_table = out_table;
  p.out_refs = out_refs;
  p.moved = moved;
  p.live = live;
  p.ws = static_cast<int32_t *>(workspace);
  return hip_status(dsl::launch_compact(c, p, static_cast<hipStream_t>(stream)), fn);
}

int dsl_rotary(const void *q, int64_t q_row, int64_t q_head, int64_t q_heads, const void *k, int64_t k_row,
               int64_t k_head, int64_t k_heads, int64_t rows, int64_t dim, int64_t pairs, const void *positions,
               int positions_64, int64_t positions_ld, int64_t axes, const int32_t *axis_of, const double *freqs,
               float magnitude, int adjacent, int x_dtype, void *q_out, int64_t qo_row, int64_t qo_head, void *k_out,
               int64_t ko_row, int64_t ko_head, void *stream) {
  const char *fn = "dsl_rotary";
  if (x_dtype != DSL_IN_BF16 && x_dtype != DSL_IN_F16)
    return fail(DSL_ERR_ARG, "%s: x_dtype %d must be bf16 or fp16", fn, x_dtype);
  if (rows < 0 || q_heads <= 0 || k_heads < 0 || dim <= 0)
    return fail(DSL_ERR_ARG, "%s: need rows, k_heads >= 0 and q_heads, dim > 0", fn);
  if (dim > 1024 || q_heads > 1 << 16 || k_heads > 1 << 16 || rows >= 1 << 24)
    return fail(DSL_ERR_UNSUPPORTED, "%s: at most 2^24 - 1 rows, 2^16 heads and dim 1024", fn);
  if (pairs < 0 || 2 * pairs > dim) return fail(DSL_ERR_ARG, "%s: need 0 <= 2 x pairs (%lld) <= dim", fn, (long long)pairs);
  if (axes <= 0 || axes > 1 << 20 || positions_ld < rows)
    return fail(DSL_ERR_ARG, "%s: need 1 .. 2^20 axes of positions, rows apart at least", fn);
  if (!axis_of && axes != 1) return fail(DSL_ERR_ARG, "%s: several axes need axis_of", fn);
  if (!(magnitude - magnitude == 0.f)) return fail(DSL_ERR_ARG, "%s: magnitude must be finite", fn);
  if (rows == 0) return ok();
  dsl::RotaryArgs p{};
  p.q = dsl::RotaryHeads{q, q_row, q_head, q_out, qo_row, qo_head, (int)q_heads};
  p.k = dsl::RotaryHeads{k, k_row, k_head, k_out, ko_row, ko_head, (int)k_heads};
  int rc;
  if ((rc = check_rotary_heads(fn, "q", p.q, dim)) || (k_heads > 0 && (rc = check_rotary_heads(fn, "k", p.k, dim))))
    return rc;
  if (pairs > 0) {
    if (!positions || !aligned(positions, positions_64 ? 8 : 4))
      return fail(DSL_ERR_ARG, "%s: positions are NULL or misaligned", fn);
    if (!freqs || !aligned(freqs, 8)) return fail(DSL_ERR_ARG, "%s: freqs is NULL or misaligned", fn);
    if (!aligned(axis_of, 4)) return fail(DSL_ERR_ARG, "%s: axis_of is misaligned", fn);
  }
  p.rows = (int)rows;
  p.dim = (int)dim;
  p.half = (int)pairs;
  p.positions = positions;
  p.pos64 = positions_64 != 0;
  p.pos_ld = positions_ld;
  p.axes = (int)axes;
  p.axis_of = axis_of;
  p.freqs = freqs;
  p.magnitude = magnitude;
  p.adjacent = adjacent != 0;
  return hip_status(dsl::launch_rotary(x_dtype == DSL_IN_BF16 ? dsl::SRC_BF16 : dsl::SRC_F16, p,
                                       static_cast<hipStream_t>(stream)),
                    fn);
}

size_t dsl_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top, int x_dtype) {
  if (logprob_sizes("dsl_token_logprobs_workspace_bytes", rows, vocab, top, x_dtype)) return 0;
  return dsl::logprob_workspace_bytes(logprob_src(x_dtype), (int)rows, (int)vocab, (int)top);
}

int dsl_token_logprobs(const void *logits, int64_t rows, int64_t vocab, int64_t ld, int x_dtype, const int32_t *ids,
                       int64_t ids_ld, int64_t n_ids, float scale, int64_t top, float *logp, float *entropy,
                       float *top_logp, int32_t *top_ids, void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "dsl_token_logprobs";
  int rc = logprob_sizes(fn, rows, vocab, top, x_dtype);
  if (rc) return rc;
  if (ld < vocab && rows > 1) return fail(DSL_ERR_ARG, "%s: ld=%lld < vocab", fn, (long long)ld);
  if (n_ids < 0 || n_ids > 1 << 20 || (ids_ld < n_ids && rows > 1))
    return fail(DSL_ERR_ARG, "%s: need 0 .. 2^20 ids of a row, rows at least as far apart", fn);
  if (!(scale > 0.f && scale < 0x1p126f)) return fail(DSL_ERR_ARG, "%s: scale must be > 0 and below 2^126", fn);
  if (rows == 0) return ok();
  if (!logits || !aligned(logits, x_dtype == DSL_IN_F32 ? 4 : 2))
    return fail(DSL_ERR_ARG, "%s: logits are NULL or misaligned", fn);
  if ((rc = check_ints(fn, "ids", ids, n_ids)) || (rc = check_ints(fn, "logp", logp, n_ids)) ||
      (rc = check_ints(fn, "entropy", entropy, 1)) || (rc = check_ints(fn, "top_logp", top_logp, top)) ||
      (rc = check_ints(fn, "top_ids", top_ids, top)))
    return rc;
  if ((rc = check_workspace(fn, workspace, workspace_bytes,
                            dsl::logprob_workspace_bytes(logprob_src(x_dtype), (int)rows, (int)vocab, (int)top))))
    return rc;
  dsl::LogprobArgs p{};
  p.x = logits;
  p.ld = ld;
  p.rows = (int)rows;
  p.vocab = (int)vocab;
  p.ids = ids;
  p.ids_ld = ids_ld;
  p.n_ids = (int)n_ids;
  p.scale = scale;
  p.top = (int)top;
  p.logp = logp;
  p.entropy = entropy;
  p.top_logp = top_logp;
  p.top_ids = top_ids;
  p.ws = workspace;
  return hip_status(dsl::launch_logprobs(logprob_src(x_dtype), p, static_cast<hipStream_t>(stream)), fn);
}

}  // extern "C"
