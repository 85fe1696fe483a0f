// extern "C" entry points of the 8-bit attention layer, declared in
// include/dsl_gemm.h: the int8 product, the residual norm, int8 row codes, the paged 8-bit cache
// and attention over it.  As in capi.hip, everything is validated on the host
// before anything is enqueued, and nothing is allocated.
#include "capi_util.h"
#include "serve_args.h"

using namespace dsl::capi;

namespace {

int src_of(int x_dtype) {
  return x_dtype == DSL_IN_BF16 ? dsl::SRC_BF16 : (x_dtype == DSL_IN_F16 ? dsl::SRC_F16 : dsl::SRC_F32);
}

int check_rows(const char *fn, const char *name, int64_t rows, int64_t cols, int64_t ld) {
  if (rows < 0 || cols <= 0 || rows >= (int64_t)1 << 31)
    return fail(DSL_ERR_ARG, "%s: need 0 <= rows < 2^31 and cols > 0 (got %lld, %lld)", fn, (long long)rows,
                (long long)cols);
  if (cols % 8 != 0) return fail(DSL_ERR_ARG, "%s: cols=%lld must be a multiple of 8", fn, (long long)cols);
  if (cols > 32768)
    return fail(DSL_ERR_UNSUPPORTED, "%s: cols=%lld > 32768 (one workgroup holds a row)", fn, (long long)cols);
  if (ld < cols || ld % 8 != 0)
    return fail(DSL_ERR_ARG, "%s: %s=%lld must be >= cols and a multiple of 8", fn, name, (long long)ld);
  return DSL_OK;
}

// The sizes of a call: what the kernels and their plans hold in ints.
int check_sizes(const char *fn, int64_t heads, int64_t page, int64_t dim, int64_t width, int64_t seqs, int64_t rows) {
  if (heads <= 0 || seqs < 0 || rows < 0 || width < 0)
    return fail(DSL_ERR_ARG, "%s: need pages, seqs, rows, width >= 0 and heads > 0", fn);
  if (rows >= (int64_t)1 << 31) return fail(DSL_ERR_ARG, "%s: pages and rows must be < 2^31", fn);
  if (dim != 64 && dim != 128 && dim != 256)
    return fail(DSL_ERR_UNSUPPORTED, "%s: head dim %lld must be 64, 128 or 256", fn, (long long)dim);
  if (page != 16 && page != 32 && page != 64 && page != 128 && page != 256)
    return fail(DSL_ERR_UNSUPPORTED, "%s: page size %lld must be 16, 32, 64, 128 or 256", fn, (long long)page);
  if (heads > 16384 || seqs > 65535)
    return fail(DSL_ERR_UNSUPPORTED, "%s: at most 16384 heads and 65535 sequences in a call", fn);
  // tokens are counted in ints, whole tiles beyond a sequence's last one included
  if (width > (((int64_t)1 << 31) - 65536) / page)
    return fail(DSL_ERR_ARG, "%s: page table rows span more than 2^31 - 65536 tokens", fn);
  return DSL_OK;
}
int check_q_heads(const char *fn, int64_t q_heads, int64_t heads, int64_t rows, int64_t max_q) {
  if (q_heads <= 0 || q_heads % heads != 0 || q_heads > 1 << 20)
    return fail(DSL_ERR_ARG, "%s: q_heads=%lld must be a multiple of heads=%lld", fn, (long long)q_heads,
                (long long)heads);
  if (max_q < 0) return fail(DSL_ERR_ARG, "%s: max_q must be >= 0", fn);
  if (rows > ((int64_t)1 << 30) / q_heads) return fail(DSL_ERR_ARG, "%s: rows x query heads must be at most 2^30", fn);
  return DSL_OK;
}

// The cache and the sequences of a call, checked and packed.
int check_cache(const char *fn, dsl::KvCacheArgs *c, const void *k, const void *v, const float *ks, const float *vs,
                int64_t pages, int64_t heads, int64_t page, int64_t dim, int fmt, const int32_t *table,
                int64_t table_ld, int64_t width, const int32_t *lens, const int32_t *starts, int64_t seqs,
                int64_t rows, int x_dtype) {
  if (pages < 0) return fail(DSL_ERR_ARG, "%s: need pages, seqs, rows, width >= 0 and heads > 0", fn);
  if (pages >= (int64_t)1 << 31) return fail(DSL_ERR_ARG, "%s: pages and rows must be < 2^31", fn);
  if (const int rc = check_sizes(fn, heads, page, dim, width, seqs, rows)) return rc;
  if (fmt != DSL_KV_INT8 && fmt != DSL_KV_FP8) return fail(DSL_ERR_ARG, "%s: unknown fmt %d", fn, fmt);
  if (x_dtype != DSL_IN_BF16 && x_dtype != DSL_IN_F16)
    return fail(DSL_ERR_ARG, "%s: x_dtype %d must be bf16 or fp16", fn, x_dtype);
  if (table_ld < width) return fail(DSL_ERR_ARG, "%s: table_ld=%lld < width=%lld", fn, (long long)table_ld,
                                    (long long)width);
  if (!starts && rows != seqs)
    return fail(DSL_ERR_ARG, "%s: without starts, rows (%lld) must be seqs (%lld)", fn, (long long)rows,
                (long long)seqs);
  if (rows > 0 && seqs > 0) {
    int rc;
    if (pages > 0) {
      if ((rc = check_out(fn, k, "k_cache")) || (rc = check_out(fn, v, "v_cache"))) return rc;
      if (!ks || !vs || !aligned(ks, 4) || !aligned(vs, 4))
        return fail(DSL_ERR_ARG, "%s: cache scales are NULL or misaligned", fn);
    }
    if (!lens || (width > 0 && !table)) return fail(DSL_ERR_ARG, "%s: seq_lens or page table is NULL", fn);
    if (!aligned(lens, 4) || !aligned(table, 4) || !aligned(starts, 4))
      return fail(DSL_ERR_ARG, "%s: int32 arrays must be 4-byte aligned", fn);
  }
  c->k = static_cast<uint8_t *>(const_cast<void *>(k));
  c->v = static_cast<uint8_t *>(const_cast<void *>(v));
  c->k_scale = const_cast<float *>(ks);
  c->v_scale = const_cast<float *>(vs);
  c->pages = pages;
  c->heads = (int)heads;
  c->page = (int)page;
  c->dim = (int)dim;
  c->fp8 = fmt == DSL_KV_FP8;
  c->table = table;
  c->table_ld = table_ld;
  c->width = pages > 0 ? (int)width : 0;         // no pages: every token is in none
  c->lens = lens;
  c->starts = starts;
  c->seqs = (int)seqs;
  c->rows = (int)rows;
  return DSL_OK;
}

// A [rows][heads][dim] tensor read or written in 16-byte words.
int check_heads(const char *fn, const char *name, const void *x, int64_t row, int64_t head, int64_t heads, int64_t dim) {
  int rc = check_out(fn, x, name);
  if (rc) return rc;
  if (row % 8 != 0 || head % 8 != 0 || head < (heads > 1 ? dim : 0) || row < 0)
    return fail(DSL_ERR_ARG, "%s: strides of %s (%lld, %lld) must be multiples of 8, heads at least dim apart", fn,
                name, (long long)row, (long long)head);
  return DSL_OK;
}

}  // namespace

extern "C" {

int dsl_int8_gemm(const int8_t *a, const int8_t *b, void *c, int64_t m, int64_t n, int64_t k, int64_t ldc,
                  int out_dtype, const float *scale_a, const float *scale_b, void *stream) {
  const char *fn = "dsl_int8_gemm";
  int rc = check_gemm_dims(fn, m, n, k, ldc, 16, out_dtype);
  if (rc) return rc;
  if (k >= 1 << 17) return fail(DSL_ERR_UNSUPPORTED, "%s: k=%lld: int32 sums hold k < 131072", fn, (long long)k);
  if (m == 0 || n == 0) return ok();
  if ((rc = check_out(fn, a, "a")) || (rc = check_out(fn, b, "b"))) return rc;
  if (!c || !aligned(c, out_dtype == DSL_OUT_F32 ? 4 : 2)) return fail(DSL_ERR_ARG, "%s: c is NULL or misaligned", fn);
  if (!scale_a || !scale_b || !aligned(scale_a, 4) || !aligned(scale_b, 4))
    return fail(DSL_ERR_ARG, "%s: scales are NULL or misaligned", fn);
  dsl::GemmArgs p{};
  p.a = reinterpret_cast<const uint8_t *>(a);
  p.b = reinterpret_cast<const uint8_t *>(b);
  p.c = c;
  p.M = (int)m;
  p.N = (int)n;
  p.K = p.Kb = (int)k;
  p.ldc = ldc;
  p.sa = scale_a;
  p.sb = scale_b;
  p.ksplit = 1;
  p.out_f32 = out_dtype == DSL_OUT_F32;
  return hip_status(dsl::launch_gemm(dsl::MODE_INT8, p, static_cast<hipStream_t>(stream)), fn);
}

int dsl_quant_int8_rows(const void *x, int64_t rows, int64_t cols, int64_t ldx, int x_dtype, int8_t *q,
                        float *scales, void *stream) {
  const char *fn = "dsl_quant_int8_rows";
  if (x_dtype != DSL_IN_BF16 && x_dtype != DSL_IN_F16 && x_dtype != DSL_IN_F32)
    return fail(DSL_ERR_ARG, "%s: unknown x_dtype %d", fn, x_dtype);
  int rc = check_rows(fn, "ldx", rows, cols, ldx);
  if (rc) return rc;
  if (rows == 0) return ok();
  if ((rc = check_out(fn, x, "x")) || (rc = check_out(fn, q, "q"))) return rc;
  if (!scales || !aligned(scales, 4)) return fail(DSL_ERR_ARG, "%s: scales is NULL or misaligned", fn);
  dsl::RowQuantArgs p{};
  p.x = x;
  p.ldx = ldx;
  p.q = reinterpret_cast<uint8_t *>(q);
  p.scales = scales;
  p.rows = (int)rows;
  p.cols = (int)cols;
  return hip_status(dsl::launch_row_quant(src_of(x_dtype), p, static_cast<hipStream_t>(stream)), fn);
}

int dsl_add_rmsnorm_quant(const void *x, int64_t rows, int64_t cols, int64_t ldx, const void *residual, int64_t ldr,
                          const void *weight, int weight_dtype, float eps, int x_dtype, int qfmt, void *h, void *q,
                          float *scales, void *stream) {
  const char *fn = "dsl_add_rmsnorm_quant";
  if (x_dtype != DSL_IN_BF16 && x_dtype != DSL_IN_F16)
    return fail(DSL_ERR_ARG, "%s: x_dtype %d must be bf16 or fp16", fn, x_dtype);
  if (qfmt != DSL_ROWQ_INT8 && qfmt != DSL_ROWQ_FP8 && qfmt != DSL_ROWQ_FP8_G128)
    return fail(DSL_ERR_ARG, "%s: unknown qfmt %d", fn, qfmt);
  if (weight_dtype != DSL_W_BF16 && weight_dtype != DSL_W_F32)
    return fail(DSL_ERR_ARG, "%s: unknown weight dtype %d", fn, weight_dtype);
  if (!(eps >= 0.f)) return fail(DSL_ERR_ARG, "%s: eps must be >= 0", fn);
  int rc = check_rows(fn, "ldx", rows, cols, ldx);
  if (!rc && residual) rc = check_rows(fn, "ldr", rows, cols, ldr);
  if (rc) return rc;
  if (rows == 0) return ok();
  if ((rc = check_out(fn, x, "x")) || (rc = check_out(fn, weight, "weight")) || (rc = check_out(fn, q, "q"))) return rc;
  if (residual && (rc = check_out(fn, residual, "residual"))) return rc;
  if (h && (rc = check_out(fn, h, "h"))) return rc;
  if (!scales || !aligned(scales, 4)) return fail(DSL_ERR_ARG, "%s: scales is NULL or misaligned", fn);
  dsl::RowQuantArgs p{};
  p.x = x;
  p.ldx = ldx;
  p.r = residual;
  p.ldr = ldr;
  p.w = weight;
  p.w_f32 = weight_dtype == DSL_W_F32;
  p.h = h;
  p.q = static_cast<uint8_t *>(q);
  p.scales = scales;
  p.rows = (int)rows;
  p.cols = (int)cols;
  p.eps = eps;
  const int fmt = qfmt == DSL_ROWQ_INT8 ? dsl::RQ_INT8 : (qfmt == DSL_ROWQ_FP8 ? dsl::RQ_FP8 : dsl::RQ_FP8_G128);
  return hip_status(dsl::launch_add_rmsnorm_quant(src_of(x_dtype), fmt, p, static_cast<hipStream_t>(stream)), fn);
}

int dsl_kv8_write(void *k_cache, void *v_cache, float *k_scale, float *v_scale, int64_t pages, int64_t heads,
                  int64_t page, int64_t dim, int fmt, const int32_t *table, int64_t table_ld, int64_t width,
                  const int32_t *seq_lens, const int32_t *starts, int64_t seqs, const void *k, int64_t k_row,
                  int64_t k_head, const void *v, int64_t v_row, int64_t v_head, int64_t rows, int64_t max_q,
                  int x_dtype, void *stream) {
  const char *fn = "dsl_kv8_write";
  dsl::KvCacheArgs c{};
  int rc = check_cache(fn, &c, k_cache, v_cache, k_scale, v_scale, pages, heads, page, dim, fmt, table, table_ld,
                       width, seq_lens, starts, seqs, rows, x_dtype);
  if (rc) return rc;
  if (max_q < 0) return fail(DSL_ERR_ARG, "%s: max_q must be >= 0", fn);
  if (rows == 0 || seqs == 0) return ok();
  if ((rc = check_heads(fn, "k", k, k_row, k_head, heads, dim)) ||
      (rc = check_heads(fn, "v", v, v_row, v_head, heads, dim)))
    return rc;
  const dsl::KvWriteArgs p{k, v, k_row, k_head, v_row, v_head};
  return hip_status(dsl::launch_kv_write(src_of(x_dtype), c, p, static_cast<hipStream_t>(stream)), fn);
}

int dsl_kv8_read(const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale, int64_t pages,
                 int64_t heads, int64_t page, int64_t dim, int fmt, const int32_t *table, int64_t table_ld,
                 int64_t width, const int32_t *seq_lens, const int32_t *starts, int64_t seqs, void *k, void *v,
                 int64_t rows, int out_dtype, void *stream) {
  const char *fn = "dsl_kv8_read";
  dsl::KvCacheArgs c{};
  if (!starts && rows > 0) return fail(DSL_ERR_ARG, "%s: starts is NULL", fn);
  int rc = check_cache(fn, &c, k_cache, v_cache, k_scale, v_scale, pages, heads, page, dim, fmt, table, table_ld,
                       width, seq_lens, starts, seqs, rows, out_dtype);
  if (rc) return rc;
  if (rows == 0 || seqs == 0) return ok();
  if ((rc = check_out(fn, k, "k")) || (rc = check_out(fn, v, "v"))) return rc;
  return hip_status(dsl::launch_kv_read(src_of(out_dtype), c, dsl::KvReadArgs{k, v}, static_cast<hipStream_t>(stream)),
                    fn);
}

size_t dsl_kv8_attention_workspace_bytes(int64_t heads, int64_t page, int64_t dim, int64_t width, int64_t seqs,
                                         int64_t rows, int64_t q_heads, int64_t max_q) {
  const char *fn = "dsl_kv8_attention_workspace_bytes";
  if (check_sizes(fn, heads, page, dim, width, seqs, rows) || check_q_heads(fn, q_heads, heads, rows, max_q)) return 0;
  if (rows == 0 || seqs == 0) return 0;
  dsl::KvCacheArgs c{};
  c.heads = (int)heads;
  c.page = (int)page;
  c.dim = (int)dim;
  c.width = (int)width;
  c.seqs = (int)seqs;
  c.rows = (int)rows;
  return dsl::attn_workspace_bytes(c, (int)q_heads, (int)(max_q < rows ? max_q : rows));
}

int dsl_kv8_attention(const void *q, int64_t q_row, int64_t q_head, int64_t q_heads, const void *k_cache,
                      const void *v_cache, const float *k_scale, const float *v_scale, int64_t pages, int64_t heads,
                      int64_t page, int64_t dim, int fmt, const int32_t *table, int64_t table_ld, int64_t width,
                      const int32_t *seq_lens, const int32_t *starts, int64_t seqs, void *out, int64_t o_row,
                      int64_t o_head, int64_t rows, int64_t max_q, float scale, int causal, int x_dtype,
                      void *workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "dsl_kv8_attention";
  dsl::KvCacheArgs c{};
  int rc = check_cache(fn, &c, k_cache, v_cache, k_scale, v_scale, pages, heads, page, dim, fmt, table, table_ld,
                       width, seq_lens, starts, seqs, rows, x_dtype);
  if (rc) return rc;
  if ((rc = check_q_heads(fn, q_heads, heads, rows, max_q))) return rc;
  if (!(scale - scale == 0.f)) return fail(DSL_ERR_ARG, "%s: scale must be finite", fn);
  if (rows == 0 || seqs == 0) return ok();
  if ((rc = check_heads(fn, "q", q, q_row, q_head, q_heads, dim)) ||
      (rc = check_heads(fn, "out", out, o_row, o_head, q_heads, dim)))
    return rc;
  dsl::AttnArgs p{};
  p.q = q;
  p.q_row = q_row;
  p.q_head = q_head;
  p.o = out;
  p.o_row = o_row;
  p.o_head = o_head;
  p.q_heads = (int)q_heads;
  p.group = (int)(q_heads / heads);
  p.max_q = (int)(max_q < rows ? max_q : rows);
  p.scale = scale;
  p.causal = causal != 0;
  p.ws = static_cast<float *>(workspace);
  // (the plan depends on the sizes alone, so the query gives the same one)
  const size_t need = dsl_kv8_attention_workspace_bytes(heads, page, dim, c.width, seqs, rows, q_heads, max_q);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(DSL_ERR_WORKSPACE, "%s: workspace of %zu bytes (16-B aligned) required", fn, need);
  return hip_status(dsl::launch_attn(src_of(x_dtype), c, p, static_cast<hipStream_t>(stream)), fn);
}

}  // extern "C"
