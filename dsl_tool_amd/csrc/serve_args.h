// Arguments of the kernels of an 8-bit attention layer: the residual norm and
// row quantizers (norm_quant.hip), the paged 8-bit cache (kvcache.hip) and
// attention over it (attn.hip).  Launchers assume arguments were validated.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dsl {

enum { SRC_BF16 = 0, SRC_F16 = 1, SRC_F32 = 2 };
enum { RQ_INT8 = 0, RQ_FP8 = 1, RQ_FP8_G128 = 2 };   // one scale per row (INT8, FP8) or per 128 columns

struct RowQuantArgs {
  const void *x;         // [rows][ldx]
  int64_t ldx;
  const void *r;         // residual [rows][ldr], nullptr: none (norm only)
  int64_t ldr;
  const void *w;         // norm weight [cols], bf16 or fp32 (w_f32)
  bool w_f32;
  void *h;               // x + r [rows][cols] (nullptr: none)
  uint8_t *q;            // codes [rows][cols]
  float *scales;         // [rows], or [rows][ceil(cols/128)]
  int rows, cols;        // cols % 8 == 0, cols <= 32768
  float eps;
};
// Codes of x itself (RQ_INT8; any source type) or of its norm (bf16, fp16).
hipError_t launch_row_quant(int src, const RowQuantArgs &p, hipStream_t st);
hipError_t launch_add_rmsnorm_quant(int src, int fmt, const RowQuantArgs &p, hipStream_t st);

// A paged cache in 8 bits: k [pages][heads][page][dim], v [pages][heads][dim][page],
// one fp32 scale per page and head.
struct KvCacheArgs {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  int64_t pages;
  int heads, page, dim;  // page 16 .. 256, a power of two; dim 64, 128 or 256
  bool fp8;              // E4M3 codes, else int8
  // the sequences: table [seqs][table_ld] page numbers, lens [seqs] tokens
  // (new ones included), starts [seqs + 1] first row of each sequence's new
  // tokens (nullptr: one row per sequence)
  const int32_t *table;
  int64_t table_ld;
  int width;             // pages per table row
  const int32_t *lens, *starts;
  int seqs;
  int rows;              // rows of the token tensors
};

struct KvWriteArgs {
  const void *k, *v;     // [rows][heads][dim], unit stride in dim
  int64_t k_row, k_head, v_row, v_head;
};
hipError_t launch_kv_write(int src, const KvCacheArgs &c, const KvWriteArgs &p, hipStream_t st);

struct KvReadArgs {
  void *k, *v;           // [rows][heads][dim]
};
hipError_t launch_kv_read(int src, const KvCacheArgs &c, const KvReadArgs &p, hipStream_t st);

struct AttnArgs {
  const void *q;         // [rows][q_heads][dim], unit stride in dim
  int64_t q_row, q_head;
  void *o;
  int64_t o_row, o_head;
  int q_heads, group;    // group = q_heads / heads
  int max_q;             // most new tokens of a sequence (sizes the launch)
  float scale;
  bool causal;
  float *ws;             // partial results of a split context
};
size_t attn_workspace_bytes(const KvCacheArgs &c, int q_heads, int max_q);
// Many query rows (attn_prompt.hip): blocks of attn_prompt_rows(dim) rows, nblk of
// them per sequence and head (each walks every nblk-th); the context in nsplit parts
// of `part` tokens.
int attn_prompt_rows(int dim);
constexpr int kPromptThreads = 512;              // of a workgroup
hipError_t launch_attn_prompt(int src, const KvCacheArgs &c, const AttnArgs &p, int nblk, int nsplit, int part, hipStream_t st);
hipError_t launch_attn(int src, const KvCacheArgs &c, const AttnArgs &p, hipStream_t st);

// Groups of sequences that share a prefix (attn_shared.hip): sequences groups[g] ..
// groups[g + 1] - 1 hold the same pages for their first shared[g] tokens.
struct SharedArgs {
  const int32_t *groups, *shared;        // [n + 1], [n]
  int n;
  int most;              // most sequences of a group (sizes the launch)
};
bool attn_shared_runs(int heads, int dim, int q_heads, int max_q);      // or the call goes to launch_attn
size_t attn_shared_workspace_bytes(const KvCacheArgs &c, int groups, int q_heads, int max_q, int max_group);
hipError_t launch_attn_shared(int src, const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, hipStream_t st);

}  // namespace dsl
