// Codes of the paged 8-bit cache and its sequences, shared by the kernels that
// write, read and attend over it (kvcache.hip, attn.hip, attn_prompt.hip).
//
// Page p, head h: keys k[p][h][token][dim] and values v[p][h][dim][token], so
// that both lie along the dimension that attention's products sum over (dim
// for the scores, tokens for the output) and both feed matrix instructions
// without a transpose.  A code c stands for c * scale[p][h].
#pragma once

#include "common.h"
#include "serve_args.h"

namespace dsl {

// One element of a 16-bit row, widened.
template <int SRC>
DSL_DEV float widen(uint16_t b) {
  if constexpr (SRC == SRC_BF16) return bf16_to_f32(b);
  else return (float)__builtin_bit_cast(_Float16, b);
}
template <int SRC>
DSL_DEV uint32_t narrow2(float a, float b) {
  if constexpr (SRC == SRC_BF16) return pack_bf16x2(a, b);
  else return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
}
template <int SRC>
DSL_DEV void widen8s(const uint4 &v, float *f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = widen<SRC>((uint16_t)w[i]);
    f[2 * i + 1] = widen<SRC>((uint16_t)(w[i] >> 16));
  }
}

// The values of four codes.
template <bool FP8>
DSL_DEV void code_values(uint32_t w, float *f) {
  if constexpr (FP8) {
    f[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
    f[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
    f[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
    f[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
  } else {
    f[0] = (float)(int8_t)w;
    f[1] = (float)(int8_t)(w >> 8);
    f[2] = (float)(int8_t)(w >> 16);
    f[3] = (float)(int8_t)(w >> 24);
  }
}

// The codes of four quotients, the first in the low byte.
template <bool FP8>
DSL_DEV uint32_t codes_pack(float a, float b, float c, float d) {
  if constexpr (FP8) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
  } else {
    const uint32_t ia = (uint32_t)(int)__builtin_rintf(a), ib = (uint32_t)(int)__builtin_rintf(b);
    const uint32_t ic = (uint32_t)(int)__builtin_rintf(c), id = (uint32_t)(int)__builtin_rintf(d);
    return __builtin_amdgcn_perm(ib, ia, 0x0c0c0400u) | __builtin_amdgcn_perm(id, ic, 0x04000c0cu);
  }
}

constexpr float kInt8Top = 127.0f;
template <bool FP8>
DSL_DEV float kv_scale_of(float amax) {
  return fmaxf(__fdiv_rn(amax, FP8 ? kE4M3Max : kInt8Top), kScaleFloor);
}

// A sequence's new tokens: n rows from row0 of the token tensors, at positions
// first .. first + n - 1 = len - 1.  Starts are held to the tensors' rows
// whatever the table says; first < 0 where there are more rows than tokens.
struct SeqView {
  int len, first, n, row0;
};
DSL_DEV SeqView seq_view(const KvCacheArgs &c, int b) {
  SeqView s;
  const int len = c.lens[b];
  s.len = len > 0 ? len : 0;
  if (c.starts) {
    const int lo = c.starts[b], hi = c.starts[b + 1];
    s.row0 = lo < 0 ? 0 : (lo > c.rows ? c.rows : lo);
    const int end = hi > c.rows ? c.rows : hi;
    s.n = end > s.row0 ? end - s.row0 : 0;
  } else {
    s.row0 = b;
    s.n = b < c.rows ? 1 : 0;
  }
  s.first = s.len - s.n;
  return s;
}

// The sequence b that item `id` of a flat launch belongs to (-1: none), and the
// item's number in it.  Sequence b's items begin at first(row, b), row its first
// row: floor(row / span) + extra * b.  As floor((s + n) / span) >= floor(s / span)
// + floor(n / span), a sequence of n rows has at least floor(n / span) + extra
// items of its own, and rows / span + extra * seqs suffice for all: few workgroups
// of a ragged batch find nothing to do, whatever its longest sequence.  All lanes
// search, 64 sequences a step, and the last step has the sequence's other numbers
// with its start.  Without starts an item is a sequence.
template <class F>
DSL_DEV SeqView item_seq(const KvCacheArgs &c, int id, const F &first, int &b, int &item) {
  SeqView s{0, 0, 0, 0};
  if (!c.starts) {
    b = id < c.seqs ? id : -1;
    item = 0;
    return b < 0 ? s : seq_view(c, b);
  }
  const int lane = threadIdx.x & 63;
  auto row = [&](int i) {
    const int v = c.starts[i];
    return v < 0 ? 0 : v > c.rows ? c.rows : v;
  };
  int lo = 0, n = c.seqs;
  while (n > 64) {
    const int step = (n + 63) >> 6, off = lane * step;
    const int f = off < n ? first(row(lo + off), lo + off) : 0;
    const int cnt = __popcll(__ballot(off < n && f <= id)), skip = (cnt > 0 ? cnt - 1 : 0) * step;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  const int at = lo + (lane < n ? lane : n - 1);
  const int from = row(at), to = row(at + 1), len = c.lens[at];
  const int f = first(from, at);
  const int cnt = __popcll(__ballot(lane < n && f <= id)), pick = cnt > 0 ? cnt - 1 : 0;
  b = cnt > 0 ? lo + pick : -1;
  item = id - __shfl(f, pick);
  s.len = __shfl(len, pick);
  s.len = s.len > 0 ? s.len : 0;
  s.row0 = __shfl(from, pick);
  s.n = __shfl(to, pick) - s.row0;
  s.n = s.n > 0 ? s.n : 0;
  s.first = s.len - s.n;
  return s;
}

// The page that holds the tokens [page * pg, ..) of sequence b, or -1: pages
// past the table's row and numbers out of range hold none.
DSL_DEV int64_t page_of(const KvCacheArgs &c, int b, int pg) {
  if (pg >= c.width) return -1;
  const int64_t pid = c.table[(int64_t)b * c.table_ld + pg];
  return pid >= 0 && pid < c.pages ? pid : -1;
}

}  // namespace dsl
