// Pieces shared by the attention kernels over the paged 8-bit cache
// (attn.hip: few query rows; attn_prompt.hip: many).
//
// With K codes kc, V codes vc and their page's scales ks, vs:
//   s = (scale ks) (kc . q),  o = sum_t exp(s_t - m) vs_t vc_t / sum_t exp(s_t - m).
// Codes of 8 bits are exact in bf16 and fp16, so both products run on the
// 16-bit matrix instructions over converted codes; the scales act on the
// fp32 scores and on the probabilities.  Everything else is fp32: scores,
// the running maximum m (in powers of two), the sum l and the output.
//
// The probabilities times vs are rounded to bf16 for the second product (an
// error of half a bf16 step of each term, like that of the bf16 result).  For
// fp16 results they enter as two bf16 numbers, hi + lo (16 bits): fp16 has no
// room for probabilities times small scales.
//
// Rows.  The query rows of a sequence and cache head are r = i * group + g:
// new token i, query head g of the group, so heads that share the cache share
// its loads.  The scores are computed transposed, S^T = K Q^T (a lane's column
// is a query row), and tokens are dealt to the rows of the K tiles so that
// the lane that needs a probability for P V holds it already: of a tile of 64
// tokens, row 4a + i of K tile t is token 16a + 4t + i, and lane group a then
// holds 16 consecutive tokens, the 16 bytes of V that it loads.
#pragma once

#include "gemm_core.h"
#include "kv_core.h"

namespace dsl {

// Eight codes as a 16-bit operand: bf16 (F16 false) or fp16.
template <bool FP8, bool F16>
DSL_DEV v4i codes8(uint32_t lo, uint32_t hi) {
  v4i r;
  if constexpr (FP8) {
    if constexpr (F16) {
      r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
      r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
      r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
      r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
    } else {
      r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
      r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
      r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
      r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    }
  } else {
    float f[8];
    code_values<false>(lo, f);
    code_values<false>(hi, f + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (F16) r[i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_pkrtz(f[2 * i], f[2 * i + 1]));
      else r[i] = (int)pack_bf16x2(f[2 * i], f[2 * i + 1]);
    }
  }
  return r;
}

template <bool F16>
DSL_DEV v4f mfma16(const v4i &a, const v4i &b, const v4f &c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

// Maximum / sum over the four lane groups of 16: every lane gets it.
DSL_DEV float groups_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  v = fmaxf(u2f(a[0]), u2f(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(b[0]), u2f(b[1]));
}
DSL_DEV float groups_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  v = u2f(a[0]) + u2f(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
  return u2f(b[0]) + u2f(b[1]);
}

constexpr float kLog2e = 1.44269504088896341f;

}  // namespace dsl
