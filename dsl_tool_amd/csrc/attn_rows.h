// The walk of few query rows over a context (attn.hip, attn_shared.hip): four
// waves take every fourth tile of 64 tokens, codes straight from memory into
// registers, and join in LDS.  attn_core.h has the mathematics and the row order.
#pragma once

#include "attn_core.h"

namespace dsl {

constexpr int kTile = 64;      // tokens per step of a wave
// Workgroups of a CU: what its registers hold.
constexpr int rows_wgs(int dim, int rb) { return dim * rb <= 128 ? 2 : 1; }

// The sum of a wave's values up to and with each lane's.
DSL_DEV int lanes_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// The NaN codes (E4M3: 0x7f, 0xff) of four, as bytes of ones.
DSL_DEV uint32_t nan_bytes(uint32_t w) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu; }
constexpr uint32_t kOnes = 0x38383838u;          // 1.0 four times

// Tokens 0 .. len - 1 of a sequence, by its row of the page table.
struct Context {
  const int32_t *table;
  int width, len;
};

// RB blocks of 16 query rows share every load.  A lane's row of block k sees
// the tokens before limit[k]; all rows of the workgroup see those before lo, and
// `causal` says that rows may differ.  Tiles t0 .. t1 - 1, every fourth of a wave.
template <bool F16, bool FP8, int D, int RB>
struct RowsWalk {
  static constexpr int NW = 4, DT = D / 16, DC = D / 64, ROWS = 16 * RB;
  v4i qf[RB][2 * DC];
  int limit[RB];
  v4f o[RB][DT];
  float m[RB], l[RB];
  DSL_DEV void walk(const KvCacheArgs &c, const Context &ctx, float scale, bool causal, int head, int t0, int t1, int lo);
};

template <bool F16, bool FP8, int D, int RB>
DSL_DEV void RowsWalk<F16, FP8, D, RB>::walk(const KvCacheArgs &c, const Context &ctx, float scale, bool causal,
                                             int head, int t0, int t1, int lo) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int ktok = 16 * (r16 >> 2) + (r16 & 3);  // the lane's token of K tile 0 (tile t: + 4 t)
  const int P = c.page;
  const int64_t hstride = (int64_t)P * D;
#pragma unroll
  for (int k = 0; k < RB; ++k) {
    m[k] = -INFINITY;
    l[k] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[k][d] = (v4f){0.f, 0.f, 0.f, 0.f};
  }

  // pages of a tile: the lane's key row, and its 16 tokens (V, scales)
  // (what the table and the scales hold past the last token's page is not read)
  auto page = [&](int tok) -> int64_t {
    if (tok >= ctx.len || tok / P >= ctx.width) return -1;
    const int64_t pid = ctx.table[tok / P];
    return pid >= 0 && pid < c.pages ? pid : -1;
  };
  auto kpage = [&](int tile) { return page(tile * kTile + 16 * (r16 >> 2)); };
  auto vpage = [&](int tile) { return page(tile * kTile + 16 * g); };
  uint4 kr[4][DC];
  auto load_k = [&](int tile, int64_t pid) {
    const uint8_t *base = c.k + ((pid < 0 ? 0 : pid) * c.heads + head) * hstride +
                          (int64_t)((tile * kTile + ktok) & (P - 1)) * D + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int x = 0; x < DC; ++x)
        kr[t][x] = *reinterpret_cast<const uint4 *>(base + 4 * t * D + 64 * x);
  };
  int tile = t0 + wave;
  int64_t kp = -1, vp = -1;
  if (tile < t1) {
    kp = kpage(tile);
    vp = vpage(tile);
    load_k(tile, kp);
  }
  for (; tile < t1; tile += NW) {
    const int64_t va = (vp < 0 ? 0 : vp) * c.heads + head;
    const float ks = vp < 0 ? 0.f : c.k_scale[va] * (scale * kLog2e);
    const float vs = vp < 0 ? 0.f : c.v_scale[va];
    uint4 vr[DT];
    const uint8_t *vb = c.v + va * hstride + ((tile * kTile + 16 * g) & (P - 1)) + (int64_t)r16 * P;
#pragma unroll
    for (int d = 0; d < DT; ++d) vr[d] = *reinterpret_cast<const uint4 *>(vb + (int64_t)d * 16 * P);
    const bool last = tile + NW >= t1;
    const int64_t kn = last ? -1 : kpage(tile + NW), vn = last ? -1 : vpage(tile + NW);

    v4f sc[RB][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int k = 0; k < RB; ++k) sc[k][t] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < DC; ++x) {
        const v4i a0 = codes8<FP8, F16>(kr[t][x].x, kr[t][x].y), a1 = codes8<FP8, F16>(kr[t][x].z, kr[t][x].w);
#pragma unroll
        for (int k = 0; k < RB; ++k) {
          sc[k][t] = mfma16<F16>(a0, qf[k][2 * x], sc[k][t]);
          sc[k][t] = mfma16<F16>(a1, qf[k][2 * x + 1], sc[k][t]);
        }
      }
    }
    if (!last) load_k(tile + NW, kn);

    // some token of the tile is hidden from some row, or in no page
    const int pos = tile * kTile + 16 * g;
    const bool masked = tile * kTile + kTile > lo || __any(vp < 0);
    if (masked && FP8) {
      // codes past the end can be NaN; probability 0 does not remove it
      int nv = ctx.len - pos;
      nv = vp < 0 || nv < 0 ? 0 : (nv > 16 ? 16 : nv);
      uint32_t keep[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int n = nv - 4 * w;
        keep[w] = n >= 4 ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * n)) - 1);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        vr[d].x &= keep[0];
        vr[d].y &= keep[1];
        vr[d].z &= keep[2];
        vr[d].w &= keep[3];
      }
    }
    if (FP8 && masked && causal) {
      // a NaN code among new tokens that only some rows see: it leaves the
      // products, and the rows that see it get it by the count of such codes
      bool any = false;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        any |= (nan_bytes(vr[d].x) | nan_bytes(vr[d].y) | nan_bytes(vr[d].z) | nan_bytes(vr[d].w)) != 0;
      if (__any(any)) {
        v4i vis[RB][2];
#pragma unroll
        for (int k = 0; k < RB; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int tok = pos + 8 * h + 2 * w;
              vis[k][h][w] = (tok < limit[k] ? 0x3f80 : 0) | (tok + 1 < limit[k] ? 0x3f800000 : 0);
            }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const uint32_t n0 = nan_bytes(vr[d].x), n1 = nan_bytes(vr[d].y), n2 = nan_bytes(vr[d].z), n3 = nan_bytes(vr[d].w);
          vr[d].x &= ~n0;
          vr[d].y &= ~n1;
          vr[d].z &= ~n2;
          vr[d].w &= ~n3;
          const v4i a0 = codes8<true, false>(n0 & kOnes, n1 & kOnes), a1 = codes8<true, false>(n2 & kOnes, n3 & kOnes);
#pragma unroll
          for (int k = 0; k < RB; ++k) {
            const v4f nans = mfma16<false>(a1, vis[k][1], mfma16<false>(a0, vis[k][0], (v4f){0.f, 0.f, 0.f, 0.f}));
            // (A choice, not a branch: with one, twice the scalar registers spill, and calls
            // of 128 columns take 2 to 4% longer: 64 sequences of 2000 tokens, 8 heads, 42.5 us
            // and 43.1, 32 of 1000 and four new ones 22.6 and 23.2.)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[k][d][i] = nans[i] != 0.f ? __builtin_nanf("") : o[k][d][i];
          }
        }
      }
    }
    v4i pf[RB][2], pl[RB][2];                  // P, tokens 8h .. 8h+7 of the lane's 16 (pl: fp16's low parts)
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = sc[k][t][i] * ks;
          if (masked) v = pos + 4 * t + i < limit[k] && vp >= 0 ? v : -INFINITY;
          sc[k][t][i] = v;
          top = fmaxf(top, v);
        }
      top = fmaxf(groups_max(top), m[k]);
      const float ref = top == -INFINITY ? 0.f : top;   // nothing seen yet
      const float alpha = __builtin_amdgcn_exp2f(m[k] - ref);
      m[k] = top;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(sc[k][t][i] - ref);
          sum += e;
          sc[k][t][i] = e * vs;
        }
      if (masked) {                            // whatever a hidden token's scale is
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(pos + 4 * t + i < limit[k])) sc[k][t][i] = 0.f;
      }
      l[k] = l[k] * alpha + sum;
      if (__any(alpha != 1.f)) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[k][d] *= alpha;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float a = sc[k][2 * h + (w >> 1)][2 * (w & 1)], z = sc[k][2 * h + (w >> 1)][2 * (w & 1) + 1];
          const uint32_t hi = pack_bf16x2(a, z);
          pf[k][h][w] = (int)hi;
          if constexpr (F16) pl[k][h][w] = (int)pack_bf16x2(a - u2f(hi << 16), z - u2f(hi & 0xffff0000u));
        }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const v4i a0 = codes8<FP8, false>(vr[d].x, vr[d].y), a1 = codes8<FP8, false>(vr[d].z, vr[d].w);
#pragma unroll
      for (int k = 0; k < RB; ++k) {
        o[k][d] = mfma16<false>(a0, pf[k][0], o[k][d]);
        o[k][d] = mfma16<false>(a1, pf[k][1], o[k][d]);
        if constexpr (F16) {
          o[k][d] = mfma16<false>(a0, pl[k][0], o[k][d]);
          o[k][d] = mfma16<false>(a1, pl[k][1], o[k][d]);
        }
      }
    }
    kp = kn;
    vp = vn;
  }
}

// The waves' shares of a workgroup's rows, joined: common maximum, then one row-major tile
// per wave.  emit(block, row, column, sums of 4 columns, maximum, sum).
template <int D>
struct RowsJoin {
  static constexpr int NW = 4, LD = D + 4;       // floats per row of the joined tile
  float so[NW][16 * LD], sm[NW][16], sl[NW][16];
};
template <int D, int RB, class Walk, class F>
DSL_DEV void join_rows(RowsJoin<D> &sh, const Walk &w_, int rows, const F &emit) {
  constexpr int NW = 4, DT = D / 16, LD = RowsJoin<D>::LD;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  #pragma unroll
  for (int k = 0; k < RB; ++k) {
    const float lw = groups_sum(w_.l[k]);
    __syncthreads();                           // the last block's readers
    if (g == 0) {
      sh.sm[wave][r16] = w_.m[k];
      sh.sl[wave][r16] = lw;
    }
    __syncthreads();
    float top = sh.sm[0][r16];
#pragma unroll
    for (int w = 1; w < NW; ++w) top = fmaxf(top, sh.sm[w][r16]);
    const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w_.m[k] - top);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<v4f *>(&sh.so[wave][r16 * LD + 16 * d + 4 * g]) = w_.o[k][d] * f;
    __syncthreads();
    // 16 rows x D: thread -> row, 4 columns at a time
    for (int x = threadIdx.x; x < 16 * (D / 4); x += 256) {
      const int row = x / (D / 4), col = (x % (D / 4)) * 4;
      if (k * 16 + row >= rows) continue;
      float mr = sh.sm[0][row];
#pragma unroll
      for (int w = 1; w < NW; ++w) mr = fmaxf(mr, sh.sm[w][row]);
      float lr = 0.f;
      v4f v = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        // (no maximum: nothing seen, 0, or nothing but NaN, NaN)
        lr += mr == -INFINITY ? sh.sl[w][row] : sh.sl[w][row] * __builtin_amdgcn_exp2f(sh.sm[w][row] - mr);
        v += *reinterpret_cast<const v4f *>(&sh.so[w][row * LD + col]);
      }
      emit(k, row, col, v, mr, lr);
    }
  }
}

}  // namespace dsl
