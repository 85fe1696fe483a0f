// The walk of 32 NB query rows per wave over a context (attn_shared.hip), for rows
// that are too many for attn_rows.h and too few, or too spread over a line, for the
// workgroups of attn_prompt.hip.  attn_core.h has the mathematics.
//
// Four waves take every fourth tile of 64 tokens, codes straight from memory into
// registers; no LDS and no barrier before they join.  A tile is converted once
// for all 32 NB rows, and its matrix products (2 NB D / 4 of 32x32x16) are about as long
// as its exponentials, so one wave per SIMD carries them behind each other's backs
// as far as the compiler deals them; keys of the next tile are on their way from the
// scores on, values from the output on.
//
// Both products take fp16 operands: codes of 8 bits are exact in it (int8 by two
// byte permutes and two packed sums per four: 1024 + (c + 128) - 1152), fp16 queries
// too.  bf16 queries are brought to a largest element of 2^7 .. 2^8 by a power of two
// per row: what then lies below 2^-14 is off by 2^-25 at most, 2^-32 of the row's largest.
// Probabilities enter as 2^8 exp(s - m) vs with m the running maximum of s + log vs, so
// that they are at most 2^8 (2^15: below) whatever the scales are: fp16's rounding of half a
// step, 2^-12, or 2^-33 of the largest where they are below 2^-22 of it (a step of fp16's
// smallest numbers: without the 2^8, 131072 small ones could lose 2^-8 together).  For
// fp16 results they enter as two numbers, hi + lo.  Page scales of no logarithm (negative, infinite, NaN) and below 2^-90
// (which count as 0) act on the probabilities.  Sums stand relative to m too, the scales in it: the factors that join
// waves and parts are fp32, so of scales 2^126 and more apart the smaller ones' tokens would be lost to the sum.
//
// S^T = K Q^T on 32x32 tiles gives a lane 16 tokens of its query row.  Tokens are dealt
// to the rows of the K tiles so that they are consecutive: row r of tile t is token
// 32 t + 16 ((r / 4) % 2) + 4 (r / 8) + r % 4, and lane half h holds tokens 32 t + 16 h
// .. + 15, one page's, the 16 bytes of V that it loads.
//
// The maximum is not looked for in a tile that every row sees: exponentials are formed
// with the last one, and only where their sum passes 2^15 (or a row has none yet) the
// tile is settled: masked, brought to its own maximum, sums and output with it.
#pragma once

#include "attn_rows.h"

namespace dsl {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef v4i __attribute__((may_alias)) Word16;   // 16 bytes of shared memory that others use as floats
constexpr float kLift = 8.f;   // log2 of the largest probability, as it stands in the products

template <class T>
DSL_DEV T *uniform(T *p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<T *>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)u) |
                               (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(u >> 32)) << 32);
}
template <bool FP8>
DSL_DEV v4i codes8_f16(uint32_t lo, uint32_t hi) {
  if constexpr (FP8) {
    return codes8<true, true>(lo, hi);
  } else {
    const v2h less = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
    auto two = [&](uint32_t w, uint32_t sel) __attribute__((always_inline)) {
      return __builtin_bit_cast(int, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, w, sel)) + less);
    };
    return (v4i){two(a, 0x04010400u), two(a, 0x04030402u), two(b, 0x04010400u), two(b, 0x04030402u)};
  }
}
DSL_DEV uint32_t pack_f16x2(float a, float b) {
  typedef float v2f_ __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f_){a, b}, v2h));
}
template <bool F16>
DSL_DEV v16f mfma32t(const v4i &a, const v4i &b, const v16f &c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
DSL_DEV float halves_most(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(a[0]), u2f(a[1]));
}
DSL_DEV float halves_total(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return u2f(a[0]) + u2f(a[1]);
}

// Pages of a tile's four groups of 16 tokens (-1: none): first and second of the
// first 32 tokens, of the second.  (No array: the compiler would index it in memory.)
struct TilePages {
  int a, b, c, d;
  DSL_DEV int of(int t, bool second) const {
    const int p = t ? c : a, q = t ? d : b;
    return second ? q : p;
  }
  DSL_DEV bool none() const { return (a | b | c | d) < 0; }
};

// WHOLE: pages of 64 tokens and more, which hold whole tiles: one number, and addresses
// that are the wave's but for a fixed offset of the lane.
template <int SRC_, bool FP8_, int D_, int NB_, bool WHOLE>
struct TileWalk {
  static constexpr int SRC = SRC_, D = D_, NB = NB_, BLOCK = 32, ROWS = 32 * NB, NW = 4;
  static constexpr bool FP8 = FP8_, F16 = SRC == SRC_F16;
  static constexpr int KX = D / 32, DT = D / 32;
  static constexpr int WGS = 1;  // of a CU: 128 columns take all of a SIMD's registers (64 about half: two are untried)
  // The queries as they stand in the products, the same for all waves, in LDS: in
  // registers they spill.
  static constexpr bool SHARED = true;
  typedef v4i Queries[NB][2 * KX][64];
  Queries &q;
  float qs[NB];                  // what the queries were divided by
  const int *limit;              // of row r32 of block b: [32 b + r32], in LDS
  v16f o[NB][DT];
  float m[NB], l[NB];
  bool nans;                     // `hide` took a NaN that some row may see

  DSL_DEV explicit TileWalk(Queries &q) : q(q) {}

  // A row's queries, block b, by one wave for all; what they were divided by.
  DSL_DEV float load(int b, const uint16_t *from) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));                // (addresses are formed here: kept through the walk, they spill)
    const int lane = tid & 63, h = lane >> 5;
    v4i qf[2 * KX];
#pragma unroll
    for (int x = 0; x < KX; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) qf[2 * x + e] = *reinterpret_cast<const v4i *>(from + 32 * x + 16 * h + 8 * e);
    float by = 1.f;
    if constexpr (!F16) {
      typedef uint16_t v2u __attribute__((ext_vector_type(2)));
      v2u most = {0, 0};                         // the largest magnitude's bits (of infinities and NaN: any power will do)
#pragma unroll
      for (int x = 0; x < 2 * KX; ++x)
#pragma unroll
        for (int w = 0; w < 4; ++w) most = __builtin_elementwise_max(most, __builtin_bit_cast(v2u, qf[x][w] & 0x7fff7fff));
      const float top = halves_most(u2f((uint32_t)(most[0] > most[1] ? most[0] : most[1]) << 16 & 0x7f800000u));
      int e = (int)(f2u(top) >> 23) - 127;       // 2^e <= the largest < 2^(e + 1)
      e = top > 0.f ? (e < -100 ? -100 : e > 127 ? 127 : e) : 7;
      by = u2f((uint32_t)(127 + e - 7) << 23);
      const float up = u2f((uint32_t)(127 + 7 - e) << 23);
#pragma unroll
      for (int x = 0; x < 2 * KX; ++x)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          qf[x][w] = (int)pack_f16x2(u2f((uint32_t)qf[x][w] << 16) * up, u2f((uint32_t)qf[x][w] & 0xffff0000u) * up);
    }
#pragma unroll
    for (int x = 0; x < 2 * KX; ++x) q[b][x][lane] = qf[x];
    return by;
  }

  // All rows see the tokens before lo.  Tiles t0 .. t1 - 1, every fourth of a wave.
  // room: 2 DT words for each lane of the wave.
  DSL_DEV void walk(const KvCacheArgs &c, const Context &ctx, float scale, int head, int t0, int t1, int lo, Word16 *room) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r32 = lane & 31, h = lane >> 5, kgroup = (r32 >> 2) & 1;
    const int P = c.page, pshift = 31 - __builtin_clz(P);
    const int64_t hstride = (int64_t)P * D;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      m[b] = -INFINITY;
      l[b] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[b][d] = (v16f){};
    }
    nans = false;
    uint4 kr[2][KX], vr[2][DT];
    float kraw[2], vraw[2];
    // Pages by scalar loads: a vector load's wait would be one for the codes on
    // their way too.
    const auto table = (const __attribute__((address_space(4))) int32_t *)uniform(ctx.table);
    const auto kscale = (const __attribute__((address_space(4))) float *)uniform(c.k_scale);
    const auto vscale = (const __attribute__((address_space(4))) float *)uniform(c.v_scale);
    const int width = __builtin_amdgcn_readfirstlane(ctx.width), len = __builtin_amdgcn_readfirstlane(ctx.len);
    auto pages = [&](int tile) __attribute__((always_inline)) {
      auto page = [&](int g) __attribute__((always_inline)) {
        const int tok = tile * kTile + 16 * g, i = tok >> pshift;
        const bool in = tile < t1 && tok < len && i < width;
        const int p = table[in ? i : 0];         // (width > 0 where there is a tile)
        return in && p >= 0 && p < c.pages ? p : -1;
      };
      TilePages pg;
      pg.a = pg.b = pg.c = pg.d = page(0);
      if constexpr (!WHOLE) {
        pg.b = page(1);
        pg.c = page(2);
        pg.d = page(3);
      }
      return pg;
    };
    const uint32_t klane = (16 * kgroup + 4 * (r32 >> 3) + (r32 & 3)) * D + 16 * h, vlane = r32 * P + 16 * h;
    auto load_k = [&](int tile, const TilePages &pg) __attribute__((always_inline)) {
      if constexpr (WHOLE) {
        const uint8_t *base = c.k + ((int64_t)(pg.a < 0 ? 0 : pg.a) * c.heads + head) * hstride + (tile * kTile & (P - 1)) * D;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < KX; ++x) kr[t][x] = *reinterpret_cast<const uint4 *>(base + 32 * t * D + 32 * x + klane);
        return;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int p = pg.of(t, kgroup != 0);
        const int at = (tile * kTile + 32 * t + 16 * kgroup) & (P - 1);
        const uint8_t *base = c.k + ((int64_t)(p < 0 ? 0 : p) * c.heads + head) * hstride +
                              (at + 4 * (r32 >> 3) + (r32 & 3)) * D + 16 * h;
#pragma unroll
        for (int x = 0; x < KX; ++x) kr[t][x] = *reinterpret_cast<const uint4 *>(base + 32 * x);
      }
    };
    auto load_v = [&](int tile, const TilePages &pg) __attribute__((always_inline)) {
      if constexpr (WHOLE) {
        const uint8_t *base = c.v + ((int64_t)(pg.a < 0 ? 0 : pg.a) * c.heads + head) * hstride + (tile * kTile & (P - 1));
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int d = 0; d < DT; ++d) vr[t][d] = *reinterpret_cast<const uint4 *>(base + 32 * t + d * 32 * P + vlane);
        return;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int p = pg.of(t, h != 0);
        const int64_t at = (int64_t)(p < 0 ? 0 : p) * c.heads + head;
        const uint8_t *base = c.v + at * hstride + r32 * P + ((tile * kTile + 32 * t + 16 * h) & (P - 1));
#pragma unroll
        for (int d = 0; d < DT; ++d) vr[t][d] = *reinterpret_cast<const uint4 *>(base + (int64_t)d * 32 * P);
      }
    };
    auto load_scales = [&](const TilePages &pg) __attribute__((always_inline)) {
      if constexpr (WHOLE) {
        const int64_t at = (int64_t)(pg.a < 0 ? 0 : pg.a) * c.heads + head;
        kraw[0] = kraw[1] = kscale[at];
        vraw[0] = vraw[1] = vscale[at];
        return;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int p = pg.of(t, h != 0);
        const int64_t at = (int64_t)(p < 0 ? 0 : p) * c.heads + head;
        kraw[t] = c.k_scale[at];
        vraw[t] = c.v_scale[at];
      }
    };
    int tile = t0 + wave;
    TilePages pg, pn, pm;                        // of this tile, of the wave's next two
    if (tile >= t1) return;
    pg = pages(tile);
    load_k(tile, pg);
    load_scales(pg);
    load_v(tile, pg);
    pn = pages(tile + NW);
    const float unit = scale * kLog2e;
    v16f s[NB][2];
    // the groups' scales: of the scores; log2 of the values'
    float kq[NB][2], lv[2];
    bool odd = false, masked = false;
    // The tile's scores and scales, and the next one's keys on their way; whether
    // a token is hidden from some row.
    auto scores = [&]() __attribute__((always_inline)) {
      int at = lane;
      asm volatile("" : "+v"(at));               // (read in every tile: kept, they would spill)
#pragma unroll
      for (int x = 0; x < KX; ++x)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const v4i a0 = codes8_f16<FP8>(kr[t][x].x, kr[t][x].y), a1 = codes8_f16<FP8>(kr[t][x].z, kr[t][x].w);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            s[b][t] = mfma32t<true>(a0, q[b][2 * x][at], x ? s[b][t] : (v16f){});
            s[b][t] = mfma32t<true>(a1, q[b][2 * x + 1][at], s[b][t]);
          }
        }
      odd = false;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool there = pg.of(t, h != 0) >= 0;
        const float ks = there ? kraw[t] * unit : 0.f, vs = there ? vraw[t] : 1.f, size = __builtin_fabsf(vs);
        const bool finite = size < INFINITY, tiny = finite && !(size >= 0x1p-90f);
        lv[t] = !finite ? 0.f : tiny ? -90.f : __builtin_amdgcn_logf(size);
        odd |= !(vs >= 0x1p-90f && finite);
#pragma unroll
        for (int b = 0; b < NB; ++b) kq[b][t] = ks * qs[b];
      }
      load_k(tile + NW < t1 ? tile + NW : tile, pn);
      load_scales(pn);
      pm = pages(tile + 2 * NW);
      odd = __any(odd) != 0;
      masked = tile * kTile + kTile > lo || pg.none();
      return masked;
    };
    // Scores to powers of two, -infinity where hidden; sums and output to their
    // maximum.  (Outside the loop of the common tiles: there, the compiler would keep a
    // second copy of the output.)
    auto settle = [&]() __attribute__((always_inline)) {
      const int pos = tile * kTile + 16 * h;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float top = m[b];
        const int end = limit[32 * b + r32];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const bool there = pg.of(t, h != 0) >= 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float v = s[b][t][i] * kq[b][t];
            const float z = pos + 32 * t + i < end && there ? v : -INFINITY;
            s[b][t][i] = z;
            top = fmaxf(top, z + lv[t]);
          }
          kq[b][t] = 1.f;
        }
        top = halves_most(top);
        const float ref = top == -INFINITY ? 0.f : top, alpha = __builtin_amdgcn_exp2f(m[b] - ref);
        m[b] = top;
        l[b] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[b][d] *= alpha;
      }
    };
    v4i pf[NB][2][2], pl[F16 ? NB : 1][2][2];    // P, tokens 8 z .. + 7 of the lane's 16 (pl: their low parts)
    float sum[NB][2];
    // True where a sum has grown past what fp16 holds, or a row has no maximum: all that it
    // has seen were missing pages or scores of -infinity.
    auto exponentials = [&]() __attribute__((always_inline)) {
      bool grown = false;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        grown |= m[b] == -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float off = kLift + lv[t] - (m[b] == -INFINITY ? 0.f : m[b]);
          float e[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][t][i], kq[b][t], off));
          sum[b][t] = (((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]))) +
                      (((e[8] + e[9]) + (e[10] + e[11])) + ((e[12] + e[13]) + (e[14] + e[15])));
          grown |= !(sum[b][t] <= 32768.f);
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float a = e[8 * z + 2 * w], y = e[8 * z + 2 * w + 1];
              const uint32_t hi = pack_f16x2(a, y);
              pf[b][t][z][w] = (int)hi;
              if constexpr (F16) {
                const v2h q = __builtin_bit_cast(v2h, hi);
                pl[b][t][z][w] = (int)pack_f16x2(a - (float)q[0], y - (float)q[1]);
              }
            }
        }
      }
      return __any(grown) != 0;
    };
    auto output = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const v4i a0 = codes8_f16<FP8>(vr[t][d].x, vr[t][d].y), a1 = codes8_f16<FP8>(vr[t][d].z, vr[t][d].w);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            o[b][d] = mfma32t<true>(a0, pf[b][t][0], o[b][d]);
            o[b][d] = mfma32t<true>(a1, pf[b][t][1], o[b][d]);
            if constexpr (F16) {
              o[b][d] = mfma32t<true>(a0, pl[b][t][0], o[b][d]);
              o[b][d] = mfma32t<true>(a1, pl[b][t][1], o[b][d]);
            }
          }
        }
    };
    // The wave's next tile; false: none.
    auto next = [&]() __attribute__((always_inline)) {
      load_v(tile + NW < t1 ? tile + NW : tile, pn);
      pg = pn;
      pn = pm;
      tile += NW;
      return tile < t1;
    };

    // Rows that have no maximum yet take one of the tile's scores for a beginning.
    auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float top = s[b][0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = kq[b][0] < 0.f ? fminf(top, s[b][0][i]) : fmaxf(top, s[b][0][i]);
        m[b] = halves_most(__builtin_fmaf(top, kq[b][0], lv[0]));
      }
    };
    bool settled = scores(), more = true;
    if (!settled) begin();
    while (more) {
      if (settled) {
        settle();
        if constexpr (FP8) {
          if (masked) nans |= hide(ctx.len, tile, pg, vr, room);
        }
      }
      for (;;) {
        if (exponentials() && !settled) break;   // back to settle it
        settled = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float inv = __builtin_amdgcn_exp2f(-lv[t]);
#pragma unroll
          for (int b = 0; b < NB; ++b) l[b] = __builtin_fmaf(sum[b][t], inv, l[b]);
        }
        if (odd) {
          asm volatile("");                      // (a branch: not computed in every tile)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            // what is not in the exponent: 0, -1 or a number that is none
            const int p = pg.of(t, h != 0);
            const float vs = p < 0 ? 1.f : c.v_scale[(int64_t)p * c.heads + head], size = __builtin_fabsf(vs);
            const float by = !(size < INFINITY) ? vs : !(size >= 0x1p-90f) ? 0.f : vs < 0.f ? -1.f : 1.f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                times(pf[b][t][z], by);
                if constexpr (F16) times(pl[b][t][z], by);
              }
          }
        }
        output();
        more = next();
        if (!more) break;
        if (scores()) break;                     // to be settled
      }
      settled = true;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) m[b] -= kLift;  // what the sums are relative to
  }

  // Probabilities by what of their group's scale is not in the exponent (0 stays: a
  // hidden token's).
  static DSL_DEV void times(v4i &p, float by) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int both = p[w];                     // (a bit cast of the element itself takes element 0's bits)
      const v2h x = __builtin_bit_cast(v2h, both);
      p[w] = (int)pack_f16x2((float)x[0] == 0.f ? 0.f : (float)x[0] * by, (float)x[1] == 0.f ? 0.f : (float)x[1] * by);
    }
  }

  // V that some row must not meet, in a tile that not all rows see: codes past the
  // end or of no page, and NaN ones, become 0 (probability 0 does not remove a
  // NaN).  True if a NaN was among those that some row may see.  (In shared memory, by a
  // loop: in registers the whole walk would spill, 126 us for 104.)
  DSL_DEV bool hide(int len, int tile, const TilePages &pg, uint4 (&vr)[2][DT], Word16 *room) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < 2 * DT; ++i) room[i * 64 + lane] = __builtin_bit_cast(v4i, vr[i / DT][i % DT]);
    uint32_t any = 0;
#pragma unroll 1
    for (int i = 0; i < 2 * DT; ++i) {
      const int t = i / DT;
      int nv = len - (tile * kTile + 32 * t + 16 * h);
      nv = pg.of(t, h != 0) < 0 || nv < 0 ? 0 : (nv > 16 ? 16 : nv);
      v4i x = room[i * 64 + lane];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int n = nv - 4 * w;
        const uint32_t y = (uint32_t)x[w] & (n >= 4 ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * n)) - 1)), nan = nan_bytes(y);
        any |= nan;
        x[w] = (int)(y & ~nan);
      }
      room[i * 64 + lane] = x;
    }
#pragma unroll
    for (int i = 0; i < 2 * DT; ++i) vr[i / DT][i % DT] = __builtin_bit_cast(uint4, (v4i)room[i * 64 + lane]);
    return __any(any != 0) != 0;
  }

  // What `hide` took from rows that see it: a NaN value is one in the row's column.
  // so: the wave's joined tile; sees(row): tokens that the row sees.  (The wave's tiles are
  // looked at again: in the walk, the registers would spill.)
  template <class F>
  DSL_DEV void restore(const KvCacheArgs &c, const Context &ctx, int head, int t0, int t1, float *so, const F &sees) const {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), P = c.page;
    const int end = ctx.len < t1 * kTile ? ctx.len : t1 * kTile;
#pragma unroll 1
    for (int tile = t0 + wave; tile < t1; tile += NW)
#pragma unroll 1
      for (int tok = tile * kTile; tok < tile * kTile + kTile && tok < end; ++tok) {
        if (tok / P >= ctx.width) return;
        const int p = ctx.table[tok / P];
        if (p < 0 || p >= c.pages) continue;
#pragma unroll 1
        for (int d = tid & 63; d < D; d += 64) {
          const uint32_t code = c.v[(((int64_t)p * c.heads + head) * D + d) * P + (tok & (P - 1))];
          if ((code & 0x7f) != 0x7f) continue;
#pragma unroll 1
          for (int r = 0; r < ROWS; ++r)
            if (tok < sees(r)) so[r * (D + 4) + d] = __builtin_nanf("");
        }
      }
  }
};

// The waves' shares of a workgroup's rows, joined: each row's maximum, sum and the waves'
// factors by a thread of its own, then one row-major tile per wave, with `restore` for
// what a wave took from it.  row_sums(row, maximum, sum); emit(row, column, sums of 4
// columns).
template <int D, int ROWS>
struct TileJoin {
  static constexpr int NW = 4, LD = D + 4;       // floats per row of the joined tile
  float so[NW][ROWS * LD], sm[NW][ROWS], sl[NW][ROWS];
};
template <class Walk, class G, class R, class F>
DSL_DEV void join_tiles(TileJoin<Walk::D, Walk::ROWS> &sh, const Walk &w, int rows, const G &restore, const R &row_sums,
                        const F &emit) {
  constexpr int NW = 4, D = Walk::D, DT = Walk::DT, LD = D + 4;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));                  // (addresses are formed here: kept through the walk, they spill)
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int b = 0; b < Walk::NB; ++b) {
    const float lw = halves_total(w.l[b]);
    if (h == 0) {
      sh.sm[wave][b * 32 + r32] = w.m[b];
      sh.sl[wave][b * 32 + r32] = lw;
    }
  }
  __syncthreads();
  if (tid < Walk::ROWS) {
    float mk[NW], lr = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) mk[k] = sh.sm[k][tid];
    const float mr = fmaxf(fmaxf(mk[0], mk[1]), fmaxf(mk[2], mk[3]));
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      // (no maximum: nothing seen, 0, or nothing but NaN, NaN)
      const float f = mr == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mk[k] - mr);
      lr += sh.sl[k][tid] * f;
      sh.sm[k][tid] = mr == -INFINITY ? 0.f : f;
    }
    if (tid < rows) row_sums(tid, mr, lr);
  }
  __syncthreads();
#pragma unroll
  for (int b = 0; b < Walk::NB; ++b) {
    const float f = sh.sm[wave][b * 32 + r32];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<v4f *>(&sh.so[wave][(b * 32 + r32) * LD + 32 * d + 8 * q + 4 * h]) =
            (v4f){w.o[b][d][4 * q] * f, w.o[b][d][4 * q + 1] * f, w.o[b][d][4 * q + 2] * f, w.o[b][d][4 * q + 3] * f};
  }
  if constexpr (Walk::FP8) {
    if (w.nans) restore(sh.so[wave]);
  }
  __syncthreads();
  // thread -> row, 4 columns at a time
  const int n = (rows < Walk::ROWS ? rows : Walk::ROWS) * (D / 4);
#pragma unroll 2
  for (int x = tid; x < n; x += 256) {
    const int row = x / (D / 4), col = (x % (D / 4)) * 4;
    v4f v = *reinterpret_cast<const v4f *>(&sh.so[0][row * LD + col]);
#pragma unroll
    for (int k = 1; k < NW; ++k) v += *reinterpret_cast<const v4f *>(&sh.so[k][row * LD + col]);
    emit(row, col, v);
  }
}

}  // namespace dsl
