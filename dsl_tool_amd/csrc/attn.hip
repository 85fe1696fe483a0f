// Attention of few query rows (single new tokens, or a few drafted ones) over
// the paged 8-bit cache; attn_core.h has the mathematics and the row order.
//
// Bound by the cache's bytes: every wave walks tiles of 64 tokens on its own,
// codes straight from memory into registers (16 bytes per lane: whole 64-byte
// runs of a key row, whole kilobytes of V^T), converted and fed to the matrix
// instructions; the next tile's keys are in flight behind the softmax, the
// tile's values behind its scores.  No LDS and no barrier in the loop.  Four
// waves of a workgroup take every fourth tile of a range of the context and
// join in LDS.  The ranges: every unit (16 RB query rows of a sequence and
// cache head) has its context in rounds of `chunk` tiles, all units' rounds
// stand in one line, and each workgroup takes an equal run of it.  So
// sequences of any lengths load the CUs alike (64 sequences of 2000 to 8192
// tokens, 645 MB: 130 us, 5.0 TB/s; 162 with a workgroup per sequence and head,
// 149 with splits of one length).  A unit that one run holds whole is written at once; the parts
// of the others a second kernel joins in their order.
#include "attn_core.h"
#include "launch.h"

#include <cstdlib>

namespace dsl {

constexpr int kTile = 64;      // tokens per step of a wave
// Workgroups of a CU: what its registers hold.
constexpr int rows_wgs(int dim, int rb) { return dim * rb <= 128 ? 2 : 1; }
// Up to kFewRows query rows of a sequence and cache head, or where the line gives a
// run kFewRounds rounds at most, the kernel of few rows serves, else
// attn_prompt.hip's: 32 query heads on 8 of dim 128, 16 sequences of up to 4000
// tokens, rows 64 / 96 / 128: 67 / 90 / 108 against 81 / 85 / 91 us; one of 8000:
// 29 / 34 / 35 against 32 / 35 / 37, and rows 256, 4 rounds: 48 against 40; one of
// 1000, rows 256: 18 against 30.
// The shortest part of a prompt's context, in tiles of 64 tokens: 893 tokens of 16
// heads on 8, 500 of 32 on 8, 4 x 400 at dim 256: 4 tiles 32 / 34 / 48 us; 8 tiles (or
// whole) 36 / 30 / 59; 2 tiles 42 / 32 / 48.
constexpr int kPartTiles = 4;
constexpr int kFewRows = 96, kFewRounds = 2;
// Whether units are split into runs (and joined, about 5 us), by the rounds R that
// the table has room for and the units U per run; else a workgroup takes a unit
// whole.  32 query heads on 8 of dim 128, ragged contexts up to 256 R, split against
// whole, us: U 1/8, R 2 / 4 / 8: 11.2 / 11.6 / 14.6 against 9.2 / 15 / 25; U 1/2, R 4
// / 6 / 8: 22 / 26 / 27 against 17 / 22 / 27; U 1, R 4: 28 against 24, R 32: 134
// against 169; U 2, R 8: 84 against 89; U 4, R 4 / 16: 98 / 271 against 95 / 315; U 8,
// R 8: 290 against 283.  Past kLineSeqs sequences the line takes long to walk.
constexpr int kFewUnits = 8, kLongRounds = 8, kLineSeqs = 512;

// The workspace of a call whose units are split: a run has at most two parts,
// the end of a unit (slot 2 w) and the beginning of one (2 w + 1).
template <int D, int ROWS>
struct Parts {
  float *v, *ml;                 // [slot][ROWS][D], [slot][ROWS][maximum, sum]
  int2 *where;                   // [row][query head]: (-1, 0) written, else (first run, last run * 64 + row of the slot)
  DSL_DEV Parts(float *ws, int runs)
      : v(ws), ml(ws + (int64_t)2 * runs * ROWS * D), where(reinterpret_cast<int2 *>(ml + (int64_t)4 * runs * ROWS)) {}
};

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

// The line of all units' rounds: by sequence, cache head, row block.  A wave
// looks at 64 sequences at a time.
struct LineUnit {
  int b, rounds, blocks;         // sequence; rounds of a unit, row blocks of a head
  int off;                       // of the position in the sequence's part
};
template <int ROWS>
struct Line {
  const KvCacheArgs &c;
  const int group, chunk, lane;
  int at, rounds, blocks;        // of this lane's sequence
  int before, total, upto;       // the line's length before these 64; theirs; theirs up to and with this lane's
  DSL_DEV Line(const KvCacheArgs &c, int group, int chunk)
      : c(c), group(group), chunk(chunk), lane(threadIdx.x & 63), at(-64), before(0), total(0), upto(0) {}
  DSL_DEV void advance() {
    before += total;
    at += 64;
    rounds = blocks = 0;
    if (at + lane < c.seqs) {
      const SeqView s = seq_view(c, at + lane);
      const int room = c.width * c.page, tiles = ((s.len < room ? s.len : room) + kTile - 1) / kTile;
      rounds = tiles > chunk ? (tiles + chunk - 1) / chunk : 1;      // of no token: one, for its zeros
      blocks = (int)(((int64_t)s.n * group + ROWS - 1) / ROWS);
    }
    upto = lanes_sum(rounds * c.heads * blocks);
    total = __builtin_amdgcn_readlane(upto, 63);
  }
  DSL_DEV int length() {                         // of the whole line; back to its beginning
    while (at + 64 < c.seqs) advance();
    const int n = before + total;
    if (at > 0) {
      at = -64;
      before = total = 0;
      advance();
    }
    return n;
  }
  DSL_DEV LineUnit find(int x) {                 // x not before an earlier one
    while (x >= before + total) advance();
    const int k = __builtin_ctzll(__ballot(before + upto > x));
    LineUnit u;
    u.b = at + k;
    u.rounds = __builtin_amdgcn_readlane(rounds, k);
    u.blocks = __builtin_amdgcn_readlane(blocks, k);
    u.off = x - before - __builtin_amdgcn_readlane(upto, k) + u.rounds * c.heads * u.blocks;
    return u;
  }
};

// The NaN codes (E4M3: 0x7f, 0xff) of four, as bytes of ones.
DSL_DEV uint32_t nan_bytes(uint32_t w) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu; }
constexpr uint32_t kOnes = 0x38383838u;          // 1.0 four times

// RB blocks of 16 query rows share every load.
template <int SRC, bool FP8, int D, int RB>
__global__ __launch_bounds__(256, rows_wgs(D, RB)) void attn_rows_kernel(const KvCacheArgs c, const AttnArgs p,
                                                                           const int chunk, const bool split) {
  constexpr bool F16 = SRC == SRC_F16;
  constexpr int NW = 4, DT = D / 16, DC = D / 64, ROWS = 16 * RB;
  constexpr int LD = D + 4;                      // floats per row of the joined tile
  __shared__ __align__(16) float so[NW][16 * LD];
  __shared__ float sm[NW][16], sl[NW][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const Parts<D, ROWS> part(p.ws, gridDim.x);
  Line<ROWS> line(c, p.group, chunk);
  int per = 1, end = 1, x = 0;
  if (split) {
    const int whole = line.length();
    per = (whole + (int)gridDim.x - 1) / (int)gridDim.x;
    x = (int)blockIdx.x * per;
    end = whole - per > x ? x + per : whole;
  }
  const int ktok = 16 * (r16 >> 2) + (r16 & 3);  // the lane's token of K tile 0 (tile t: + 4 t)
  const int P = c.page;
  const int64_t hstride = (int64_t)P * D;

  while (x < end) {
    int b, head, rb, r0 = 0, left = 1, count = 1;
    SeqView s;
    if (split) {
      const LineUnit u = line.find(x);
      const int unit = u.off / u.rounds;
      b = u.b;
      r0 = u.off % u.rounds;
      head = unit / u.blocks;
      rb = unit % u.blocks;
      left = u.rounds - r0;
      count = left < end - x ? left : end - x;
      s = seq_view(c, b);
    } else if (c.starts) {                       // x row block, y cache head
      s = item_seq(c, blockIdx.x, [&](int row, int q) { return row * p.group / ROWS + q; }, b, rb);
      b = __builtin_amdgcn_readfirstlane(b);
      rb = __builtin_amdgcn_readfirstlane(rb);
      head = blockIdx.y;
      if (b < 0 || rb < 0) return;
    } else {
      const int blocks = (p.group + ROWS - 1) / ROWS;
      b = blockIdx.x / blocks;
      rb = blockIdx.x % blocks;
      head = blockIdx.y;
      s = seq_view(c, b);
    }
    const bool parted = left > count || r0 > 0;
    x += count;
    const int rows = s.n * p.group;
    if (rb * ROWS >= rows) return;               // (a workgroup for every block there may be)
    const int room = c.width * c.page;           // tokens that the table has pages for
    const int seen = s.len < room ? s.len : room, ntiles = (seen + kTile - 1) / kTile;
    int nsee = ntiles;                           // tiles that some row of the block sees
    if (p.causal) {
      const int high = s.first + ((rb + 1) * ROWS < rows ? (rb + 1) * ROWS - 1 : rows - 1) / p.group + 1;
      const int h = high < seen ? high : seen;
      nsee = h > 0 ? (h + kTile - 1) / kTile : 0;
    }
    const int t0 = r0 * chunk, t1 = split && nsee - t0 > count * chunk ? t0 + count * chunk : nsee;
    // the rows' queries, as they stand in the products
    v4i qf[RB][2 * DC];
    int limit[RB];
    int lo = s.len;                              // tokens that every row sees
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      const int r = rb * ROWS + k * 16 + r16, rr = r < rows ? r : rows - 1;
      const int i = rr / p.group, hq = head * p.group + rr % p.group;
      const uint16_t *qp = static_cast<const uint16_t *>(p.q) + (int64_t)(s.row0 + i) * p.q_row + (int64_t)hq * p.q_head;
#pragma unroll
      for (int x = 0; x < DC; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          qf[k][2 * x + h] = *reinterpret_cast<const v4i *>(qp + 64 * x + 16 * g + 8 * h);
      const int last = s.first + i + 1;
      limit[k] = p.causal ? (last > 0 ? last : 0) : s.len;
    }
    if (p.causal) {
      lo = s.first + (rb * ROWS) / p.group + 1;
      lo = lo > 0 ? lo : 0;
    }

    v4f o[RB][DT];
    float m[RB], l[RB];
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      m[k] = -INFINITY;
      l[k] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[k][d] = (v4f){0.f, 0.f, 0.f, 0.f};
    }

    // pages of a tile: the lane's key row, and its 16 tokens (V, scales)
    // (what the table and the scales hold past the last token's page is not read)
    auto page = [&](int tok) { return tok < s.len ? page_of(c, b, tok / P) : -1; };
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
      const float ks = vp < 0 ? 0.f : c.k_scale[va] * (p.scale * kLog2e);
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
        int nv = s.len - pos;
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
      if (FP8 && masked && p.causal) {
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
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (nans[i] != 0.f) o[k][d][i] = __builtin_nanf("");
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

    // join the waves: common maximum, then one row-major tile per wave
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      const float lw = groups_sum(l[k]);
      __syncthreads();                           // the last block's readers
      if (g == 0) {
        sm[wave][r16] = m[k];
        sl[wave][r16] = lw;
      }
      __syncthreads();
      float top = sm[0][r16];
#pragma unroll
      for (int w = 1; w < NW; ++w) top = fmaxf(top, sm[w][r16]);
      const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[k] - top);
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<v4f *>(&so[wave][r16 * LD + 16 * d + 4 * g]) = o[k][d] * f;
      __syncthreads();
      // 16 rows x D: thread -> row, 4 columns at a time
      for (int x = threadIdx.x; x < 16 * (D / 4); x += 256) {
        const int row = x / (D / 4), col = (x % (D / 4)) * 4;
        const int r = rb * ROWS + k * 16 + row;
        if (r >= rows) continue;
        float mr = sm[0][row];
#pragma unroll
        for (int w = 1; w < NW; ++w) mr = fmaxf(mr, sm[w][row]);
        float lr = 0.f;
        v4f v = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          // (no maximum: nothing seen, 0, or nothing but NaN, NaN)
          lr += mr == -INFINITY ? sl[w][row] : sl[w][row] * __builtin_amdgcn_exp2f(sm[w][row] - mr);
          v += *reinterpret_cast<const v4f *>(&so[w][row * LD + col]);
        }
        const int i = r / p.group, hq = head * p.group + r % p.group;
        if (split && r0 == 0 && col == 0) {
          const int last = (int)blockIdx.x + (left - count + per - 1) / per;
          part.where[(int64_t)(s.row0 + i) * p.q_heads + hq] =
              parted ? make_int2((int)blockIdx.x, last * 64 + k * 16 + row) : make_int2(-1, 0);
        }
        if (parted) {
          const int64_t at = ((int64_t)2 * blockIdx.x + (r0 == 0)) * ROWS + k * 16 + row;
          *reinterpret_cast<v4f *>(part.v + at * D + col) = v;
          if (col == 0) {
            part.ml[2 * at] = lr == lr ? mr : lr;          // a NaN sum without a maximum stays NaN in the join
            part.ml[2 * at + 1] = lr;
          }
        } else {
          const float inv = lr > 0.f ? 1.0f / lr : 0.f;    // a row that sees nothing is 0
          uint16_t *op = static_cast<uint16_t *>(p.o) + (int64_t)(s.row0 + i) * p.o_row + (int64_t)hq * p.o_head + col;
          *reinterpret_cast<uint2 *>(op) = make_uint2(narrow2<SRC>(v[0] * inv, v[1] * inv), narrow2<SRC>(v[2] * inv, v[3] * inv));
        }
      }
    }
  }
}

// Joins the parts of one query row and head in a workgroup: a part per thread for
// the maximum and the sum, then four columns per thread, the parts dealt to 1024 / D
// threads of each.  (All parts in one thread's loop, a load's latency each, took 14
// to 27 us.)  A part without a maximum saw no token and has sums of 0; one whose
// sum is NaN comes with a NaN for its maximum, and so has a NaN factor.  Values enter
// whatever the factor: a NaN in them is one behind a factor of 0 too.
constexpr int kMaxParts = 1024;
template <int SRC, int D, int ROWS>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs p, const int runs) {
  constexpr int CG = D / 4, SL = 256 / CG;
  __shared__ float s_f[kMaxParts], s_red[8];
  __shared__ v4f s_v[SL][CG];
  const int64_t at = blockIdx.x;
  const int tid = threadIdx.x;
  const Parts<D, ROWS> part(p.ws, runs);
  const int2 w = part.where[at];
  // written already.  (A row of no sequence has what the workspace held: in bounds, and
  // its result is not specified.)
  if (w.x < 0 || w.x >= runs) return;
  const float *const ml = part.ml;
  const int first = w.x, row = w.y & (ROWS - 1), many = (w.y >> 6) - first + 1;
  const int parts = many < runs - first ? many : runs - first;
  auto index = [&](int s) { return (int64_t)(s == 0 ? 2 * first + 1 : 2 * (first + s)) * ROWS + row; };
  float top = -INFINITY, l = 0.f;
  for (int s = tid; s < parts; s += 256) {
    const float m = ml[index(s) * 2];
    s_f[s] = m;
    top = fmaxf(top, m);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((tid & 63) == 0) s_red[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  for (int s = tid; s < parts; s += 256) {
    const float m = s_f[s], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    s_f[s] = f;
    l += ml[index(s) * 2 + 1] * f;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = l;
  __syncthreads();
  const int cg = tid % CG, sl = tid / CG;
  v4f v = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = sl; s < parts; s += SL) {
    v += *reinterpret_cast<const v4f *>(p.ws + index(s) * D + cg * 4) * s_f[s];
  }
  s_v[sl][cg] = v;
  __syncthreads();
  if (tid >= CG) return;
#pragma unroll
  for (int k = 1; k < SL; ++k) v += s_v[k][cg];
  l = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  uint16_t *op = static_cast<uint16_t *>(p.o) + (at / p.q_heads) * p.o_row + (at % p.q_heads) * p.o_head + cg * 4;
  *reinterpret_cast<uint2 *>(op) = make_uint2(narrow2<SRC>(v[0] * inv, v[1] * inv), narrow2<SRC>(v[2] * inv, v[3] * inv));
}

// Joins the parts [part][row][head] of a prompt's context: D / 4 threads of each row
// and head, as there are many of them and few parts (a workgroup each: 18 us for 500
// rows of 32 heads and two parts).  A part without a maximum may have no sums; NaN ones
// as above.
template <int SRC, int D>
__global__ __launch_bounds__(256) void attn_join_prompt_kernel(const AttnArgs p, const int64_t rows, const int parts) {
  constexpr int CG = D / 4;
  const int64_t n = rows * p.q_heads, at = (int64_t)blockIdx.x * (256 / CG) + threadIdx.x / CG;
  const int col = threadIdx.x % CG * 4;
  if (at >= n) return;
  const float2 *ml = reinterpret_cast<const float2 *>(p.ws + (int64_t)parts * n * D) + at;
  float top = -INFINITY, l = 0.f;
#pragma unroll 4
  for (int s = 0; s < parts; ++s) top = fmaxf(top, ml[s * n].x);
  v4f v = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float2 x = ml[s * n];
    if (x.x == -INFINITY) continue;
    const float f = __builtin_amdgcn_exp2f(x.x - top);
    l += x.y * f;
    v += *reinterpret_cast<const v4f *>(p.ws + (s * n + at) * D + col) * f;
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  uint16_t *op = static_cast<uint16_t *>(p.o) + (at / p.q_heads) * p.o_row + (at % p.q_heads) * p.o_head + col;
  *reinterpret_cast<uint2 *>(op) = make_uint2(narrow2<SRC>(v[0] * inv, v[1] * inv), narrow2<SRC>(v[2] * inv, v[3] * inv));
}

// A launch has fewer than 2^32 threads.  Only calls whose max_q is not that of their
// sequences come near it (max_q far above it: prompts' row blocks; far below: rows of
// few, and the joins), and any plan is right for them.
static bool launchable(int64_t workgroups, int threads) { return workgroups * threads < (int64_t)1 << 32; }

struct AttnPlan {
  bool prompt;
  int rb, nblk, nsplit;          // prompts: row blocks, parts of the context
  int runs, chunk;               // few rows: workgroups, tiles of a round; prompts: tokens of a part
  bool split;                    // they are runs of the line, and parts are joined
};
static AttnPlan attn_plan(const KvCacheArgs &c, int q_heads, int max_q) {
  AttnPlan a{};
  const int64_t rows = (int64_t)max_q * (q_heads / c.heads);
  // (dim 256: two blocks of rows spill)
  a.rb = rows <= 16 || c.dim > 128 ? 1 : 2;
  const int64_t group = q_heads / c.heads, most = c.rows < c.seqs ? c.rows : c.seqs;
  const int64_t likely = c.heads * most * ((rows + 16 * a.rb - 1) / (16 * a.rb));        // units
  const int64_t tiles = ((int64_t)c.width * c.page + kTile - 1) / kTile;
  a.runs = rows_wgs(c.dim, a.rb) * device_cu_count();
  if (a.runs > kMaxParts) a.runs = kMaxParts;
  const char *few = getenv("DSL_ATTN_FEW_ROWS");       // read per launch (tests switch it)
  if (few) a.prompt = rows > atoi(few);
  else a.prompt = rows > kFewRows && (double)likely * (double)((tiles + 3) / 4) > (double)(kFewRounds * a.runs);
  const int64_t pairs = (int64_t)c.heads * c.seqs;
  if (!launchable((int64_t)c.rows * group / (16 * a.rb) + c.seqs, 256)) a.prompt = true;
  if (!launchable(pairs, kPromptThreads)) a.prompt = false;     // (65535 sequences: more than 128 heads, and few rows of each)
  if (a.prompt) {
    const int per = attn_prompt_rows(c.dim);
    const int64_t blocks = (rows + per - 1) / per;
    const int64_t room = (((int64_t)1 << 32) - 1) / kPromptThreads / pairs;   // (a workgroup walks every nblk-th block)
    a.nblk = (int)(blocks < room ? blocks : room);
    // Parts of equal length, the shortest that one round of workgroups (one per CU)
    // holds if block i of n sees the first i / n of the new tokens; none where that
    // saves fewer tiles than a part has at least.
    const int64_t q = tiles < max_q / kTile ? tiles : max_q / kTile, room_for = device_cu_count() / pairs;
    auto fits = [&](int64_t len) {
      int64_t parts = 0;
      for (int64_t i = 1; i <= a.nblk; ++i) parts += (tiles - q + (q * i + a.nblk - 1) / a.nblk + len - 1) / len;
      return parts <= room_for;
    };
    int64_t len = tiles, lo = kPartTiles > (tiles + 63) / 64 ? kPartTiles : (tiles + 63) / 64;
    if (a.nblk < room_for) {
      for (int64_t hi = tiles; lo < hi;) {
        const int64_t mid = (lo + hi) / 2;
        if (fits(mid)) len = hi = mid;
        else lo = mid + 1;
      }
    }
    len += len & 1;                              // whole tiles of 128 tokens
    a.nsplit = len + kPartTiles > tiles || !launchable(((int64_t)c.rows * q_heads * c.dim + 1023) / 1024, 256)
                   ? 1 : (int)((tiles + len - 1) / len);
    a.chunk = (int)len * kTile;
    return a;
  }
  // rounds of a tile per wave, longer ones where the line's length would pass an int
  const int64_t units = c.heads * ((int64_t)c.rows * group / (16 * a.rb) + most);        // at most
  a.chunk = 4;
  while ((tiles + a.chunk - 1) / a.chunk * units > 1 << 30 && a.chunk < tiles) a.chunk *= 2;
  const int64_t rounds = (tiles + a.chunk - 1) / a.chunk;
  a.split = likely < kFewUnits * (int64_t)a.runs && c.seqs <= kLineSeqs && launchable((int64_t)c.rows * q_heads, 256) &&
            (rounds >= kLongRounds || (rounds - 3) * a.runs >= 8 * likely);
  if (!a.split) {
    const int64_t per = 16 * a.rb;
    a.runs = (int)(c.starts ? c.rows * group / per + c.seqs : c.seqs * ((group + per - 1) / per));
  }
  return a;
}

size_t attn_workspace_bytes(const KvCacheArgs &c, int q_heads, int max_q) {
  const AttnPlan a = attn_plan(c, q_heads, max_q);
  const size_t n = (size_t)c.rows * q_heads, row = (c.dim + 2) * sizeof(float);
  if (a.prompt) return a.nsplit > 1 ? a.nsplit * n * row : 0;
  return a.split ? (size_t)2 * a.runs * 16 * a.rb * row + n * sizeof(int2) : 0;
}

template <int SRC, int D, int RB>
static void launch_rows(const KvCacheArgs &c, const AttnArgs &p, const AttnPlan &a, hipStream_t st) {
  const dim3 grid((unsigned)a.runs, a.split ? 1u : (unsigned)c.heads);
  if (c.fp8) attn_rows_kernel<SRC, true, D, RB><<<grid, 256, 0, st>>>(c, p, a.chunk, a.split);
  else attn_rows_kernel<SRC, false, D, RB><<<grid, 256, 0, st>>>(c, p, a.chunk, a.split);
  if (a.split) attn_join_kernel<SRC, D, 16 * RB><<<(unsigned)c.rows * (unsigned)p.q_heads, 256, 0, st>>>(p, a.runs);
}

template <int SRC, int D>
static hipError_t launch_dim(const KvCacheArgs &c, const AttnArgs &p, hipStream_t st) {
  const AttnPlan a = attn_plan(c, p.q_heads, p.max_q);
  if (a.prompt) {
    const hipError_t e = launch_attn_prompt(SRC, c, p, a.nblk, a.nsplit, a.chunk, st);
    if (e != hipSuccess) return e;
    constexpr int each = 1024 / D;               // rows and heads of a workgroup
    const int64_t n = (int64_t)c.rows * p.q_heads;
    if (a.nsplit > 1) attn_join_prompt_kernel<SRC, D><<<(unsigned)((n + each - 1) / each), 256, 0, st>>>(p, c.rows, a.nsplit);
  } else if (a.rb == 1) {
    launch_rows<SRC, D, 1>(c, p, a, st);
  } else if constexpr (D <= 128) {
    launch_rows<SRC, D, 2>(c, p, a, st);
  }
  return hipGetLastError();
}

template <int SRC>
static hipError_t launch_src(const KvCacheArgs &c, const AttnArgs &p, hipStream_t st) {
  if (c.dim == 64) return launch_dim<SRC, 64>(c, p, st);
  if (c.dim == 128) return launch_dim<SRC, 128>(c, p, st);
  return launch_dim<SRC, 256>(c, p, st);
}

hipError_t launch_attn(int src, const KvCacheArgs &c, const AttnArgs &p, hipStream_t st) {
  if (c.seqs == 0 || c.rows == 0) return hipSuccess;
  return src == SRC_BF16 ? launch_src<SRC_BF16>(c, p, st) : launch_src<SRC_F16>(c, p, st);
}

}  // namespace dsl
