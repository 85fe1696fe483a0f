// Attention of few query rows (single new tokens, or a few drafted ones) over
// the paged 8-bit cache; attn_core.h has the mathematics and the row order.
//
// Bound by the cache's bytes: every wave walks tiles of 64 tokens on its own,
// codes straight from memory into registers (16 bytes per lane: whole 64-byte
// runs of a key row, whole kilobytes of V^T), converted and fed to the matrix
// instructions; the next tile's keys are in flight behind the softmax, the
// tile's values behind its scores.  No LDS and no barrier in the loop.  Four
// waves of a workgroup take every fourth tile of a split of the context and
// join in LDS; with too few sequences and heads for the chip the context is
// split over workgroups, whose partial sums a second kernel joins in split
// order.
#include "attn_core.h"
#include "launch.h"

namespace dsl {

constexpr int kTile = 64;      // tokens per step of a wave
constexpr int SPLIT_WGS = 2;
constexpr int kPromptRows = 64;   // query rows of a sequence and cache head from which attn_prompt.hip serves

// RB blocks of 16 query rows share every load.  blockIdx: x split * pairs + pair
// (sequence and head), y row block.  Workgroups go to the XCDs in turn: with the
// split running fastest, the late splits, which only long sequences have, all
// landed on the same ones (64 sequences of 2000 to 8192 tokens: 170 against 12x us).
template <int SRC, bool FP8, int D, int RB>
__global__ __launch_bounds__(256) void attn_rows_kernel(const KvCacheArgs c, const AttnArgs p, const int nsplit,
                                                        const int chunk, const int nblk) {
  constexpr bool F16 = SRC == SRC_F16;
  constexpr int NW = 4, DT = D / 16, DC = D / 64;
  constexpr int LD = D + 4;                      // floats per row of the joined tile
  __shared__ __align__(16) float so[NW][16 * LD];
  __shared__ float sm[NW][16], sl[NW][16];
  const int pairs = c.heads * c.seqs, pair = blockIdx.x % pairs;
  const int b = pair / c.heads, head = pair % c.heads, split = blockIdx.x / pairs;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const SeqView s = seq_view(c, b);
  const int rows = s.n * p.group;
  const int room = c.width * c.page;             // tokens that the table has pages for
  const int ntiles = ((s.len < room ? s.len : room) + kTile - 1) / kTile;
  const int t0 = split * chunk, t1 = t0 + chunk < ntiles ? t0 + chunk : ntiles;
  const int ktok = 16 * (r16 >> 2) + (r16 & 3);  // the lane's token of K tile 0 (tile t: + 4 t)
  const int P = c.page;
  const int64_t hstride = (int64_t)P * D;

  if (nsplit > 1 && t0 >= t1) {                  // behind the sequence's end: no sums
    for (int r = blockIdx.y * 256 + threadIdx.x; r < rows; r += nblk * 256) {
      const int i = r / p.group, hq = head * p.group + r % p.group;
      float *ml = p.ws + (int64_t)nsplit * c.rows * p.q_heads * D + (((int64_t)split * c.rows + s.row0 + i) * p.q_heads + hq) * 2;
      ml[0] = -INFINITY;
      ml[1] = 0.f;
    }
    return;
  }
  for (int rb = blockIdx.y; rb * 16 * RB < rows; rb += nblk) {
    // the rows' queries, as they stand in the products
    v4i qf[RB][2 * DC];
    int limit[RB];
    int lo = s.len;                              // tokens that every row sees
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      const int r = rb * 16 * RB + k * 16 + r16, rr = r < rows ? r : rows - 1;
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
      lo = s.first + (rb * 16 * RB) / p.group + 1;
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
    auto kpage = [&](int tile) { return page_of(c, b, (tile * kTile + 16 * (r16 >> 2)) / P); };
    auto vpage = [&](int tile) { return page_of(c, b, (tile * kTile + 16 * g) / P); };
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
        const int r = rb * 16 * RB + k * 16 + row;
        if (r >= rows) continue;
        float mr = sm[0][row];
#pragma unroll
        for (int w = 1; w < NW; ++w) mr = fmaxf(mr, sm[w][row]);
        float lr = 0.f;
        v4f v = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          lr += mr == -INFINITY ? 0.f : sl[w][row] * __builtin_amdgcn_exp2f(sm[w][row] - mr);
          v += *reinterpret_cast<const v4f *>(&so[w][row * LD + col]);
        }
        const int i = r / p.group, hq = head * p.group + r % p.group;
        if (nsplit > 1) {
          const int64_t at = ((int64_t)split * c.rows + s.row0 + i) * p.q_heads + hq;
          *reinterpret_cast<v4f *>(p.ws + at * D + col) = v;
          if (col == 0) {
            float *ml = p.ws + (int64_t)nsplit * c.rows * p.q_heads * D + at * 2;
            ml[0] = mr;
            ml[1] = lr;
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

// Joins the splits of one query row and head in a workgroup: a split per thread for
// the maximum and the sum, then four columns per thread, the splits dealt to 1024 / D
// threads of each.  (All splits in one thread's loop, a load's latency each, took 14
// to 27 us.)  An empty split has no sums.
constexpr int kMaxSplits = 256;
template <int SRC, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs p, const int64_t rows, const int nsplit) {
  constexpr int CG = D / 4, SL = 256 / CG;
  __shared__ float s_f[kMaxSplits], s_red[8];
  __shared__ v4f s_v[SL][CG];
  const int64_t at = blockIdx.x, n = rows * p.q_heads;
  const int tid = threadIdx.x;
  const float *ml = p.ws + (int64_t)nsplit * n * D;
  float m = -INFINITY, l = 0.f;
  if (tid < nsplit) {
    m = ml[(tid * n + at) * 2];
    l = ml[(tid * n + at) * 2 + 1];
  }
  float top = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((tid & 63) == 0) s_red[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
  s_f[tid] = f;
  l *= f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = l;
  __syncthreads();
  const int cg = tid % CG, sl = tid / CG;
  v4f v = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = sl; s < nsplit; s += SL) {
    const float fs = s_f[s];
    if (fs != 0.f) v += *reinterpret_cast<const v4f *>(p.ws + (s * n + at) * D + cg * 4) * fs;
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

struct AttnPlan {
  bool prompt;
  int rb, nblk, nsplit, chunk;   // chunk: tiles of a split (few rows)
};
static AttnPlan attn_plan(const KvCacheArgs &c, int q_heads, int max_q) {
  AttnPlan a;
  const int64_t rows = (int64_t)max_q * (q_heads / c.heads);
  a.prompt = rows > kPromptRows;
  a.chunk = 0;
  if (a.prompt) {
    const int per = attn_prompt_rows(c.dim);
    const int64_t pairs = (int64_t)c.heads * c.seqs, blocks = (rows + per - 1) / per;
    const int64_t room = ((int64_t)1 << 30) / pairs;
    a.rb = 0;
    a.nblk = (int)(blocks < room ? blocks : room);
    // one workgroup per CU; a split has four tiles at least
    const int64_t tiles = ((int64_t)c.width * c.page + kTile - 1) / kTile;
    int64_t ns = device_cu_count() / (pairs * a.nblk);
    if (ns > tiles / 4) ns = tiles / 4;
    if (ns > 64) ns = 64;
    a.nsplit = ns < 1 ? 1 : (int)ns;
    return a;
  }
  // (dim 256: two blocks of rows spill)
  a.rb = rows <= 16 || c.dim > 128 ? 1 : 2;
  const int64_t blocks = (rows + 16 * a.rb - 1) / (16 * a.rb), room = 65535;
  a.nblk = (int)(blocks < 1 ? 1 : (blocks < room ? blocks : room));   // each walks every nblk-th
  // Splits of equal length, so that sequences of any lengths load the CUs evenly
  // (those behind a sequence's end leave at once); at least one tile for every wave.
  const int64_t units = (int64_t)c.heads * c.seqs * a.nblk, want = SPLIT_WGS * (int64_t)device_cu_count();
  const int64_t tiles = ((int64_t)c.width * c.page + kTile - 1) / kTile, most = (tiles + 3) / 4;
  int64_t ns = units > 0 ? want / units : 1;
  if (ns > most) ns = most;
  if (ns > kMaxSplits) ns = kMaxSplits;
  if (ns < 1) ns = 1;
  a.chunk = (int)((tiles + ns - 1) / ns);
  a.chunk = (a.chunk + 3) / 4 * 4;               // whole rounds of the four waves
  a.nsplit = (int)((tiles + a.chunk - 1) / (a.chunk > 0 ? a.chunk : 1));
  if (a.nsplit < 1) a.nsplit = 1;
  return a;
}

size_t attn_workspace_bytes(const KvCacheArgs &c, int q_heads, int max_q) {
  const AttnPlan a = attn_plan(c, q_heads, max_q);
  return a.nsplit > 1 ? (size_t)a.nsplit * c.rows * q_heads * (c.dim + 2) * sizeof(float) : 0;
}

template <int SRC, bool FP8, int D>
static void launch_rows(const KvCacheArgs &c, const AttnArgs &p, const AttnPlan &a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.nsplit * c.heads * c.seqs), (unsigned)a.nblk);
  if (a.rb == 1) attn_rows_kernel<SRC, FP8, D, 1><<<grid, 256, 0, st>>>(c, p, a.nsplit, a.chunk, a.nblk);
  else if constexpr (D <= 128) attn_rows_kernel<SRC, FP8, D, 2><<<grid, 256, 0, st>>>(c, p, a.nsplit, a.chunk, a.nblk);
}

template <int SRC>
static hipError_t launch_src(const KvCacheArgs &c, const AttnArgs &p, hipStream_t st) {
  const AttnPlan a = attn_plan(c, p.q_heads, p.max_q);
  if (a.prompt) {
    const hipError_t e = launch_attn_prompt(SRC, c, p, a.nblk, a.nsplit, st);
    if (e != hipSuccess) return e;
  } else if (c.fp8) {
    if (c.dim == 64) launch_rows<SRC, true, 64>(c, p, a, st);
    else if (c.dim == 128) launch_rows<SRC, true, 128>(c, p, a, st);
    else launch_rows<SRC, true, 256>(c, p, a, st);
  } else {
    if (c.dim == 64) launch_rows<SRC, false, 64>(c, p, a, st);
    else if (c.dim == 128) launch_rows<SRC, false, 128>(c, p, a, st);
    else launch_rows<SRC, false, 256>(c, p, a, st);
  }
  if (a.nsplit > 1) {
    const unsigned n = (unsigned)c.rows * (unsigned)p.q_heads;
    if (c.dim == 64) attn_join_kernel<SRC, 64><<<n, 256, 0, st>>>(p, c.rows, a.nsplit);
    else if (c.dim == 128) attn_join_kernel<SRC, 128><<<n, 256, 0, st>>>(p, c.rows, a.nsplit);
    else attn_join_kernel<SRC, 256><<<n, 256, 0, st>>>(p, c.rows, a.nsplit);
  }
  return hipGetLastError();
}

hipError_t launch_attn(int src, const KvCacheArgs &c, const AttnArgs &p, hipStream_t st) {
  if (c.seqs == 0 || c.rows == 0) return hipSuccess;
  return src == SRC_BF16 ? launch_src<SRC_BF16>(c, p, st) : launch_src<SRC_F16>(c, p, st);
}

}  // namespace dsl
