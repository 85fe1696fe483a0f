// Attention of many query rows (prompts) over the paged 8-bit cache;
// attn_core.h has the mathematics.
//
// Bound by the matrix units and the softmax's vector operations side by side:
// per 64 tokens a wave of 32 rows (dim 128) feeds 32 32x32x16 products, about
// 1000 cycles, and spends about as many on 2048 exponentials and their sums.  So
// two waves share a SIMD, one's products behind the other's softmax, and the
// codes are converted once per workgroup, not once per wave: eight waves (256
// rows) stage a tile of 64 tokens in LDS as 16-bit operands, while the tile
// after next is on its way from memory into registers.  One barrier per tile.
//
// S^T = K Q^T on 32x32 tiles gives a lane 16 tokens of its query row: register
// i of lane half h is token 8 (i / 4) + 4 h + i % 4 of the tile's 32.  V's LDS
// rows hold their tokens in that order, 8 to a 16-byte chunk (chunk 2 s + h:
// registers 8 (s % 2) .. + 7 of tile s / 2), so probabilities enter O^T = V^T P^T
// from the registers they were computed in.  Registers 8 j .. 8 j + 7 are 16
// consecutive tokens over both halves: one page, so scales do not differ between
// lanes, and a group's largest score takes its scale once.
//
// The output is brought to a new maximum only where a row's grew by more than
// 2^8; until then its probabilities may reach 2^8, which the 16-bit and 32-bit
// numbers hold as well as 1.
#include "attn_core.h"
#include "launch.h"
#include "pipe_core.h"

namespace dsl {

constexpr int kPTile = 64;     // tokens per tile

template <bool F16>
DSL_DEV v16f mfma32(const v4i &a, const v4i &b, const v16f &c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

DSL_DEV float halves_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(a[0]), u2f(a[1]));
}
DSL_DEV float halves_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return u2f(a[0]) + u2f(a[1]);
}

// LDS slot of 16-byte chunk c of row r: rows of D bytes * 2 (K) and 128 bytes
// (V); both readers (32 rows, chunks c and c + 1 by lane half) meet no bank twice.
template <int CHUNKS>
DSL_DEV int pslot(int row, int c) {
  if constexpr (CHUNKS == 8) return c ^ pipe::swz<128>(row);
  else return c ^ (row & 15);
}

// Bit 7 of each byte that is an E4M3 NaN code.
DSL_DEV uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <int D>
struct PromptCfg {
  static constexpr int NW = D > 128 ? 4 : 8, NT = NW * 64, ROWS = NW * 32;
  static constexpr int WPS = NW / 4;                         // waves per SIMD
  static constexpr int KC = D / 8;                           // 16-byte chunks of a K row
  static constexpr int TILE = kPTile * D * 2;                // bytes of K or V
  static constexpr int UNITS = 2 * kPTile * D / 16 / NT;     // 16-code loads per thread
  static constexpr int STAGE = 2 * TILE;
};

// blockIdx: x (row block from the last on) * heads * sequences + ..., y split.
template <int SRC, bool FP8, int D>
__global__ __launch_bounds__(PromptCfg<D>::NT) __attribute__((amdgpu_waves_per_eu(PromptCfg<D>::WPS, PromptCfg<D>::WPS)))
void attn_prompt_kernel(const KvCacheArgs c, const AttnArgs p, const int nblk, const int nsplit) {
  using Cfg = PromptCfg<D>;
  constexpr bool F16 = SRC == SRC_F16;
  constexpr int KK = D / 16, DT = D / 32, U = Cfg::UNITS, KU = kPTile * D / 16;
  __shared__ __align__(16) uint8_t lds[2 * Cfg::STAGE];
  __shared__ float s_scale[2][8];                // of a tile's four 16-token groups: ks, vs
  __shared__ int s_flag[2][2];                   // groups in no page (bits), NaN codes among V
  // tokens (bits) whose V code is NaN, by column: staged as 0, since 0 * NaN
  // would carry one to rows that do not see it
  __shared__ uint64_t s_nan[2][FP8 ? D : 1];
  const int pairs = c.heads * c.seqs;
  const int blk = nblk - 1 - blockIdx.x / pairs, pair = blockIdx.x % pairs;   // the longest first
  const int head = pair % c.heads, b = pair / c.heads, split = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const SeqView s = seq_view(c, b);
  const int rows = s.n * p.group;
  const int P = c.page, room = c.width * P;
  const int len = s.len < room ? s.len : room;
  const int64_t hstride = (int64_t)P * D;

  for (int rb = blk; rb * Cfg::ROWS < rows; rb += nblk) {
    // tokens that the block's last row sees
    int end = len;
    if (p.causal) {
      int last = rb * Cfg::ROWS + Cfg::ROWS - 1;
      last = last < rows ? last : rows - 1;
      const int lim = s.first + last / p.group + 1;
      end = lim < end ? (lim > 0 ? lim : 0) : end;
    }
    const int ntiles = (end + kPTile - 1) / kPTile;
    const int t0 = (int)((int64_t)ntiles * split / nsplit), t1 = (int)((int64_t)ntiles * (split + 1) / nsplit);

    const int row = rb * Cfg::ROWS + wave * 32 + r32, rr = row < rows ? row : rows - 1;
    const int qi = rr / p.group, hq = head * p.group + rr % p.group;
    v4i qf[KK];
    {
      const uint16_t *qp = static_cast<const uint16_t *>(p.q) + (int64_t)(s.row0 + qi) * p.q_row + (int64_t)hq * p.q_head;
#pragma unroll
      for (int k = 0; k < KK; ++k) qf[k] = *reinterpret_cast<const v4i *>(qp + 16 * k + 8 * h);
    }
    const int seen = s.first + qi + 1;
    const int limit = p.causal ? (seen > 0 ? (seen < len ? seen : len) : 0) : len;
    int low = len;                               // tokens that every row of the wave sees
    if (p.causal) {
      const int r0 = rb * Cfg::ROWS + wave * 32;
      const int f = s.first + (r0 < rows ? r0 : rows - 1) / p.group + 1;
      low = f > 0 ? (f < len ? f : len) : 0;
    }

    v16f o[DT];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = (v16f){};

    // this thread's loads of a tile: units tid + NT j, K's first
    int pid[U], spid = -1;                       // pages of its units, of its scale
    uint4 raw[U];
    float sraw = 0.f;
    auto find = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = tid + Cfg::NT * j;
        const int tok = tile * kPTile + (u < KU ? u / (D / 16) : (u & 3) * 16);
        pid[j] = tok < len ? (int)page_of(c, b, tok / P) : -1;
      }
      const int tok = tile * kPTile + (tid & 3) * 16;
      spid = tid < 8 && tok < len ? (int)page_of(c, b, tok / P) : -1;
    };
    auto load = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = tid + Cfg::NT * j;
        const int64_t base = ((int64_t)(pid[j] < 0 ? 0 : pid[j]) * c.heads + head) * hstride;
        const uint8_t *at = u < KU ? c.k + base + (int64_t)((tile * kPTile + u / (D / 16)) & (P - 1)) * D + (u % (D / 16)) * 16
                                   : c.v + base + (int64_t)((u - KU) >> 2) * P + ((tile * kPTile + (u & 3) * 16) & (P - 1));
        raw[j] = *reinterpret_cast<const uint4 *>(at);
        if (u >= KU && pid[j] < 0) raw[j] = make_uint4(0, 0, 0, 0);
      }
      if (tid < 8) sraw = spid < 0 ? 0.f : (tid < 4 ? c.k_scale : c.v_scale)[(int64_t)spid * c.heads + head];
    };
    // the loaded tile as 16-bit operands
    auto stage = [&](int tile, int buf, bool absent) __attribute__((always_inline)) {
      uint8_t *kb = lds + buf * Cfg::STAGE, *vb = kb + Cfg::TILE;
      uint32_t bad = 0;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = tid + Cfg::NT * j;
        uint4 w = raw[j];
        if (u < KU) {
          const int r = u / (D / 16), ch = (u % (D / 16)) * 2;
          *reinterpret_cast<v4i *>(kb + r * (2 * D) + pslot<Cfg::KC>(r, ch) * 16) = codes8<FP8, F16>(w.x, w.y);
          *reinterpret_cast<v4i *>(kb + r * (2 * D) + pslot<Cfg::KC>(r, ch + 1) * 16) = codes8<FP8, F16>(w.z, w.w);
        } else {
          const int d = (u - KU) >> 2, g = u & 3;
          if constexpr (FP8) {                   // codes past the end can be NaN
            const int nv = len - (tile * kPTile + g * 16);
            if (nv < 16) {
              uint32_t *x = &w.x;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int n = nv - 4 * i;
                x[i] &= n >= 4 ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * n)) - 1);
              }
            }
            const uint32_t bx = nan_bytes(w.x), by = nan_bytes(w.y), bz = nan_bytes(w.z), bw = nan_bytes(w.w);
            uint32_t at = 0;
            if (bx | by | bz | bw) {
              auto nibble = [](uint32_t m) { return ((m >> 7) * 0x01020408u) >> 24 & 15; };
              at = nibble(bx) | nibble(by) << 4 | nibble(bz) << 8 | nibble(bw) << 12;
              w.x &= ~((bx >> 7) * 255u);
              w.y &= ~((by >> 7) * 255u);
              w.z &= ~((bz >> 7) * 255u);
              w.w &= ~((bw >> 7) * 255u);
            }
            reinterpret_cast<uint16_t *>(&s_nan[buf][d])[g] = (uint16_t)at;
            bad |= at;
          }
          *reinterpret_cast<v4i *>(vb + d * 128 + pslot<8>(d, 2 * g) * 16) = codes8<FP8, false>(w.x, w.z);
          *reinterpret_cast<v4i *>(vb + d * 128 + pslot<8>(d, 2 * g + 1) * 16) = codes8<FP8, false>(w.y, w.w);
        }
      }
      if (tid < 8) s_scale[buf][tid] = sraw * (tid < 4 ? p.scale * kLog2e : 1.f);
      if (tid < 64) {
        const uint64_t none = __ballot(absent && tid < 4);
        if (tid == 0) s_flag[buf][0] = (int)none;
      }
      if constexpr (FP8) {
        if (__any(bad) && lane == 0) s_flag[buf][1] = 1;
      }
    };

    if (tid < 2) s_flag[tid][1] = 0;
    __syncthreads();                             // also: the last block's readers
    bool absent = false;                         // of the loaded tile: this thread's scale has no page
    if (t0 < t1) {
      find(t0);
      load(t0);
      absent = spid < 0;
      if (t0 + 1 < t1) find(t0 + 1);
      stage(t0, t0 & 1, absent);
      if (t0 + 1 < t1) {
        load(t0 + 1);
        absent = spid < 0;
      }
      if (t0 + 2 < t1) find(t0 + 2);
    }
    for (int tile = t0; tile < t1; ++tile) {
      __syncthreads();                           // the tile is staged, the other stage is read
      const int buf = tile & 1;
      const uint8_t *kb = lds + buf * Cfg::STAGE, *vb = kb + Cfg::TILE;
      // the fragments' addresses: the rows' swizzles do not depend on t and d, and
      // flip no bit of 32 k, so one register each; formed afresh in every tile
      // (kept for all k they spill)
      int kat = r32 * (2 * D) + pslot<Cfg::KC>(r32, h) * 16, vat = r32 * 128 + pslot<8>(r32, h) * 16;
      asm volatile("" : "+v"(kat), "+v"(vat));
      const bool work = tile * kPTile < limit;
      const bool any = __any(work);

      v16f sc[2];
      float ks[4], vs[4];
      bool masked = false;
      int none = 0, nans = 0;
      if (any) {
        const v4f k4 = *reinterpret_cast<const v4f *>(&s_scale[buf][0]), v4 = *reinterpret_cast<const v4f *>(&s_scale[buf][4]);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          ks[g] = k4[g];
          vs[g] = v4[g];
        }
        none = s_flag[buf][0];
        nans = FP8 ? s_flag[buf][1] : 0;
        masked = __builtin_amdgcn_readfirstlane(
            (int)(tile * kPTile + kPTile > low || none || !(fminf(fminf(ks[0], ks[1]), fminf(ks[2], ks[3])) >= 0.f)));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          sc[t] = (v16f){};
#pragma unroll
          for (int k = 0; k < KK; ++k) {
            const v4i a = *reinterpret_cast<const v4i *>(kb + (kat ^ (32 * k)) + t * 32 * 2 * D);
            sc[t] = mfma32<F16>(a, qf[k], sc[t]);
          }
        }
      }
      if (tile + 1 < t1) {
        if (tid == 0 && FP8) s_flag[buf ^ 1][1] = 0;
        stage(tile + 1, buf ^ 1, absent);
        if (tile + 2 < t1) {
          load(tile + 2);
          absent = spid < 0;
        }
        if (tile + 3 < t1) find(tile + 3);
      }
      if (!any) continue;
      __builtin_amdgcn_sched_barrier(0);

      float top;
      if (!masked) {
        top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float x = sc[g >> 1][8 * (g & 1)];
#pragma unroll
          for (int i = 1; i < 8; ++i) x = fmaxf(x, sc[g >> 1][8 * (g & 1) + i]);
          top = fmaxf(top, x * ks[g]);
        }
      } else {
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int tok = tile * kPTile + 32 * (i >> 4) + 8 * ((i & 15) >> 2) + 4 * h + (i & 3);
          float v = sc[i >> 4][i & 15] * ks[i >> 3];
          v = tok < limit && !(none >> (i >> 3) & 1) ? v : -INFINITY;
          sc[i >> 4][i & 15] = v;
          top = fmaxf(top, v);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) ks[g] = 1.f;
      }
      top = halves_max(top);
      if (__any(top > m + 8.f || m == -INFINITY)) {
        const float now = fmaxf(m, top), ref = now == -INFINITY ? 0.f : now;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = now;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= alpha;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      v4i pf[4], pl[F16 ? 4 : 1];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = sc[g >> 1][8 * (g & 1) + i];
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, ks[g], -ref));
          l += e[i];
          sc[g >> 1][8 * (g & 1) + i] = x;
        }
        if (masked) {                            // 0 stays 0 whatever the scale
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = sc[g >> 1][8 * (g & 1) + i] == -INFINITY ? 0.f : e[i] * vs[g];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] *= vs[g];
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t hi = pack_bf16x2(e[2 * w], e[2 * w + 1]);
          pf[g][w] = (int)hi;
          if constexpr (F16) pl[g][w] = (int)pack_bf16x2(e[2 * w] - u2f(hi << 16), e[2 * w + 1] - u2f(hi & 0xffff0000u));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const v4i a = *reinterpret_cast<const v4i *>(vb + (vat ^ (32 * g)) + d * 32 * 128);
          o[d] = mfma32<false>(a, pf[g], o[d]);
          if constexpr (F16) o[d] = mfma32<false>(a, pl[g], o[d]);
        }
      if (FP8 && nans) {                         // NaN where the row sees a NaN code
        const int n = limit - tile * kPTile;
        const uint64_t sees = n >= 64 ? ~0ull : (n > 0 ? (1ull << n) - 1 : 0);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (s_nan[buf][32 * d + 8 * (i >> 2) + 4 * h + (i & 3)] & sees) o[d][i] = __builtin_nanf("");
      }
    }

    // lane: row r32, columns 32 d + 8 q + 4 h .. + 3 of register quad q
    l = halves_sum(l);
    if (row < rows) {
      if (nsplit > 1) {
        const int64_t n = (int64_t)c.rows * p.q_heads, at = (int64_t)split * n + (int64_t)(s.row0 + qi) * p.q_heads + hq;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<v4f *>(p.ws + at * D + 32 * d + 8 * q + 4 * h) =
                (v4f){o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
        if (h == 0) {
          float *ml = p.ws + (int64_t)nsplit * n * D + at * 2;
          ml[0] = m;
          ml[1] = l;
        }
      } else {
        const float inv = l > 0.f ? 1.0f / l : 0.f;      // a row that sees nothing is 0
        uint16_t *op = static_cast<uint16_t *>(p.o) + (int64_t)(s.row0 + qi) * p.o_row + (int64_t)hq * p.o_head;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint2 *>(op + 32 * d + 8 * q + 4 * h) =
                make_uint2(narrow2<SRC>(o[d][4 * q] * inv, o[d][4 * q + 1] * inv),
                           narrow2<SRC>(o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv));
      }
    }
  }
}

template <int SRC, bool FP8, int D>
static hipError_t launch_prompt_cfg(const KvCacheArgs &c, const AttnArgs &p, int nblk, int nsplit, hipStream_t st) {
  const dim3 grid((unsigned)(nblk * c.heads * c.seqs), (unsigned)nsplit);
  attn_prompt_kernel<SRC, FP8, D><<<grid, PromptCfg<D>::NT, 0, st>>>(c, p, nblk, nsplit);
  return hipGetLastError();
}

int attn_prompt_rows(int dim) { return dim > 128 ? PromptCfg<256>::ROWS : PromptCfg<128>::ROWS; }

hipError_t launch_attn_prompt(int src, const KvCacheArgs &c, const AttnArgs &p, int nblk, int nsplit, hipStream_t st) {
  auto go = [&](auto src_tag, auto fp8_tag) {
    constexpr int S = decltype(src_tag)::value;
    constexpr bool F = decltype(fp8_tag)::value;
    if (c.dim == 64) return launch_prompt_cfg<S, F, 64>(c, p, nblk, nsplit, st);
    if (c.dim == 128) return launch_prompt_cfg<S, F, 128>(c, p, nblk, nsplit, st);
    return launch_prompt_cfg<S, F, 256>(c, p, nblk, nsplit, st);
  };
  using B = std::integral_constant<int, SRC_BF16>;
  using H = std::integral_constant<int, SRC_F16>;
  if (src == SRC_BF16) return c.fp8 ? go(B{}, std::true_type{}) : go(B{}, std::false_type{});
  return c.fp8 ? go(H{}, std::true_type{}) : go(H{}, std::false_type{});
}

}  // namespace dsl
