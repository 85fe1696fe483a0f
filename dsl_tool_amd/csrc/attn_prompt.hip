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

// v *= f when the wave-uniform `on` is non-zero.  The branch is inside the asm:
// one in the source made the compiler keep a second copy of the output and move
// all of it there and back in every tile.  (The products that wrote v are done:
// the caller has read later ones' results; f comes from v_exp_f32, hence the
// s_nop.)
DSL_DEV void scale_if(int on, v16f &v, float f) {
  float e[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) e[i] = v[i];
  asm volatile(
      "s_cmp_eq_u32 %17, 0\n\t"
      "s_cbranch_scc1 .Lscale_skip_%=\n\t"
      "s_nop 1\n\t"
      "v_mul_f32 %0, %0, %16\n\tv_mul_f32 %1, %1, %16\n\tv_mul_f32 %2, %2, %16\n\tv_mul_f32 %3, %3, %16\n\t"
      "v_mul_f32 %4, %4, %16\n\tv_mul_f32 %5, %5, %16\n\tv_mul_f32 %6, %6, %16\n\tv_mul_f32 %7, %7, %16\n\t"
      "v_mul_f32 %8, %8, %16\n\tv_mul_f32 %9, %9, %16\n\tv_mul_f32 %10, %10, %16\n\tv_mul_f32 %11, %11, %16\n\t"
      "v_mul_f32 %12, %12, %16\n\tv_mul_f32 %13, %13, %16\n\tv_mul_f32 %14, %14, %16\n\tv_mul_f32 %15, %15, %16\n"
      ".Lscale_skip_%=:"
      : "+v"(e[0]), "+v"(e[1]), "+v"(e[2]), "+v"(e[3]), "+v"(e[4]), "+v"(e[5]), "+v"(e[6]), "+v"(e[7]), "+v"(e[8]),
        "+v"(e[9]), "+v"(e[10]), "+v"(e[11]), "+v"(e[12]), "+v"(e[13]), "+v"(e[14]), "+v"(e[15])
      : "v"(f), "s"(on)
      : "scc");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = e[i];
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
  __shared__ __align__(16) float s_scale[2][8];  // of a tile's four 16-token groups: ks, vs
  __shared__ float2 s_log[2][4];                 // log2 vs, 1 / vs
  __shared__ __align__(16) int s_page[4][4];     // the groups' pages, -1: none
  __shared__ int s_odd[2], s_bad[4];             // scales off the common path; NaN codes among V
  // tokens (bits) whose V code is NaN, by column: staged as 0, since 0 * NaN
  // would carry one to rows that do not see it
  __shared__ uint64_t s_nan[2][FP8 ? D : 1];
  __shared__ uint32_t s_row[FP8 ? Cfg::ROWS : 1][DT];   // ... and the columns (bits) that a row gets one in
  const int pairs = c.heads * c.seqs;
  // Row blocks from the last, the longest, on.  Workgroups go to the eight XCDs,
  // and there to four shader engines, in turn: the pairs of an XCD (whose rows
  // share its L2) are rotated from row to row, or every other engine could get
  // one sequence's and run idle where that is the shorter one (two prompts of
  // 3600 and 2000 tokens: CUs busy 54% of the time).
  int blk = blockIdx.x / pairs, pair = blockIdx.x % pairs;
  if (pairs % 8 == 0) {
    const int n = pairs / 8, j = (blockIdx.x >> 3) % n;
    pair = (j + (n == 2 ? blk / 2 : blk)) % n * 8 + (blockIdx.x & 7);
  }
  blk = nblk - 1 - blk;
  const int head = pair % c.heads, b = pair / c.heads, split = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const SeqView s = seq_view(c, b);
  const int rows = s.n * p.group;
  const int P = c.page, pshift = 31 - __builtin_clz(P), room = c.width * P;
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
    // they have arrived before the loop: a wait for them there would be one for
    // the tiles' loads too
#pragma unroll
    for (int k = 0; k < KK; ++k) asm volatile("" : "+v"(qf[k]));
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

    // Pages go to LDS three tiles ahead (four threads look them up a tile before
    // that), codes and scales to registers two tiles ahead.
    uint4 raw[U];
    float sraw = 0.f;
    int page = -1;
    auto find = [&](int tile) __attribute__((always_inline)) {
      const int tok = tile * kPTile + tid * 16;
      if (tid < 4) page = tile < t1 && tok < len ? (int)page_of(c, b, tok >> pshift) : -1;
    };
    auto keep = [&](int tile) __attribute__((always_inline)) {
      if (tid < 4) s_page[tile & 3][tid] = page;
    };
    // this thread's unit j: 16 codes of K (D <= 64: by wave) or of V
    auto is_k = [&](int j) __attribute__((always_inline)) { return U > 1 ? j < U / 2 : wave < Cfg::NW / 2; };
    auto load = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = tid + Cfg::NT * j;
        if (is_k(j)) {
          const int r = u / (D / 16), pg = s_page[tile & 3][r >> 4];
          const uint8_t *at = c.k + ((int64_t)(pg < 0 ? 0 : pg) * c.heads + head) * hstride +
                              (((tile * kPTile + r) & (P - 1)) * D + (u % (D / 16)) * 16);
          raw[j] = *reinterpret_cast<const uint4 *>(at);
        } else {
          const int g = u & 3, pg = s_page[tile & 3][g];
          const uint8_t *at = c.v + ((int64_t)(pg < 0 ? 0 : pg) * c.heads + head) * hstride +
                              ((((u - KU) >> 2) << pshift) + ((tile * kPTile + g * 16) & (P - 1)));
          raw[j] = *reinterpret_cast<const uint4 *>(at);
          if (FP8 && pg < 0) raw[j] = make_uint4(0, 0, 0, 0);
        }
      }
      if (tid < 8) {
        const int pg = s_page[tile & 3][tid & 3];
        sraw = pg < 0 ? 0.f : (tid < 4 ? c.k_scale : c.v_scale)[(int64_t)pg * c.heads + head];
      }
    };
    // the loaded tile as 16-bit operands
    auto stage = [&](int tile, int buf) __attribute__((always_inline)) {
      uint8_t *kb = lds + buf * Cfg::STAGE, *vb = kb + Cfg::TILE;
      uint32_t bad = 0;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = tid + Cfg::NT * j;
        uint4 w = raw[j];
        if (is_k(j)) {
          const int r = u / (D / 16), ch = (u % (D / 16)) * 2;
          uint8_t *to = kb + r * (2 * D);
          const int at = pslot<Cfg::KC>(r, ch) * 16;
          *reinterpret_cast<v4i *>(to + at) = codes8<FP8, F16>(w.x, w.y);
          *reinterpret_cast<v4i *>(to + (at ^ 16)) = codes8<FP8, F16>(w.z, w.w);
        } else {
          const int d = (u - KU) >> 2, g = u & 3;
          if constexpr (FP8) {
            if (tile * kPTile + kPTile > len) {  // codes past the end can be NaN
              const int nv = len - (tile * kPTile + g * 16);
              auto first = [&](int n) { return n >= 4 ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * n)) - 1); };
              w.x &= first(nv);
              w.y &= first(nv - 4);
              w.z &= first(nv - 8);
              w.w &= first(nv - 12);
            }
            const uint32_t bx = nan_bytes(w.x), by = nan_bytes(w.y), bz = nan_bytes(w.z), bw = nan_bytes(w.w);
            uint32_t at = 0;
            if (bx | by | bz | bw) {
              auto nibble = [](uint32_t x) { return ((x >> 7) * 0x01020408u) >> 24 & 15; };
              at = nibble(bx) | nibble(by) << 4 | nibble(bz) << 8 | nibble(bw) << 12;
              w.x &= ~((bx >> 7) * 255u);
              w.y &= ~((by >> 7) * 255u);
              w.z &= ~((bz >> 7) * 255u);
              w.w &= ~((bw >> 7) * 255u);
            }
            reinterpret_cast<uint16_t *>(&s_nan[buf][d])[g] = (uint16_t)at;
            bad |= at;
          }
          uint8_t *to = vb + d * 128;
          const int at = pslot<8>(d, 2 * g) * 16;
          *reinterpret_cast<v4i *>(to + at) = codes8<FP8, false>(w.x, w.z);
          *reinterpret_cast<v4i *>(to + (at ^ 16)) = codes8<FP8, false>(w.y, w.w);
        }
      }
      if (tid < 8) {
        const float x = tid < 4 ? sraw * (p.scale * kLog2e) : sraw;
        s_scale[buf][tid] = x;
        // scales that the common path takes: its scores' maximum follows the
        // codes', and probabilities take theirs as a logarithm
        const bool odd = tid < 4 ? !(x >= 0.f) : !(x >= 0x1p-60f && x <= 0x1p60f);
        const uint64_t some = __ballot(odd);
        if (tid == 0) s_odd[buf] = some != 0;
        if (tid >= 4) s_log[buf][tid & 3] = make_float2(__builtin_amdgcn_logf(x), 1.0f / x);
      }
      if constexpr (FP8) {
        if (__any(bad) && lane == 0) s_bad[tile & 3] = 1;
      }
    };

    __syncthreads();                             // the last block's readers
    if (tid < 4) s_bad[tid] = 0;
    if constexpr (FP8) {
      for (int i = tid; i < Cfg::ROWS * DT; i += Cfg::NT) s_row[i / DT][i % DT] = 0;
    }
    if (t0 < t1) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        find(t0 + i);
        keep(t0 + i);
      }
      find(t0 + 3);
      __syncthreads();
      load(t0);
      stage(t0, t0 & 1);
      if (t0 + 1 < t1) load(t0 + 1);
    }
    // what follows a tile, behind its scores: the next one's operands, the loads of
    // the one after, the pages of the third
    auto advance = [&](int tile) __attribute__((always_inline)) {
      if (tile + 1 < t1) {
        if (FP8 && tid == 0) s_bad[(tile + 2) & 3] = 0;   // set a tile later at the earliest
        stage(tile + 1, (tile + 1) & 1);
        if (tile + 2 < t1) load(tile + 2);
        keep(tile + 3);
        find(tile + 4);
      }
    };
    // a tile whose tokens all rows of the wave see, in pages that there are, of
    // common scales
    auto common = [&](int tile) __attribute__((always_inline)) {
      const v4i pg = *reinterpret_cast<const v4i *>(s_page[tile & 3]);
      const bool none = min(min(pg[0], pg[1]), min(pg[2], pg[3])) < 0;
      return __builtin_amdgcn_readfirstlane((int)(tile * kPTile + kPTile <= low && !none && !s_odd[tile & 1])) != 0;
    };
    // fragment addresses: the rows' swizzles do not depend on t and d, and flip no
    // bit of 32 k, so one register each; formed afresh in every tile (kept for all
    // k they spill)
    const int kat0 = r32 * (2 * D) + pslot<Cfg::KC>(r32, h) * 16, vat0 = r32 * 128 + pslot<8>(r32, h) * 16;
    auto step = [&](auto slow_tag, int tile) __attribute__((always_inline)) {
      constexpr bool SLOW = decltype(slow_tag)::value;
      const int buf = tile & 1;
      const uint8_t *kb = lds + buf * Cfg::STAGE, *vb = kb + Cfg::TILE;
      int kat = kat0, vat = vat0;
      asm volatile("" : "+v"(kat), "+v"(vat));
      // four fragments ahead of the products that take them
      v16f sc[2] = {};
      {
        v4i a[2][4];
        auto read = [&](int n) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            a[n & 1][i] = *reinterpret_cast<const v4i *>(kb + (kat ^ (32 * (2 * n + (i >> 1)))) + (i & 1) * 32 * 2 * D);
        };
        read(0);
#pragma unroll
        for (int n = 0; n < KK / 2; ++n) {
          if (n + 1 < KK / 2) read(n + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[i & 1] = mfma32<F16>(a[n & 1][i], qf[2 * n + (i >> 1)], sc[i & 1]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      advance(tile);
      __builtin_amdgcn_sched_barrier(0);

      const v4f ks = *reinterpret_cast<const v4f *>(&s_scale[buf][0]);
      float top = -INFINITY;
      if constexpr (!SLOW) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float x = -INFINITY;
#pragma unroll
          for (int i = 0; i < 8; i += 2) x = fmaxf(fmaxf(x, sc[g >> 1][8 * (g & 1) + i]), sc[g >> 1][8 * (g & 1) + i + 1]);
          top = fmaxf(top, x * ks[g]);
        }
      } else {
        const v4i pg = *reinterpret_cast<const v4i *>(s_page[tile & 3]);
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int tok = tile * kPTile + 16 * g + 8 * (i >> 2) + 4 * h + (i & 3);
            const float v = tok < limit && pg[g] >= 0 ? sc[g >> 1][8 * (g & 1) + i] * ks[g] : -INFINITY;
            sc[g >> 1][8 * (g & 1) + i] = v;
            top = fmaxf(top, v);
          }
      }
      top = halves_max(top);
      const int grow = __builtin_amdgcn_readfirstlane((int)__any(top > m + 8.f || m == -INFINITY));
      const float now = grow ? fmaxf(m, top) : m, ref = now == -INFINITY ? 0.f : now;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);   // 1 unless it grew
      m = now;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) scale_if(grow, o[d], alpha);
      v4i va[2][4];
      auto read_v = [&](int n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int g = (4 * n + i) / DT, d = (4 * n + i) % DT;
          va[n & 1][i] = *reinterpret_cast<const v4i *>(vb + (vat ^ (32 * g)) + d * 32 * 128);
        }
      };
      read_v(0);
      v4i pf[4], pl[F16 ? 4 : 1];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float e[8];
        if constexpr (!SLOW) {
          // exp(s - m) vs from one exponential; the sum takes 1 / vs per group
          const float2 lg = s_log[buf][g];
          const float off = lg.x - ref;
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[g >> 1][8 * (g & 1) + i], ks[g], off));
            sum = i ? sum + e[i] : e[i];
          }
          l = __builtin_fmaf(sum, lg.y, l);
        } else {
          const float vs = s_scale[buf][4 + g];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = sc[g >> 1][8 * (g & 1) + i];
            e[i] = __builtin_amdgcn_exp2f(x - ref);
            l += e[i];
            e[i] = x == -INFINITY ? 0.f : e[i] * vs;       // whatever the scale
          }
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
      for (int n = 0; n < DT; ++n) {
        if (n + 1 < DT) read_v(n + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int g = (4 * n + i) / DT, d = (4 * n + i) % DT;
          o[d] = mfma32<false>(va[n & 1][i], pf[g], o[d]);
          if constexpr (F16) o[d] = mfma32<false>(va[n & 1][i], pl[g], o[d]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (FP8) {
        if (__builtin_amdgcn_readfirstlane(s_bad[tile & 3])) {   // columns that get a NaN
          const int n = limit - tile * kPTile;
          const uint64_t sees = n >= 64 ? ~0ull : (n > 0 ? (1ull << n) - 1 : 0);
          for (int d = h; d < D; d += 2)
            if (s_nan[buf][d] & sees) atomicOr(&s_row[wave * 32 + r32][d >> 5], 1u << (d & 31));
        }
      }
    };

    int tile = t0;
    while (tile < t1) {
      __syncthreads();                           // the tile is staged, the other stage is read
      if (!__any(tile * kPTile < limit)) break;
      if (common(tile)) {
        for (;;) {
          step(std::false_type{}, tile);
          if (++tile >= t1) break;
          __syncthreads();
          if (!common(tile)) break;
        }
        if (tile >= t1 || !__any(tile * kPTile < limit)) break;
      }
      step(std::true_type{}, tile++);
    }
    // rows that see no more: the workgroup's others do (the tile's barrier is passed)
    for (; tile < t1; ++tile) {
      advance(tile);
      if (tile + 1 < t1) __syncthreads();
    }
    if constexpr (FP8) {
      __syncthreads();
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const uint32_t bad = s_row[wave * 32 + r32][d];
        if (__any(bad)) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (bad >> (8 * (i >> 2) + 4 * h + (i & 3)) & 1) o[d][i] = __builtin_nanf("");
        }
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
