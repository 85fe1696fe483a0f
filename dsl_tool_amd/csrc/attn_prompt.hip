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
  if constexpr (CHUNKS == 4) return c ^ pipe::swz<64>(row);
  else if constexpr (CHUNKS == 8) return c ^ pipe::swz<128>(row);
  else return c ^ (row & 15);
}

// LDS writes of this wave have landed; then the workgroup's barrier.  Loads from
// memory stay in flight (__syncthreads would wait for them).
DSL_DEV void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int D>
struct PromptCfg {
  static constexpr int NW = 8, NT = NW * 64;                 // two waves per SIMD
  // dim 256: tiles of 32 tokens, and two waves compute the same scores, each half
  // of the output's columns (all of them would take 128 of its 256 registers)
  static constexpr int HALVES = D > 128 ? 2 : 1, T = D >= 128 ? 32 : 64;
  static constexpr int ROWS = NW / HALVES * 32;              // query rows
  static constexpr int G = T / 16, TS = T / 32;              // 16-token groups, 32-token score tiles
  static constexpr int DH = D / HALVES, DT = DH / 32;        // the wave's output columns
  static constexpr int KC = D / 8, VC = T / 8;               // 16-byte chunks of K's and V's rows
  static constexpr int TILE = T * D * 2;                     // bytes of K or V
  static constexpr int UNITS = 2 * T * D / 16 / NT;          // 16-code loads per thread
  // dim 128: the queries stay in LDS (kept in registers, others spill)
  static constexpr bool QLDS = false;
  static constexpr int QBYTES = QLDS ? NW * (D / 16) * 1024 : 0;
};

// blockIdx: x (row block from the last on) * heads * sequences + ..., y split.
template <int SRC, bool FP8, int D>
__global__ __launch_bounds__(PromptCfg<D>::NT) __attribute__((amdgpu_waves_per_eu(2, 2)))
void attn_prompt_kernel(const KvCacheArgs c, const AttnArgs p, const int nblk, const int nsplit) {
  using Cfg = PromptCfg<D>;
  constexpr bool F16 = SRC == SRC_F16;
  constexpr int T = Cfg::T, G = Cfg::G, TS = Cfg::TS, DT = Cfg::DT;
  constexpr int KK = D / 16, U = Cfg::UNITS, KU = T * D / 16;
  constexpr int VBASE = 2 * Cfg::TILE, QBASE = 4 * Cfg::TILE;
  __shared__ __align__(16) uint8_t lds[4 * Cfg::TILE + Cfg::QBYTES];   // two tiles of K, two of V, queries
  __shared__ __align__(16) float s_ks[4][4], s_vs[4][4];     // scales of a tile's 16-token groups
  __shared__ __align__(16) float s_log[4][4], s_inv[4][4];   // log2 vs, 1 / vs
  __shared__ __align__(16) int s_page[4][4];                 // the groups' pages, -1: none
  __shared__ int s_none[4], s_oddk[4], s_oddv[4];            // a group in no page; scales off the common path
  __shared__ int s_bad[4];                                   // NaN codes among V
  // tokens (bits) whose V code is NaN, by column: staged as 0, since 0 * NaN
  // would carry one to rows that do not see it
  __shared__ uint64_t s_nan[2][FP8 ? D : 1];
  __shared__ uint32_t s_row[FP8 ? Cfg::ROWS : 1][D / 32];   // ... and the columns (bits) that a row gets one in
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
  const int wrow = wave / Cfg::HALVES * 32, half = wave % Cfg::HALVES;
  const SeqView s = seq_view(c, b);
  const int rows = s.n * p.group;
  const int P = c.page, pshift = 31 - __builtin_clz(P), room = c.width * P;
  const int len = s.len < room ? s.len : room;
  const uint32_t hstride = (uint32_t)P * D, pstride = hstride * (uint32_t)c.heads;   // < 2^31
  const uint8_t *const kbase = c.k + (int64_t)head * hstride, *const vbase = c.v + (int64_t)head * hstride;

  for (int rb = blk; rb * Cfg::ROWS < rows; rb += nblk) {
    // tokens that the block's first and last rows see
    auto sees = [&](int r) {
      const int n = s.first + (r < rows ? r : rows - 1) / p.group + 1;
      return p.causal ? (n > 0 ? (n < len ? n : len) : 0) : len;
    };
    const int every = sees(rb * Cfg::ROWS), end = sees(rb * Cfg::ROWS + Cfg::ROWS - 1);
    const int ntiles = (end + T - 1) / T;
    const int t0 = (int)((int64_t)ntiles * split / nsplit), t1 = (int)((int64_t)ntiles * (split + 1) / nsplit);

    v4i qf[KK];
    const int qrow = rb * Cfg::ROWS + wrow + r32;
    {
      const int rr = qrow < rows ? qrow : rows - 1, qi = rr / p.group, hq = head * p.group + rr % p.group;
      const uint16_t *qp = static_cast<const uint16_t *>(p.q) + (int64_t)(s.row0 + qi) * p.q_row + (int64_t)hq * p.q_head;
#pragma unroll
      for (int k = 0; k < KK; ++k) qf[k] = *reinterpret_cast<const v4i *>(qp + 16 * k + 8 * h);
    }
    const int limit = sees(qrow);
    // tokens that every row of the wave sees, and that one of them sees
    const int low = __builtin_amdgcn_readfirstlane(limit);
    const int high = __builtin_amdgcn_readlane(limit, 31);
    int w1 = (high + T - 1) / T;                 // the wave's tiles: t0 .. w1 - 1
    w1 = w1 < t1 ? w1 : t1;

    v16f o[DT];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = (v16f){};

    // Pages go to LDS four tiles ahead (four threads look them up a tile before
    // that), codes and scales to registers a tile before they are staged.  Past the
    // last tile the pages are none, which read page 0 and stage it where nobody
    // looks.
    uint4 raw[U];
    float kraw = 0.f, vraw = 0.f;
    int page = -1;
    auto find = [&](int tile) __attribute__((always_inline)) {
      const int tok = tile * T + tid * 16;
      if (tid < G) page = tile < t1 && tok < len ? (int)page_of(c, b, tok >> pshift) : -1;
    };
    auto keep = [&](int tile) __attribute__((always_inline)) {
      if (tid < G) {
        s_page[tile & 3][tid] = page;
        const uint64_t none = __ballot(page < 0);
        if (tid == 0) s_none[tile & 3] = none != 0;
      }
    };
    // this thread's unit j: 16 codes of K (dim 64: by wave) or of V
    auto is_k = [&](int j) __attribute__((always_inline)) { return U > 1 ? j < U / 2 : wave < Cfg::NW / 2; };
    // (K of `tile`, V of the one before)
    auto load = [&](int tk) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = tid + Cfg::NT * j;
        const bool isk = is_k(j);
        const int tile = isk ? tk : tk - 1;
        const int g = isk ? u / (D / 16) >> 4 : u & (G - 1), pg = s_page[tile & 3][g];
        const uint32_t off = isk ? (uint32_t)(((tile * T + u / (D / 16)) & (P - 1)) * D + (u % (D / 16)) * 16)
                                 : (uint32_t)((((u - KU) / G) << pshift) + ((tile * T + g * 16) & (P - 1)));
        raw[j] = *reinterpret_cast<const uint4 *>((isk ? kbase : vbase) + (uint64_t)(uint32_t)(pg < 0 ? 0 : pg) * pstride + off);
      }
    };
    // this thread's part of K of a tile and of V of the one before as 16-bit operands
    auto stage = [&](int tk) __attribute__((always_inline)) {
      uint8_t *kb = lds + (tk & 1) * Cfg::TILE, *vb = lds + VBASE + ((tk - 1) & 1) * Cfg::TILE;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = tid + Cfg::NT * j;
        const uint4 w = raw[j];
        if (is_k(j)) {
          const int r = u / (D / 16), ch = (u % (D / 16)) * 2;
          uint8_t *to = kb + r * (2 * D);
          const int at = pslot<Cfg::KC>(r, ch) * 16;
          *reinterpret_cast<v4i *>(to + at) = codes8<FP8, F16>(w.x, w.y);
          *reinterpret_cast<v4i *>(to + (at ^ 16)) = codes8<FP8, F16>(w.z, w.w);
        } else {
          const int d = (u - KU) / G, g = u & (G - 1);
          uint8_t *to = vb + d * (2 * T);
          const int at = pslot<Cfg::VC>(d, 2 * g) * 16;
          *reinterpret_cast<v4i *>(to + at) = codes8<FP8, false>(w.x, w.z);
          *reinterpret_cast<v4i *>(to + (at ^ 16)) = codes8<FP8, false>(w.y, w.w);
        }
      }
    };
    // V of `tile` that some row must not meet, in the thread's own staged units: codes
    // past the end or of no page, which can be NaN, become 0; NaN ones that a row
    // may not see move to s_nan.  (Here, not in registers before: that spilled.)
    auto clean = [&](int tile) __attribute__((always_inline)) {
      if constexpr (FP8) {
        if (!__builtin_amdgcn_readfirstlane((int)(tile * T + T > every || s_none[tile & 3]))) return;
        int t = tid;
        asm volatile("" : "+v"(t));
        uint32_t bad = 0;
#pragma unroll 1
        for (int j = U > 1 ? U / 2 : 0; j < U; ++j) {
          const int u = t + Cfg::NT * j, d = (u - KU) / G, g = u & (G - 1);
          if (u < KU) continue;
          const int nv = s_page[tile & 3][g] < 0 ? 0 : len - (tile * T + g * 16);
          uint8_t *row = lds + VBASE + (tile & 1) * Cfg::TILE + d * (2 * T);
          uint32_t at = 0;
#pragma unroll 1
          for (int x = 0; x < 8; ++x) {          // two tokens of a chunk: half x / 4, word x % 4
            uint32_t *w = reinterpret_cast<uint32_t *>(row + pslot<Cfg::VC>(d, 2 * g + (x >> 2)) * 16) + (x & 3);
            const int tok = 4 * (x >> 2) + 8 * ((x & 3) >> 1) + 2 * (x & 1);
            uint32_t v = *w;
            if (tok >= nv) v &= 0xffff0000u;
            if (tok + 1 >= nv) v &= 0xffffu;
            if ((v & 0x7fffu) > 0x7f80u) {
              at |= 1u << tok;
              v &= 0xffff0000u;
            }
            if ((v & 0x7fffffffu) > 0x7f80ffffu) {
              at |= 2u << tok;
              v &= 0xffffu;
            }
            *w = v;
          }
          reinterpret_cast<uint16_t *>(&s_nan[tile & 1][d])[g] = (uint16_t)at;
          bad |= at;
        }
        if (__any(bad) && lane == 0) s_bad[tile & 3] = 1;
      }
    };
    // the scales: four threads of wave 1
    const int sg = tid - 64;
    auto load_scales = [&](int tile) __attribute__((always_inline)) {
      if (sg >= 0 && sg < G) {
        const int pg = s_page[tile & 3][sg];
        const int64_t at = (int64_t)(pg < 0 ? 0 : pg) * c.heads + head;
        kraw = c.k_scale[at];
        vraw = c.v_scale[at];
      }
    };
    auto stage_scales = [&](int tile) __attribute__((always_inline)) {
      if (sg >= 0 && sg < G) {
        const bool none = s_page[tile & 3][sg] < 0;
        const float ks = none ? 0.f : kraw * (p.scale * kLog2e), vs = none ? 1.f : vraw;
        const bool odd = !(vs >= 0x1p-60f && vs <= 0x1p60f);
        s_ks[tile & 3][sg] = ks;
        s_vs[tile & 3][sg] = odd ? vs : 1.f;
        s_log[tile & 3][sg] = odd ? 0.f : __builtin_amdgcn_logf(vs);
        s_inv[tile & 3][sg] = odd ? 1.f : __builtin_amdgcn_rcpf(vs);
        const uint64_t ok = __ballot(!(ks >= 0.f)), ov = __ballot(odd);
        if (sg == 0) {
          s_oddk[tile & 3] = ok != 0;
          s_oddv[tile & 3] = ov != 0;
        }
      }
    };

    // in step `tile`, once stage(tile + 2) has taken the codes
    auto fetch = [&](int tile) __attribute__((always_inline)) {
      load(tile + 3);
      if (wave == 0) {
        if (FP8 && tid == 0) s_bad[(tile + 2) & 3] = 0;      // set in the next step at the earliest
        keep(tile + 4);
        find(tile + 5);
      }
      if (wave == 1) {
        stage_scales(tile + 2);
        load_scales(tile + 3);
      }
    };

    __syncthreads();                             // the last block's readers
    if (tid < 4) s_bad[tid] = 0;
    if constexpr (FP8) {
      for (int i = tid; i < Cfg::ROWS * (D / 32); i += Cfg::NT) s_row[i / (D / 32)][i % (D / 32)] = 0;
    }
    if (t0 < t1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        find(t0 + i);
        keep(t0 + i);
      }
      __syncthreads();
      load(t0);                                  // (V of no tile: overwritten below)
      load_scales(t0);
      stage(t0);
      stage_scales(t0);
      __syncthreads();
      load(t0 + 1);
      load_scales(t0 + 1);
      stage(t0 + 1);
      clean(t0);
      stage_scales(t0 + 1);
      load(t0 + 2);
      load_scales(t0 + 2);
      find(t0 + 4);
    }
    // the queries have arrived before the loop: a wait for them there would be one
    // for the tiles' loads too
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      if constexpr (Cfg::QLDS) *reinterpret_cast<v4i *>(lds + QBASE + (wave * KK + k) * 1024 + lane * 16) = qf[k];
      else asm volatile("" : "+v"(qf[k]));
    }
    auto query = [&](int k) __attribute__((always_inline)) {
      if constexpr (Cfg::QLDS) return *reinterpret_cast<const v4i *>(lds + QBASE + (wave * KK + k) * 1024 + lane * 16);
      else return qf[k];
    };

    // fragment addresses: the rows' swizzles do not depend on t and d, and flip no
    // bit of 32 k, so one register each; formed afresh in every tile (kept for all
    // k they spill)
    const int kat0 = r32 * (2 * D) + pslot<Cfg::KC>(r32, h) * 16;
    const int vat0 = (half * Cfg::DH + r32) * (2 * T) + pslot<Cfg::VC>(r32, h) * 16;
    float kq[G], off[G];                         // the current scores' factors; log2 vs - m
    auto group_max = [&](const v16f (&sc)[TS], int g) __attribute__((always_inline)) {
      float x = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; i += 2) x = fmaxf(fmaxf(x, sc[g >> 1][8 * (g & 1) + i]), sc[g >> 1][8 * (g & 1) + i + 1]);
      return x;
    };
    // The scores of `tile` are there.  True where they need `settle` first: a token
    // is hidden from some row, a scale is off the common path, a row's maximum grew
    // by more than 2^16, or the wave is done.
    auto common = [&](int tile, const v16f (&sc)[TS]) __attribute__((always_inline)) {
      const v4f ks = *reinterpret_cast<const v4f *>(s_ks[tile & 3]), lg = *reinterpret_cast<const v4f *>(s_log[tile & 3]);
      const int odd = s_none[tile & 3] | s_oddk[tile & 3];
      float top = -INFINITY;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        kq[g] = ks[g];
        off[g] = lg[g] - m;
        top = fmaxf(top, group_max(sc, g) * ks[g]);
      }
      top = halves_max(top);
      return __builtin_amdgcn_readfirstlane((int)(__any(!(top <= m + 16.f)) || odd || tile * T + T > low || tile >= w1)) != 0;
    };
    // The same in general: scores to powers of two, -infinity where hidden, and sum
    // and output to their maximum.  (Outside the loop of the common tiles: there,
    // the compiler kept a second copy of the output and moved all of it in every
    // tile.)
    auto settle = [&](int tile, v16f (&sc)[TS]) __attribute__((always_inline)) {
      const v4f ks = *reinterpret_cast<const v4f *>(s_ks[tile & 3]), lg = *reinterpret_cast<const v4f *>(s_log[tile & 3]);
      const v4i pg = *reinterpret_cast<const v4i *>(s_page[tile & 3]);
      const int lim = limit - tile * T - 4 * h;
      float top = m;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = sc[g >> 1][8 * (g & 1) + i] * ks[g];
          const float x = 16 * g + 8 * (i >> 2) + (i & 3) < lim && pg[g] >= 0 ? v : -INFINITY;
          sc[g >> 1][8 * (g & 1) + i] = x;
          top = fmaxf(top, x);
        }
      top = halves_max(top);
      const float ref = top == -INFINITY ? 0.f : top, alpha = __builtin_amdgcn_exp2f(m - ref);
      m = top;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= alpha;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        kq[g] = 1.f;
        off[g] = lg[g] - ref;
      }
    };
    // One tile: the exponentials of its scores `sc` between the products of the next
    // tile's scores `nx`; its output's products between the staging of the tile after
    // that; then the next scores' maximum.
    auto step = [&](int tile, const v16f (&sc)[TS], v16f (&nx)[TS]) __attribute__((always_inline)) {
      const uint8_t *kb = lds + ((tile + 1) & 1) * Cfg::TILE, *vb = lds + VBASE + (tile & 1) * Cfg::TILE;
      int kat = kat0, vat = vat0;
      asm volatile("" : "+v"(kat), "+v"(vat));
      const v4f inv = *reinterpret_cast<const v4f *>(s_inv[tile & 3]);
      const int oddv = __builtin_amdgcn_readfirstlane(s_oddv[tile & 3]);
      const int nans = FP8 ? __builtin_amdgcn_readfirstlane(s_bad[tile & 3]) : 0;
      v4i pf[G], pl[F16 ? G : 1];
      // fragment f of K: step f / TS, part f % TS of the tokens; three are on their way
      constexpr int NF = KK * TS, PER = NF / G;
      v4i a[4], q[2];
      auto read = [&](int f) __attribute__((always_inline)) {
        if (f < NF) a[f & 3] = *reinterpret_cast<const v4i *>(kb + (kat ^ (32 * (f / TS))) + (f % TS) * 32 * 2 * D);
      };
#pragma unroll
      for (int f = 0; f < 3; ++f) read(f);
      q[0] = query(0);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int f = g * PER + i;
          read(f + 3);
          if (f % TS == 0 && f / TS + 1 < KK) q[(f / TS + 1) & 1] = query(f / TS + 1);
          nx[f % TS] = mfma32<F16>(a[f & 3], q[f / TS & 1], f >= TS ? nx[f % TS] : (v16f){});
        }
        float e[8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // exp(s - m) vs from one exponential; the sum takes 1 / vs
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[g >> 1][8 * (g & 1) + i], kq[g], off[g]));
          sum = i ? sum + e[i] : e[i];
        }
        l = __builtin_fmaf(sum, inv[g], l);
        asm volatile("" : "+v"(l));              // here, not where l is used: the 32 terms would be kept until then
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t hi = pack_bf16x2(e[2 * w], e[2 * w + 1]);
          pf[g][w] = (int)hi;
          if constexpr (F16) pl[g][w] = (int)pack_bf16x2(e[2 * w] - u2f(hi << 16), e[2 * w + 1] - u2f(hi & 0xffff0000u));
        }
        // a product, then the vector operations that run beside it
#pragma unroll
        for (int i = 0; i < PER / TS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x100, TS + Cfg::QLDS, 0);
#pragma unroll
          for (int t = 0; t < TS; ++t) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x402, (F16 ? 48 : 32) / PER, 0);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (oddv) {                                // scales no logarithm is taken of
        const v4f vs = *reinterpret_cast<const v4f *>(s_vs[tile & 3]);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            auto scaled = [&](int x) {
              const float lo = u2f((uint32_t)x << 16), hi = u2f((uint32_t)x & 0xffff0000u);
              return (int)pack_bf16x2(lo == 0.f ? 0.f : lo * vs[g], hi == 0.f ? 0.f : hi * vs[g]);
            };
            pf[g][w] = scaled(pf[g][w]);
            if constexpr (F16) pl[g][w] = scaled(pl[g][w]);
          }
      }
      auto read_v = [&](int f) __attribute__((always_inline)) {
        if (f < G * DT) a[f & 3] = *reinterpret_cast<const v4i *>(vb + (vat ^ (32 * (f / DT))) + (f % DT) * 32 * 2 * T);
      };
#pragma unroll
      for (int f = 0; f < 3; ++f) read_v(f);
#pragma unroll
      for (int f = 0; f < G * DT; ++f) {
        if (f % 4 == 0) __builtin_amdgcn_sched_barrier(0);
        read_v(f + 3);
        o[f % DT] = mfma32<false>(a[f & 3], pf[f / DT], o[f % DT]);
        if constexpr (F16) o[f % DT] = mfma32<false>(a[f & 3], pl[f / DT], o[f % DT]);
        if (f == 3) stage(tile + 2);
      }
      __builtin_amdgcn_sched_barrier(0);
      clean(tile + 1);
      fetch(tile);
      if (FP8 && nans) {                         // columns that get a NaN
        const int n = limit - tile * T;
        const uint64_t seen = n >= 64 ? ~0ull : (n > 0 ? (1ull << n) - 1 : 0);
#pragma unroll 1
        for (int d = half * Cfg::DH + h; d < (half + 1) * Cfg::DH; d += 2)
          if (s_nan[tile & 1][d] & seen) atomicOr(&s_row[wrow + r32][d >> 5], 1u << (d & 31));
      }
      return common(tile + 1, nx);
    };

    if (t0 < t1) {
      lds_barrier();
      int tile = t0;
      if (t0 < w1) {
        v16f sa[TS] = {}, sb[TS];
        {
          const uint8_t *kb = lds + (t0 & 1) * Cfg::TILE;
#pragma unroll
          for (int k = 0; k < KK; ++k)
#pragma unroll
            for (int t = 0; t < TS; ++t)
              sa[t] = mfma32<F16>(*reinterpret_cast<const v4i *>(kb + (kat0 ^ (32 * k)) + t * 32 * 2 * D), query(k), sa[t]);
        }
        // (a barrier behind settle too: the next step takes the tile's page entries)
        settle(tile, sa);
        lds_barrier();                           // step t0 stages over these K
        for (;;) {
          for (;;) {
            if (step(tile++, sa, sb)) {
#pragma unroll
              for (int t = 0; t < TS; ++t) sa[t] = sb[t];
              break;
            }
            lds_barrier();
            if (step(tile++, sb, sa)) break;
            lds_barrier();
          }
          if (tile < w1) settle(tile, sa);
          lds_barrier();
          if (tile >= w1) break;
        }
      } else {
        lds_barrier();
      }
      for (; tile < t1; ++tile) {                // no row of this wave sees more
        stage(tile + 2);
        clean(tile + 1);
        fetch(tile);
        lds_barrier();
      }
    }
    if constexpr (FP8) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const uint32_t bad = s_row[wrow + r32][half * DT + d];
        if (__any(bad)) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (bad >> (8 * (i >> 2) + 4 * h + (i & 3)) & 1) o[d][i] = __builtin_nanf("");
        }
      }
    }

    // lane: row r32, columns 32 d + 8 q + 4 h .. + 3 of register quad q (of the half)
    l = halves_sum(l);
    // (the row's place is formed afresh: kept through the loop it spills)
    int ln = tid & 63;
    asm volatile("" : "+v"(ln));
    const int row = rb * Cfg::ROWS + wrow + (ln & 31), h = ln >> 5, col = half * Cfg::DH + 4 * h;
    if (row < rows) {
      const int qi = row / p.group, hq = head * p.group + row % p.group;
      if (nsplit > 1) {
        const int64_t n = (int64_t)c.rows * p.q_heads, at = (int64_t)split * n + (int64_t)(s.row0 + qi) * p.q_heads + hq;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<v4f *>(p.ws + at * D + col + 32 * d + 8 * q) =
                (v4f){o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
        if (h == 0 && half == 0) {
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
            *reinterpret_cast<uint2 *>(op + col + 32 * d + 8 * q) =
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
