// Attention of many query rows (prompts) over the paged 8-bit cache;
// attn_core.h has the mathematics.
//
// Bound by the matrix units and the softmax's vector operations together:
// per 64 tokens a wave of 32 rows (dim 128) feeds 32 32x32x16 products, about
// 1000 cycles, and spends about as many on 2048 exponentials and their sums.  Two
// waves share a SIMD and are in phase (one barrier per tile), so the two kinds
// overlap in part: over the prompts below matrix units are busy 31% of the time,
// vector instructions at work 41%, CUs busy 80% (profiles/serving_counters.txt).
// The codes are converted once per workgroup, not once per wave: eight waves (256
// rows; 128 at dim 256) stage a tile of 8192 / D tokens in LDS as 16-bit
// operands, one 16-byte chunk of K and of V per thread, while the tile after
// next is on its way from memory into registers.  K and V have two tiles each
// and a step has one barrier.  Two prompts of up to 3600 tokens, contexts of up to
// 4600 (32 query heads on 8 of dim 128, 193 GFLOP): 246 to 258 us by card, 750 to 785
// TFLOP/s from E4M3; int8 233 us; fp16 results, whose second product runs twice, 331.
// (A wave that converted its own tiles from memory, as attn.hip's do: 951.)
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
// 2^16; until then its probabilities may reach 2^16, which bf16 and fp32 numbers
// hold as well as 1.
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

// 16 bits of a 64-bit word in LDS, which a thread writes and another reads whole.
typedef uint16_t __attribute__((may_alias)) Piece16;

// A wave's LDS reads but the last N (all: more false) have returned.
template <int N>
DSL_DEV void wait_reads(bool more) {
  if (more) __builtin_amdgcn_s_waitcnt((15 << 0) | (7 << 4) | (N << 8) | (3 << 14));
  else pipe::wait_lds();
}

template <int D>
struct PromptCfg {
  static constexpr int NT = kPromptThreads, NW = NT / 64;    // two waves per SIMD
  // Dim 256: two waves compute the same scores, each half of the output's columns
  // (all of them would take 128 of its 256 registers).
  static constexpr int HALVES = D > 128 ? 2 : 1;
  static constexpr int T = 8192 / D;                         // tokens of a step
  static constexpr int ROWS = NW / HALVES * 32;              // query rows
  static constexpr int G = T / 16, TS = T / 32;              // 16-token groups, 32-token score tiles
  static constexpr int DH = D / HALVES, DT = DH / 32;        // the wave's output columns
  static constexpr int VT = T < 64 ? T : 64;                 // tokens of a row of V in LDS (128: two matrices)
  static constexpr int KC = D / 8, VC = VT / 8;              // 16-byte chunks of K's and V's rows
  static constexpr int STAGE = T * D * 2;                    // bytes of K or V
  static_assert(T * D / 16 == NT, "a thread stages 16 codes of K and of V");
};

// blockIdx: x (row block from the last on) * heads * sequences + ..., y split.
template <int SRC, bool FP8, int D>
__global__ __launch_bounds__(PromptCfg<D>::NT) __attribute__((amdgpu_waves_per_eu(2, 2)))
void attn_prompt_kernel(const KvCacheArgs c, const AttnArgs p, const int nblk, const int nsplit, const int part) {
  using Cfg = PromptCfg<D>;
  constexpr bool F16 = SRC == SRC_F16;
  constexpr int T = Cfg::T, G = Cfg::G, TS = Cfg::TS, DT = Cfg::DT, VT = Cfg::VT, VG = VT / 16;
  constexpr int KK = D / 16, VBASE = 2 * Cfg::STAGE;
  __shared__ __align__(16) uint8_t lds[4 * Cfg::STAGE];      // two tiles of K, two of V
  // per 16-token group of a stage: score and V scales, log2 and 1 / of the latter,
  // pages (-1: none)
  __shared__ __align__(16) float s_ks[4][G], s_vs[4][G], s_log[4][G], s_inv[4][G];
  __shared__ __align__(16) int s_page[8][G];
  __shared__ int s_odd[4];                       // scales off the common path (bit 1: of V), or a group of no page
  __shared__ int s_none[8];                      // a group of no page
  __shared__ int s_bad[4];                       // NaN codes among V
  // tokens (bits) whose V code is NaN, by column: staged as 0, since 0 * NaN
  // would carry one to rows that do not see it
  __shared__ uint64_t s_nan[2][T / VT][FP8 ? D : 1];
  __shared__ uint32_t s_row[FP8 ? Cfg::ROWS : 1][D / 32];   // ... and the columns (bits) that a row gets one in
  const int pairs = c.heads * c.seqs;
  // Row blocks from the last, the longest, on.  Workgroups go to the eight XCDs,
  // and there to four shader engines, in turn: the pairs of an XCD (whose rows
  // share its L2) are rotated from row to row, or every other engine could get
  // one sequence's and run idle where that is the shorter one.  n = pairs / 8; the
  // pairs moved by blk, by blk / 2 and not at all, ragged prompts, us: n 2, two of
  // 3600 on 8 heads 368 / 258 / 375, four of 2000 on 4 126 / 120 / 126; n 3 158 / 158 /
  // 156; n 4 168 / 171 / 245; n 8 147 / 155 / 186.
  int blk = blockIdx.x / pairs, pair = blockIdx.x % pairs;
  if (pairs % 8 == 0) {
    const int n = pairs / 8, j = (blockIdx.x >> 3) % n;
    pair = (j + (n == 2 ? blk / 2 : blk)) % n * 8 + (blockIdx.x & 7);
  } else {                                       // an XCD would get every 2nd, 4th or 8th pair only
    pair = (pair + blockIdx.x / (pairs * (8 / (pairs & -pairs)))) % pairs;
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
    int t0 = nsplit > 1 ? split * (part / T) : 0;
    int t1 = nsplit > 1 && ntiles - t0 > part / T ? t0 + part / T : ntiles;
    asm volatile("" : "+s"(t0), "+s"(t1));       // (what they are made of would be kept in registers, which spill)
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
    int w1 = (high + T - 1) / T;                 // the wave's steps: t0 .. w1 - 1
    w1 = w1 < t1 ? w1 : t1;

    v16f o[DT];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = (v16f){};

    // Pages go to LDS three tiles ahead (looked up a tile before that), codes and
    // scales to registers a tile before they are staged.  Past the last tile the
    // pages are none, which read page 0 and stage it where nobody looks.
    uint4 rawk, rawv;
    float kraw = 0.f, vraw = 0.f;
    int page = -1;
    auto find = [&](int tile) __attribute__((always_inline)) {
      const int tok = tile * T + tid * 16;
      if (tid < G) page = tile < t1 && tok < len ? (int)page_of(c, b, tok >> pshift) : -1;
    };
    auto keep = [&](int tile) __attribute__((always_inline)) {
      if (tid < G) s_page[tile & 7][tid] = page;
    };
    const int krow = tid / (D / 16), kcol = tid % (D / 16);  // the thread's 16 codes of K
    const int vd = tid / G, vg = tid % G;                    // ... and of V: column, group
    auto load_pages = [&](int tile, int pk, int pv) __attribute__((always_inline)) {
      rawk = *reinterpret_cast<const uint4 *>(kbase + (uint64_t)(uint32_t)(pk < 0 ? 0 : pk) * pstride +
                                              (uint32_t)(((tile * T + krow) & (P - 1)) * D + kcol * 16));
      rawv = *reinterpret_cast<const uint4 *>(vbase + (uint64_t)(uint32_t)(pv < 0 ? 0 : pv) * pstride +
                                              (uint32_t)((vd << pshift) + ((tile * T + vg * 16) & (P - 1))));
    };
    auto load = [&](int tile) __attribute__((always_inline)) {
      load_pages(tile, s_page[tile & 7][krow >> 4], s_page[tile & 7][vg]);
    };
    // as 16-bit operands
    const int kput = krow * (2 * D) + pslot<Cfg::KC>(krow, 2 * kcol) * 16;
    const int vput = vg / VG * (VT * D * 2) + vd * (2 * VT) + pslot<Cfg::VC>(vd, 2 * (vg % VG)) * 16;
    auto stage = [&](int tile) __attribute__((always_inline)) {
      uint8_t *kb = lds + (tile & 1) * Cfg::STAGE, *vb = lds + VBASE + (tile & 1) * Cfg::STAGE;
      *reinterpret_cast<v4i *>(kb + kput) = codes8<FP8, F16>(rawk.x, rawk.y);
      *reinterpret_cast<v4i *>(kb + (kput ^ 16)) = codes8<FP8, F16>(rawk.z, rawk.w);
      *reinterpret_cast<v4i *>(vb + vput) = codes8<FP8, false>(rawv.x, rawv.z);
      *reinterpret_cast<v4i *>(vb + (vput ^ 16)) = codes8<FP8, false>(rawv.y, rawv.w);
    };
    // V that some row must not meet, in the thread's own staged codes: those past the
    // end or of no page, which can be NaN, become 0; NaN ones that a row may not see
    // move to s_nan.  (Here, not in registers before: that spilled.)
    auto clean = [&](int tile, int none) __attribute__((always_inline)) {
      if constexpr (FP8) {
        if (!(tile * T + T > every || __builtin_amdgcn_readfirstlane(none))) return;
        int t = tid;
        asm volatile("" : "+v"(t));
        const int d = t / G, g = t % G;
        const int nv = s_page[tile & 7][g] < 0 ? 0 : len - (tile * T + g * 16);
        uint8_t *row = lds + VBASE + (tile & 1) * Cfg::STAGE + g / VG * (VT * D * 2) + d * (2 * VT);
        uint32_t at = 0;
#pragma unroll 1
        for (int x = 0; x < 8; ++x) {            // two tokens of a chunk: half x / 4, word x % 4
          uint32_t *w = reinterpret_cast<uint32_t *>(row + pslot<Cfg::VC>(d, 2 * (g % VG) + (x >> 2)) * 16) + (x & 3);
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
        reinterpret_cast<Piece16 *>(&s_nan[tile & 1][g / VG][d])[g % VG] = (Piece16)at;
        if (__any(at) && lane == 0) s_bad[tile & 3] = 1;
      }
    };
    // the scales: G threads of wave 1
    const int sg = tid - 64;
    auto load_scales = [&](int tile) __attribute__((always_inline)) {
      if (sg >= 0 && sg < G) {
        const int pg = s_page[tile & 7][sg];
        const int64_t at = (int64_t)(pg < 0 ? 0 : pg) * c.heads + head;
        kraw = c.k_scale[at];
        vraw = c.v_scale[at];
      }
    };
    auto stage_scales = [&](int tile) __attribute__((always_inline)) {
      if (sg >= 0 && sg < G) {
        const bool none = s_page[tile & 7][sg] < 0;
        const float ks = none ? 0.f : kraw * (p.scale * kLog2e), vs = none ? 1.f : vraw;
        const bool odd = !(vs >= 0x1p-60f && vs <= 0x1p60f);
        s_ks[tile & 3][sg] = ks;
        s_vs[tile & 3][sg] = odd ? vs : 1.f;
        s_log[tile & 3][sg] = odd ? 0.f : __builtin_amdgcn_logf(vs);
        s_inv[tile & 3][sg] = odd ? 1.f : __builtin_amdgcn_rcpf(vs);
        const uint64_t ok = __ballot(none || !(ks >= 0.f)), ov = __ballot(odd);
        if (sg == 0) s_odd[tile & 3] = (ok != 0) | (ov != 0) << 1;
      }
    };
    // what a wave does for later tiles around the output's products of `tile`
    auto advance = [&](int tile, auto between) __attribute__((always_inline)) {
      // (read ahead of the products: each wait would be exposed behind them)
      const int none = FP8 ? s_none[(tile + 1) & 7] : 0, bad = FP8 ? s_bad[tile & 3] : 0;
      const int pk = s_page[(tile + 2) & 7][krow >> 4], pv = s_page[(tile + 2) & 7][vg];
      between(bad);
      stage(tile + 1);
      load_pages(tile + 2, pk, pv);
      clean(tile + 1, none);
      if (wave == 0) {
        if (FP8 && tid == 0) s_bad[(tile + 2) & 3] = 0;      // set behind the next barrier at the earliest
        keep(tile + 3);
        if constexpr (FP8) {
          const uint64_t none = __ballot(tid < G && page < 0);
          if (tid == 0) s_none[(tile + 3) & 7] = none != 0;
        }
        find(tile + 4);
      }
      if (wave == 1) {
        stage_scales(tile + 1);
        load_scales(tile + 2);
      }
    };

    __syncthreads();                             // the last block's readers
    if (tid < 4) s_bad[tid] = 0;
    if (tid < 8) s_none[tid] = 1;                // (the first tiles: as if)
    if constexpr (FP8) {
      for (int i = tid; i < Cfg::ROWS * (D / 32); i += Cfg::NT) s_row[i / (D / 32)][i % (D / 32)] = 0;
    }
    if (t0 < t1) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        find(t0 + i);
        keep(t0 + i);
      }
      __syncthreads();
      load(t0);
      load_scales(t0);
      stage(t0);
      clean(t0, 1);
      stage_scales(t0);
      load(t0 + 1);
      load_scales(t0 + 1);
      find(t0 + 3);
    }
    // the queries have arrived before the loop: a wait for them there would be one
    // for the tiles' loads too
#pragma unroll
    for (int k = 0; k < KK; ++k) asm volatile("" : "+v"(qf[k]));

    // fragment addresses: the rows' swizzles do not depend on t and d, and flip no
    // bit of 32 k, so one register each; formed afresh in every tile (kept for all
    // k they spill)
    const int kat0 = r32 * (2 * D) + pslot<Cfg::KC>(r32, h) * 16;
    const int vat0 = (half * Cfg::DH + r32) * (2 * VT) + pslot<Cfg::VC>(r32, h) * 16;
    v16f sc[TS];
    float kq[G], off[G];                         // the scores' factors; log2 vs - m
    int odd = 0;                                 // s_odd of the scores' tile
    // S^T, four fragments ahead of the products that take them
    auto scores = [&](int tile) __attribute__((always_inline)) {
      const uint8_t *kb = lds + (tile & 1) * Cfg::STAGE;
      int kat = kat0;
      asm volatile("" : "+v"(kat));
      constexpr int NF = KK * TS, PER = 4;       // fragment f: step f / TS, part f % TS of the tokens
      v4i a[2][PER];
      auto read = [&](int n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int f = n * PER + i;
          a[n & 1][i] = *reinterpret_cast<const v4i *>(kb + (kat ^ (32 * (f / TS))) + (f % TS) * 32 * 2 * D);
        }
      };
      read(0);
#pragma unroll
      for (int n = 0; n < NF / PER; ++n) {
        if (n + 1 < NF / PER) read(n + 1);
        __builtin_amdgcn_sched_barrier(0);
        wait_reads<PER>(n + 1 < NF / PER);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int f = n * PER + i;
          sc[f % TS] = mfma32<F16>(a[n & 1][i], qf[f / TS], f >= TS ? sc[f % TS] : (v16f){});
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // True where the scores need no `settle`: no token hidden from a row, no scale
    // off the common path, no row's maximum grown by more than 2^16.  (Of a row that has
    // none yet, all scores minus infinity, the difference is NaN: settle.)
    auto common = [&](int tile) __attribute__((always_inline)) {
      odd = s_odd[tile & 3];
      float top = -INFINITY;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        kq[g] = s_ks[tile & 3][g];
        off[g] = s_log[tile & 3][g] - m;
        float x = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i += 2) x = fmaxf(fmaxf(x, sc[g >> 1][8 * (g & 1) + i]), sc[g >> 1][8 * (g & 1) + i + 1]);
        top = fmaxf(top, x * kq[g]);
      }
      top = halves_max(top);
      return !__builtin_amdgcn_readfirstlane((int)(__any(!(top - m <= 16.f)) || odd || tile * T + T > low));
    };
    // In general: scores to powers of two, -infinity where hidden; sum and output to
    // their maximum.  (Outside the loop of the common tiles: there, the compiler kept
    // a second copy of the output and moved all of it in every tile.)
    auto settle = [&](int tile) __attribute__((always_inline)) {
      odd = s_odd[tile & 3];
      const int lim = limit - tile * T - 4 * h;
      float top = m;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float ks = s_ks[tile & 3][g];
        const bool there = s_page[tile & 7][g] >= 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = sc[g >> 1][8 * (g & 1) + i] * ks;
          const float x = 16 * g + 8 * (i >> 2) + (i & 3) < lim && there ? v : -INFINITY;
          sc[g >> 1][8 * (g & 1) + i] = x;
          top = fmaxf(top, x);
        }
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
        off[g] = s_log[tile & 3][g] - ref;
      }
    };
    v4i pf[G], pl[F16 ? G : 1];
    auto exponentials = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float e[8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // exp(s - m) vs from one exponential; the sum takes 1 / vs
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[g >> 1][8 * (g & 1) + i], kq[g], off[g]));
          sum = i ? sum + e[i] : e[i];
        }
        l = __builtin_fmaf(sum, s_inv[tile & 3][g], l);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t hi = pack_bf16x2(e[2 * w], e[2 * w + 1]);
          pf[g][w] = (int)hi;
          if constexpr (F16) pl[g][w] = (int)pack_bf16x2(e[2 * w] - u2f(hi << 16), e[2 * w + 1] - u2f(hi & 0xffff0000u));
        }
      }
      asm volatile("" : "+v"(l));                // here, not where l is used: the terms would be kept until then
    };
    auto output = [&](int tile, int bad) __attribute__((always_inline)) {
      const uint8_t *vb = lds + VBASE + (tile & 1) * Cfg::STAGE;
      int vat = vat0;
      asm volatile("" : "+v"(vat));
      constexpr int NF = G * DT, PER = 4;        // fragment f: group f / DT, columns f % DT
      v4i a[2][PER];
      auto read = [&](int n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int g = (n * PER + i) / DT, d = (n * PER + i) % DT;
          a[n & 1][i] = *reinterpret_cast<const v4i *>(vb + g / VG * (VT * D * 2) + (vat ^ (32 * (g % VG))) + d * 32 * 2 * VT);
        }
      };
      read(0);
#pragma unroll
      for (int n = 0; n < NF / PER; ++n) {
        if (n + 1 < NF / PER) read(n + 1);
        __builtin_amdgcn_sched_barrier(0);
        wait_reads<PER>(n + 1 < NF / PER);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int g = (n * PER + i) / DT, d = (n * PER + i) % DT;
          o[d] = mfma32<false>(a[n & 1][i], pf[g], o[d]);
          if constexpr (F16) o[d] = mfma32<false>(a[n & 1][i], pl[g], o[d]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (FP8) {
        if (__builtin_amdgcn_readfirstlane(bad)) {   // columns that get a NaN
          const int n = limit - tile * T;
#pragma unroll 1
          for (int d = half * Cfg::DH + h; d < (half + 1) * Cfg::DH; d += 2)
#pragma unroll 1
            for (int x = 0; x < T / VT; ++x) {
              const int k = n - x * VT < VT ? n - x * VT : VT;   // (bits past VT are not written)
              const uint64_t seen = k >= 64 ? ~0ull : (k > 0 ? (1ull << k) - 1 : 0);
              if (s_nan[tile & 1][x][d] & seen) atomicOr(&s_row[wrow + r32][d >> 5], 1u << (d & 31));
            }
        }
      }
    };
    auto odd_scales = [&](int tile) __attribute__((always_inline)) {   // those that no logarithm is taken of
      if (__builtin_amdgcn_readfirstlane(odd) & 2) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float vs = s_vs[tile & 3][g];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            // (two roundings to bf16 in such a tile; fp16's two parts are joined first)
            float a = u2f((uint32_t)pf[g][w] << 16), z = u2f((uint32_t)pf[g][w] & 0xffff0000u);
            if constexpr (F16) {
              a += u2f((uint32_t)pl[g][w] << 16);
              z += u2f((uint32_t)pl[g][w] & 0xffff0000u);
            }
            a = a == 0.f ? 0.f : a * vs;
            z = z == 0.f ? 0.f : z * vs;
            const uint32_t hi = pack_bf16x2(a, z);
            pf[g][w] = (int)hi;
            if constexpr (F16) pl[g][w] = (int)pack_bf16x2(a - u2f(hi << 16), z - u2f(hi & 0xffff0000u));
          }
        }
      }
    };

    if (t0 < t1) {
      // One barrier per tile.  (A SIMD's second wave half a tile behind the first, so
      // that one's products always ran beside the other's exponentials, was slower:
      // 270 against 255 us.)
      lds_barrier();
      int tile = t0;
      if (t0 < w1) {
        scores(t0);
        bool more = true;
        do {
          settle(tile);
          for (;;) {
            exponentials(tile);
            odd_scales(tile);
            advance(tile, [&](int bad) __attribute__((always_inline)) { output(tile, bad); });
            lds_barrier();
            if (++tile >= w1) {
              more = false;
              break;
            }
            scores(tile);
            if (!common(tile)) break;
          }
        } while (more);
      }
      for (; tile < t1; ++tile) {                // no row of this wave sees more
        advance(tile, [](int) {});
        lds_barrier();
      }
    }
    if constexpr (FP8) {
      // (of no tile: no barrier since other waves cleared s_row, and nothing in it)
      if (t0 < t1) {
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
        if (t0 < t1) {                           // (a part of no tile has no sums)
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<v4f *>(p.ws + at * D + col + 32 * d + 8 * q) =
                  (v4f){o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
        }
        if (h == 0 && half == 0) {
          float *ml = p.ws + (int64_t)nsplit * n * D + at * 2;
          ml[0] = l == l ? m : l;                // (attn_join_prompt_kernel skips a part without a maximum)
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
static hipError_t launch_prompt_cfg(const KvCacheArgs &c, const AttnArgs &p, int nblk, int nsplit, int part, hipStream_t st) {
  const dim3 grid((unsigned)(nblk * c.heads * c.seqs), (unsigned)nsplit);
  attn_prompt_kernel<SRC, FP8, D><<<grid, PromptCfg<D>::NT, 0, st>>>(c, p, nblk, nsplit, part);
  return hipGetLastError();
}

int attn_prompt_rows(int dim) { return dim > 128 ? PromptCfg<256>::ROWS : PromptCfg<128>::ROWS; }

hipError_t launch_attn_prompt(int src, const KvCacheArgs &c, const AttnArgs &p, int nblk, int nsplit, int part, hipStream_t st) {
  auto go = [&](auto src_tag, auto fp8_tag) {
    constexpr int S = decltype(src_tag)::value;
    constexpr bool F = decltype(fp8_tag)::value;
    if (c.dim == 64) return launch_prompt_cfg<S, F, 64>(c, p, nblk, nsplit, part, st);
    if (c.dim == 128) return launch_prompt_cfg<S, F, 128>(c, p, nblk, nsplit, part, st);
    return launch_prompt_cfg<S, F, 256>(c, p, nblk, nsplit, part, st);
  };
  using B = std::integral_constant<int, SRC_BF16>;
  using H = std::integral_constant<int, SRC_F16>;
  if (src == SRC_BF16) return c.fp8 ? go(B{}, std::true_type{}) : go(B{}, std::false_type{});
  return c.fp8 ? go(H{}, std::true_type{}) : go(H{}, std::false_type{});
}

}  // namespace dsl
