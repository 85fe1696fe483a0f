// Attention where groups of sequences share a prefix, over the paged 8-bit
// cache; attn_core.h has the mathematics and the row order.
//
// A group's sequences hold the same pages for its first E tokens (whole pages).
// Their query rows stand together, so the prefix is the context of one unit with
// all of the group's rows, read once for 16, 32 or 64 of them instead of once per
// sequence; what lies behind it is each sequence's own.  Units stand in lines of
// rounds of 256 tokens, of which workgroups take equal runs, as in attn.hip: up to
// 16 rows to a group both kinds in one line, else prefixes in one and own tokens in
// another, at the same time or in a launch of their own.  Every row has parts of both; a second
// kernel joins them in their order.  A row sees of the prefix what its length and
// its position allow, so rows of sequences that are shorter than it, or empty, are
// right too.
#include "attn_tile.h"
#include "launch.h"

#include <cstdlib>
#include <type_traits>

namespace dsl {

constexpr int kMaxRuns = 512, kPad = 4;

// The workspace.  The beginning of a unit is kept by its rows, the first of two
// for each query row and head's prefix and own tokens; what a run holds of a unit
// that began before it (one at most) by the run.
struct SharedParts {
  float *first;                  // [row][query head][2][D]
  float2 *first_ml;              // [row][query head][2]: maxima and sums
  int2 *where;                   // ...: (run of the beginning, or -1: no part; last run * 64 + row of its block)
  // of prefixes and of own tokens, the same where one line has both
  float *more[2];                // [run][ROWS][D]
  float2 *more_ml[2];            // [run][ROWS]
  int runs[2], rows[2];
};
enum { UNITS_PREFIX = 1, UNITS_OWN = 2 };        // what a line has

// Tokens of group g's prefix: whole pages that the table has room for.
DSL_DEV int prefix_of(const KvCacheArgs &c, const SharedArgs &h, int g) {
  const int n = h.shared[g], room = c.width * c.page;
  return (n < 0 ? 0 : n < room ? n : room) & -c.page;
}
DSL_DEV int group_start(const KvCacheArgs &c, const SharedArgs &h, int g) {
  const int b = h.groups[g];
  return b < 0 ? 0 : b > c.seqs ? c.seqs : b;
}
DSL_DEV int first_row(const KvCacheArgs &c, int b) {
  const int v = c.starts ? c.starts[b] : b;
  return v < 0 ? 0 : v > c.rows ? c.rows : v;
}
// The largest of each N lanes (16, 32 or 64).  (No shuffles: what their addresses
// are made of would be kept through the walk, and spill.)
template <int N>
DSL_DEV int lanes_most(int v) {
  auto most = [](int a, int b) { return a > b ? a : b; };
  v = most(v, __builtin_amdgcn_update_dpp(v, v, 0xb1, 0xf, 0xf, false));    // lanes ^ 1, ^ 2, then mirrors of 8 and 16
  v = most(v, __builtin_amdgcn_update_dpp(v, v, 0x4e, 0xf, 0xf, false));
  v = most(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, false));
  v = most(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xf, 0xf, false));
  if constexpr (N >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = most((int)a[0], (int)a[1]);
  }
  if constexpr (N >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    v = most((int)a[0], (int)a[1]);
  }
  return v;
}
DSL_DEV int one(int v) { return __builtin_amdgcn_readfirstlane(v); }
// The last i of 0 .. n - 1 with at(i) <= x, or -1.
template <class F>
DSL_DEV int last_upto(int n, int x, const F &at) {
  int lo = -1, hi = n;
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (at(mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}
// Tokens of sequence b's prefix.
DSL_DEV int prefix_behind(const KvCacheArgs &c, const SharedArgs &h, int b) {
  const int g = last_upto(h.n, b, [&](int i) { return h.groups[i]; });
  return g >= 0 && b < h.groups[g + 1] ? prefix_of(c, h, g) : 0;
}

// Unit u of the line: a group's prefix (u < groups), then a sequence's own tokens.
struct SharedUnit {
  int rows0, n;                  // rows of the token tensors
  int off, len;                  // tokens off .. len - 1 (of a prefix: 0 .. len - 1)
  int from;                      // the sequence whose table row has them (-1: a longer one than the group's first)
};
DSL_DEV SharedUnit shared_unit(const KvCacheArgs &c, const SharedArgs &h, int u) {
  SharedUnit s;
  if (u < h.n) {
    const int b0 = group_start(c, h, u), b1 = group_start(c, h, u + 1);
    s.rows0 = first_row(c, b0);
    const int end = b1 > b0 ? first_row(c, b1) : s.rows0;
    s.n = end > s.rows0 ? end - s.rows0 : 0;
    s.off = 0;
    s.len = prefix_of(c, h, u);
    s.from = b1 > b0 && c.lens[b0] >= s.len ? b0 : -1;
  } else {
    const SeqView v = seq_view(c, u - h.n);
    s.rows0 = v.row0;
    s.n = v.n;
    s.off = prefix_behind(c, h, u - h.n);
    s.len = v.len;
    s.from = u - h.n;
  }
  return s;
}

// The line of all units' rounds: by unit, cache head, row block.  64 units are looked
// at at a time; what a wave knows of them is in shared memory (the same for all waves),
// not in registers, which a walk needs.
struct LineUnits {
  int rounds[64], blocks[64], upto[64];          // of a unit; the line's length up to and with it, from the first of the 64
  SharedUnit unit[64];
};
struct SharedLine {
  const KvCacheArgs &c;
  const SharedArgs &h;
  LineUnits &in;
  const int group, block, chunk, begin, units;     // rows of a block; tiles of a round
  int per;                       // rounds that a unit's are rounded up to
  int at, before, total;         // the first of the 64; the line's length before them, theirs
  DSL_DEV SharedLine(const KvCacheArgs &c, const SharedArgs &h, LineUnits &in, int group, int block, int chunk, int what)
      : c(c), h(h), in(in), group(group), block(block), chunk(chunk), begin(what & UNITS_PREFIX ? 0 : h.n),
        units(what & UNITS_OWN ? h.n + c.seqs : h.n), per(1), at(begin - 64), before(0), total(0) {}
  // What the lanes have of the 64, rounds rounded up, into shared memory.
  DSL_DEV void put(int lane, int rounds, int blocks) {
    rounds = (rounds + per - 1) / per * per;
    const int upto = lanes_sum(rounds * c.heads * blocks);
    total = __builtin_amdgcn_readlane(upto, 63);
    __syncthreads();                             // the last 64's readers
    in.rounds[lane] = rounds;
    in.blocks[lane] = blocks;
    in.upto[lane] = upto;
  }
  DSL_DEV void advance() {
    before += total;
    at += 64;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, u = at + lane;
    int rounds = 0, blocks = 0;
    SharedUnit s{};
    if (u < units) {
      s = shared_unit(c, h, u);
      const int room = c.width * c.page, len = s.len < room ? s.len : room;
      const int tiles = len > s.off ? (len - s.off + kTile - 1) / kTile : 0;
      rounds = (tiles + chunk - 1) / chunk;
      if (u >= h.n && rounds == 0) rounds = 1;   // of no token: one, for its parts
      blocks = rounds ? (int)(((int64_t)s.n * group + block - 1) / block) : 0;
    }
    put(lane, rounds, blocks);
    in.unit[lane] = s;
    __syncthreads();
  }
  DSL_DEV void rewind() {
    at = begin - 64;
    before = total = 0;
    advance();
  }
  // The rounds of a run, of `runs` equal ones; back to the line's beginning.  A run that
  // holds the end of a unit and the beginning of the next takes up two (about 8 us):
  // units' rounds are rounded up to whole runs where runs no more than kPad rounds longer
  // hold them so (prefixes of 30000 tokens, 32 samples: 44 us unrounded, 39 rounded).
  DSL_DEV int length() {
    while (at + 64 < units) advance();
    return one(before + total);
  }
  DSL_DEV int share(int runs) {
    const int least = one((length() + runs - 1) / runs);
    if (least <= 1) {
      if (at > begin) rewind();
      return least;
    }
    int need[kPad + 1] = {};
    if (at > begin) rewind();
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
    int r, n;
    for (;;) {
      r = in.rounds[lane];
      n = in.blocks[lane];
#pragma unroll
      for (int k = 0; k <= kPad; ++k)
        need[k] += __builtin_amdgcn_readlane(lanes_sum(n * c.heads * ((r + least + k - 1) / (least + k))), 63);
      if (at + 64 >= units) break;
      advance();
    }
    int share = least;
#pragma unroll
    for (int k = kPad; k >= 0; --k)
      if (need[k] <= runs) share = per = least + k;
    if (at > begin) {
      rewind();
    } else if (per > 1) {
      put(lane, r, n);
      __syncthreads();
    }
    return share;
  }
  // The unit of position x, not before an earlier one; its rounds and row
  // blocks, and x in it.  (-1: none, of groups or starts that do not ascend.)
  DSL_DEV int find(int x, int &ur, int &ub, int &off, SharedUnit &s) {
    while (x >= before + total && at + 64 < units) advance();
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int upto = in.upto[tid & 63];
    const uint64_t past = __ballot(before + upto > x);
    if (!past) return -1;
    const int k = __builtin_ctzll(past);
    ur = __builtin_amdgcn_readfirstlane(in.rounds[k]);
    ub = __builtin_amdgcn_readfirstlane(in.blocks[k]);
    off = x - before - __builtin_amdgcn_readlane(upto, k) + ur * c.heads * ub;
    s = in.unit[k];
    s = SharedUnit{one(s.rows0), one(s.n), one(s.off), one(s.len), one(s.from)};
    return at + k;
  }
};

// Up to 16 rows of a unit, by attn.hip's walk.
template <int SRC_, bool FP8_, int D_>
struct FewWalk : RowsWalk<SRC_ == SRC_F16, FP8_, D_, 1> {
  static constexpr int SRC = SRC_, D = D_, NB = 1, BLOCK = 16, ROWS = 16, WGS = rows_wgs(D, 1);
  static constexpr bool FP8 = FP8_;
  using Base = RowsWalk<SRC_ == SRC_F16, FP8_, D_, 1>;
  static constexpr bool SHARED = false;          // (queries in registers)
  typedef int Queries;
  DSL_DEV explicit FewWalk(Queries &) {}
  float qs[NB];
  DSL_DEV float load(int b, const uint16_t *q) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int y = 0; y < D / 64; ++y)
#pragma unroll
      for (int z = 0; z < 2; ++z) this->qf[b][2 * y + z] = *reinterpret_cast<const v4i *>(q + 64 * y + 16 * g + 8 * z);
    return 1.f;
  }
  DSL_DEV void walk(const KvCacheArgs &c, const Context &ctx, float scale, int head, int t0, int t1, int lo, Word16 *) {
    Base::walk(c, ctx, scale, true, head, t0, t1, lo);
  }
};
template <class Walk>
struct JoinOf {
  using type = TileJoin<Walk::D, Walk::ROWS>;
};
template <int SRC, bool FP8, int D>
struct JoinOf<FewWalk<SRC, FP8, D>> {
  using type = RowsJoin<D>;
};
template <class Walk, class G, class R, class F>
DSL_DEV void join_waves(TileJoin<Walk::D, Walk::ROWS> &sh, const Walk &w, int rows, const G &restore, const R &row_sums,
                        const F &emit) {
  join_tiles(sh, w, rows, restore, row_sums, emit);
}
template <class Walk, class G, class R, class F>
DSL_DEV void join_waves(RowsJoin<Walk::D> &sh, const Walk &w, int rows, const G &, const R &row_sums, const F &emit) {
  join_rows<Walk::D, 1>(sh, w, rows, [&](int, int row, int col, const v4f &v, float m, float l) {
    if (col == 0) row_sums(row, m, l);
    emit(row, col, v);
  });
}

// Workgroups go to the eight XCDs in turn: each XCD takes a piece of the line, so that
// the row blocks of a head, which read the same tokens, share its L2.
DSL_DEV int run_of(int block, int runs) { return runs % 8 == 0 ? block % 8 * (runs / 8) + block / 8 : block; }

// What a workgroup's walk of a line needs of shared memory.
template <class Walk>
struct WalkRoom {
  __align__(16) typename JoinOf<Walk>::type sh;
  __align__(16) typename Walk::Queries queries;
  int limit[Walk::ROWS];                         // (every wave writes all)
  float2 row[Walk::NB][Walk::BLOCK];             // what a row's queries were divided by, the tokens it sees
};

// Run `run` of `runs` equal ones of a line.
template <class Walk>
DSL_DEV void walk_run(const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, const SharedParts &part, int chunk,
                      SharedLine &line, WalkRoom<Walk> &room_, int run, int runs) {
  constexpr int D = Walk::D, ROWS = Walk::ROWS, BLOCK = Walk::BLOCK, NB = Walk::NB;
  auto &sh = room_.sh;
  auto &queries = room_.queries;
  auto &s_limit = room_.limit;
  auto &s_row = room_.row;
  const int per = line.share(runs);
  int x = run * per;
  const int end = x + per;

  while (x < end) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));                // (what is made of it is formed in each unit: kept, it spills)
    const int lane = tid & 63, mine = lane & (BLOCK - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int rounds, blocks, off;
    SharedUnit s;
    const int u = line.find(x, rounds, blocks, off, s);
    if (u < 0) return;
    const bool prefix = u < h.n;
    // (one number for the wave, each: in scalar registers)
    const int unit = one(off / rounds), r0 = off - unit * rounds, head = one(unit / blocks), rb = unit - head * blocks;
    const int left = rounds - r0, count = left < end - x ? left : end - x;
    x += count;
    const int rows = s.n * p.group, room = c.width * c.page, seen = s.len < room ? s.len : room;
    // whose table row, from which page on; tokens of it
    int from = s.from;
    if (from < 0) {
      // the group's first sequence that is as long as the prefix, else the longest
      const int b0 = group_start(c, h, u), b1 = group_start(c, h, u + 1);
      int best = -1;
      from = b0;
      for (int b = b0; b < b1 && best < s.len; b += 64) {
        const int at = b + lane, n = at < b1 ? c.lens[at] : -1;
        const uint64_t enough = __ballot(n >= s.len);
        if (enough) {
          best = s.len;
          from = b + __builtin_ctzll(enough);
          break;
        }
        const int most = lanes_most<64>(n);
        if (most > best) {
          best = most;
          from = b + __builtin_ctzll(__ballot(n == most));
        }
      }
      from = one(from);
    }
    const int skip = one(s.off / c.page);
    const Context ctx{c.table + (int64_t)from * c.table_ld + skip, c.width - skip, s.len - s.off};
    Walk w(queries);
    if constexpr (Walk::SHARED) w.limit = s_limit;
    // A row of the block: its queries, and the tokens of the unit that it sees; by
    // one wave for all where they share them.
    auto row_of = [&](int k) __attribute__((always_inline)) {
      const int r = rb * ROWS + k * BLOCK + mine, rr = r < rows ? r : rows - 1;
      const int i = rr / p.group, hq = head * p.group + rr % p.group, row = s.rows0 + i;
      const float by = w.load(k, static_cast<const uint16_t *>(p.q) + (int64_t)row * p.q_row + (int64_t)hq * p.q_head);
      int b = u - h.n;
      if (prefix) b = c.starts ? last_upto(c.seqs, row, [&](int j) { return first_row(c, j); }) : row;
      const SeqView v = seq_view(c, b);
      int n = p.causal ? v.first + (row - v.row0) + 1 : v.len;
      n = (n < seen ? n : seen) - s.off;
      s_row[k][mine] = make_float2(by, __builtin_bit_cast(float, n > 0 ? n : 0));
    };
    if (Walk::SHARED) {
      if (wave < NB) row_of(wave);
      __syncthreads();
    } else {
      row_of(0);
    }
    int lo = 0x7fffffff, high = 0;               // tokens that every other row sees, that some row sees
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const float2 x = s_row[k][mine];
      const int n = __builtin_bit_cast(int, x.y);
      w.qs[k] = x.x;
      // (a row that sees no token of the unit keeps no tile off the common path: it goes
      // along, and is cleared)
      const int limit = n == 0 ? 0x7fffffff : n;
      if constexpr (Walk::SHARED) s_limit[k * BLOCK + mine] = limit;
      else w.limit[k] = limit;
      lo = lo < limit ? lo : limit;
      high = high > n ? high : n;
    }
    lo = __builtin_amdgcn_readfirstlane(-lanes_most<BLOCK>(-lo));
    const int nsee = (__builtin_amdgcn_readfirstlane(lanes_most<BLOCK>(high)) + kTile - 1) / kTile;
    const int t0 = r0 * chunk, t1 = nsee - t0 > count * chunk ? t0 + count * chunk : nsee;
    w.walk(c, ctx, p.scale, head, t0, t1, lo, reinterpret_cast<Word16 *>(sh.so[wave]));
#pragma unroll
    for (int k = 0; k < NB; ++k)
      if (__builtin_bit_cast(int, s_row[k][mine].y) == 0) {
        w.m[k] = -INFINITY;
        w.l[k] = 0.f;
#pragma unroll
        for (int d = 0; d < (int)(sizeof(w.o[k]) / sizeof(w.o[k][0])); ++d)
#pragma unroll
          for (int i = 0; i < (int)(sizeof(w.o[k][0]) / sizeof(float)); ++i) w.o[k][d][i] = 0.f;
      }
    const int last = one(run + (left - count + per - 1) / per), kind = prefix ? 0 : 1;
    auto restore = [&](float *so) __attribute__((always_inline)) {
      if constexpr (Walk::SHARED)
        w.restore(c, ctx, head, t0, t1, so, [&](int r) { return __builtin_bit_cast(int, s_row[r / BLOCK][r % BLOCK].y); });
    };
    auto place = [&](int row) __attribute__((always_inline)) {       // of a row's beginning
      const int r = rb * ROWS + row, i = r / p.group;
      return 2 * ((s.rows0 + i) * p.q_heads + head * p.group + r - i * p.group) + kind;
    };
    join_waves(
        sh, w, rows - rb * ROWS, restore,
        [&](int row, float mr, float lr) __attribute__((always_inline)) {
          const float2 ml = make_float2(lr == lr ? mr : lr, lr);     // a NaN sum without a maximum stays NaN in the join
          if (r0 == 0) {
            const int at = place(row);
            part.first_ml[at] = ml;
            part.where[at] = make_int2(run, last * 64 + row);
            if (!prefix && s.off == 0) part.where[at - 1] = make_int2(-1, 0);
          } else {
            part.more_ml[kind][(int64_t)run * ROWS + row] = ml;
          }
        },
        [&](int row, int col, const v4f &v) __attribute__((always_inline)) {
          float *to = r0 == 0 ? part.first + (int64_t)place(row) * D : part.more[kind] + ((int64_t)run * ROWS + row) * D;
          *reinterpret_cast<v4f *>(to + col) = v;
        });
  }
}

// Both kinds of units in one line.
template <class Walk>
__global__ __launch_bounds__(256, Walk::WGS) void attn_shared_kernel(const KvCacheArgs c, const AttnArgs p,
                                                                     const SharedArgs h, const SharedParts part,
                                                                     const int chunk, const int what) {
  __shared__ WalkRoom<Walk> s_room;
  __shared__ LineUnits s_units;
  SharedLine line(c, h, s_units, p.group, Walk::ROWS, chunk, what);
  walk_run<Walk>(c, p, h, part, chunk, line, s_room, run_of(blockIdx.x, gridDim.x), gridDim.x);
}

// Prefixes by some of the workgroups, 32 or 64 rows a wave, own tokens by the others, 16
// rows a wave where no sequence has more.  (own_chunk 0: prefixes only.)  The workgroups
// are dealt by what the lines take: a round of either as much where a head has at most 128
// columns, one of own tokens twice that where it has 256; taking up a sequence's own tokens
// 1.5 rounds, or 1.  (128 columns, 8 heads, 32 sequences of 4 rows and 200 tokens behind a
// prefix of 10000 or 30000: 34 and 48 us; both kinds in one line of 64 rows 48 and 94, a
// launch for each kind 40 and 53.  256 columns, 64 sequences behind 30000: 133 us, dealt
// as for 128 columns 143.)
template <class Walk, class Own>
__global__ __launch_bounds__(256, 1) void attn_shared_two_kernel(const KvCacheArgs c, const AttnArgs p, const SharedArgs h,
                                                                 const SharedParts part, const int chunk,
                                                                 const int own_chunk) {
  __shared__ union Room {
    WalkRoom<Walk> prefix;
    WalkRoom<Own> own;
    DSL_DEV Room() {}
  } s_room;
  __shared__ LineUnits s_units;
  const int runs = gridDim.x;
  int few = 0;
  if (own_chunk > 0) {
    SharedLine own(c, h, s_units, p.group, Own::ROWS, own_chunk, UNITS_OWN);
    few = own.length();
  }
  SharedLine prefix(c, h, s_units, p.group, Walk::ROWS, chunk, UNITS_PREFIX);
  const float much = (float)prefix.length(), take = Walk::D <= 128 ? 1.5f : 1.f;
  const float rest = (float)few * (Walk::D <= 128 ? 1.f : 2.f) + (float)c.heads * c.seqs * take;
  const int step = runs % 8 || runs < 16 ? 1 : 8;          // (whole pieces of the line for the XCDs)
  int n = one((int)(much / (much + rest) * runs / step + 0.5f)) * step;
  n = n < step ? step : n > runs - step ? runs - step : n;
  if (much == 0.f) n = 0;
  if (own_chunk == 0) n = runs;
  const int block = blockIdx.x;
  if constexpr (std::is_same_v<Walk, Own>) {
    const bool mine = block < n;
    SharedLine line(c, h, s_units, p.group, Walk::ROWS, chunk, mine ? UNITS_PREFIX : UNITS_OWN);
    walk_run<Walk>(c, p, h, part, chunk, line, s_room.prefix, mine ? run_of(block, n) : run_of(block - n, runs - n),
                   mine ? n : runs - n);
  } else if (block < n) {
    walk_run<Walk>(c, p, h, part, chunk, prefix, s_room.prefix, run_of(block, n), n);
  } else {
    SharedLine line(c, h, s_units, p.group, Own::ROWS, own_chunk, UNITS_OWN);
    walk_run<Own>(c, p, h, part, own_chunk, line, s_room.own, run_of(block - n, runs - n), runs - n);
  }
}

// Joins the parts of one query row and head in a workgroup, as attn.hip's does: a
// part per lane for the maximum and the sum, then four columns per thread, the
// parts dealt to 1024 / D threads of each.
template <int SRC, int D>
__global__ __launch_bounds__(256) void attn_shared_join_kernel(const AttnArgs p, const SharedParts part) {
  constexpr int CG = D / 4, SL = 256 / CG;
  __shared__ float s_f[2 * kMaxRuns], s_red[8];
  __shared__ v4f s_v[SL][CG];
  const int64_t at = blockIdx.x;
  const int tid = threadIdx.x;
  // (A row of no sequence has what the workspace held: in bounds, and its result
  // is not specified.)
  auto span = [&](const int2 &w, int runs) {
    if (w.x < 0 || w.x >= runs) return 0;
    const int many = (w.y >> 6) - w.x + 1, most = runs - w.x;
    return many < 0 ? 0 : many < most ? many : most;
  };
  const int2 wp = part.where[2 * at], wo = part.where[2 * at + 1];
  const int np = span(wp, part.runs[0]), parts = np + span(wo, part.runs[1]);
  // part s: a row's beginning, or the run that holds more of it
  auto beginning = [&](int s) { return s == 0 && np > 0 ? 2 * at : s == np ? 2 * at + 1 : (int64_t)-1; };
  auto run_row = [&](int s) {
    const int kind = s < np ? 0 : 1;
    const int2 w = kind ? wo : wp;
    return (int64_t)(w.x + (kind ? s - np : s)) * part.rows[kind] + (w.y & (part.rows[kind] - 1));
  };
  auto max_sum = [&](int s) {
    const int64_t b = beginning(s);
    return b >= 0 ? part.first_ml[b] : part.more_ml[s < np ? 0 : 1][run_row(s)];
  };
  float top = -INFINITY, l = 0.f;
  auto weight = [&](const float2 &ml) {
    const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
    l += ml.y * f;
    return f;
  };
  const float *weights = s_f;
  // Up to 64 parts each wave looks through all, without barriers (3808 rows and heads of 64
  // columns: 7.6 us, with them 9.0).
  const bool few = parts <= 64;
  if (few) {
    const int lane = tid & 63, wave = tid >> 6;
    const float2 ml = lane < parts ? max_sum(lane) : make_float2(-INFINITY, 0.f);
    top = ml.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    s_f[wave * 64 + lane] = weight(ml);
    weights = s_f + wave * 64;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  } else {
    constexpr int U = 2 * kMaxRuns / 256;
    float2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ml[u] = tid + 256 * u < parts ? max_sum(tid + 256 * u) : make_float2(-INFINITY, 0.f);
      top = fmaxf(top, ml[u].x);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((tid & 63) == 0) s_red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
#pragma unroll
    for (int u = 0; u < U; ++u) s_f[tid + 256 * u] = weight(ml[u]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
    if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = l;
    __syncthreads();
    l = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  }
  const int cg = tid % CG, sl = tid / CG;
  v4f v = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = sl; s < parts; s += SL) {
    const int64_t b = beginning(s);
    v += *reinterpret_cast<const v4f *>((b >= 0 ? part.first + b * D : part.more[s < np ? 0 : 1] + run_row(s) * D) + cg * 4) * weights[s];
  }
  s_v[sl][cg] = v;
  __syncthreads();
  if (tid >= CG) return;
#pragma unroll
  for (int k = 1; k < SL; ++k) v += s_v[k][cg];
  const float inv = l > 0.f ? 1.0f / l : 0.f;    // a row that sees nothing is 0
  uint16_t *op = static_cast<uint16_t *>(p.o) + (at / p.q_heads) * p.o_row + (at % p.q_heads) * p.o_head + cg * 4;
  *reinterpret_cast<uint2 *>(op) = make_uint2(narrow2<SRC>(v[0] * inv, v[1] * inv), narrow2<SRC>(v[2] * inv, v[3] * inv));
}

// How units of a kind are walked: query rows of a block (16, 32 or 64 a wave),
// workgroups, tiles of a round.
struct SharedWalk {
  int rows, runs, chunk;
};
struct SharedPlan {
  SharedWalk prefix, own;
  bool apart;                    // own tokens in a launch of their own
  size_t bytes;                  // of the workspace
  SharedParts parts;             // in a workspace at 0
};
static SharedWalk shared_walk(const KvCacheArgs &c, int64_t group, int rows, int64_t kinds, int64_t many) {
  SharedWalk a{rows, (rows == 16 ? rows_wgs(c.dim, 1) : 1) * device_cu_count(), 4};
  a.runs = a.runs < 2 ? 2 : a.runs > kMaxRuns ? kMaxRuns : a.runs;
  // rounds of a tile per wave, longer ones where the line's length would pass an int
  const int64_t tiles = ((int64_t)c.width * c.page + kTile - 1) / kTile;
  const int64_t units = c.heads * (kinds * ((int64_t)c.rows * group / a.rows) + many);          // at most
  while ((tiles + a.chunk - 1) / a.chunk * units > 1 << 30 && a.chunk < tiles) a.chunk *= 2;
  return a;
}
static int rows_set(int dim) {
  const char *set = getenv("DSL_ATTN_SHARED_ROWS");    // read per launch (tests switch it)
  const int n = set ? atoi(set) : 0;
  return n == 16 || n == 32 || (n == 64 && dim <= 128) ? n : 0;
}
// A sequence whose own rows fill a workgroup of attn_prompt.hip gains nothing from the
// others': above 96 of them to a cache head (64 of 64 columns), attention as if nothing were shared.
// (128 columns behind 20000 tokens, shared and not: 96 rows of 4 sequences 108 and 120 us, of 32
// 635 and 698; 128 rows 112 and 101, 722 and 646; 256 rows 189 and 106, 1394 and 696.
// 64 columns: 64 rows 44 and 45, 281 and 259; 96 rows 75 and 64, 400 and 340.)
bool attn_shared_runs(int heads, int dim, int q_heads, int max_q) {
  return (int64_t)max_q * (q_heads / heads) <= (dim == 64 ? 64 : 96) || rows_set(dim);
}
static int shared_rows(const KvCacheArgs &c, int64_t rows) {
  if (const int n = rows_set(c.dim)) return n;
  // As many as a group has, but 64 above 64 only.  128 columns, 8 heads, behind 3000, 10000
  // and 30000 tokens, with 64 rows: 16 a wave 17.5, 33 and 57 us, 32 a wave 19, 25 and 37,
  // 64 a wave 24, 28 and 36; with 128 rows: 26, 54 and 116, 24, 34 and 61, 29, 33 and 47.
  // 256 columns have no registers for 64.
  return rows <= 16 ? 16 : rows <= 64 || c.dim > 128 ? 32 : 64;
}
static SharedPlan shared_plan(const KvCacheArgs &c, int groups, int q_heads, int max_q, int max_group) {
  SharedPlan a{};
  const int64_t group = q_heads / c.heads, most = (int64_t)max_q * max_group;
  const int64_t own = (max_q < c.rows ? max_q : c.rows) * group;
  const int rows = shared_rows(c, groups ? (most < c.rows ? most : c.rows) * group : own);
  const bool same = rows == 16 || groups == 0;    // no prefixes, or both kinds of units in one line
  a.prefix = shared_walk(c, group, rows, same ? 2 : 1, (same ? c.seqs : 0) + (int64_t)groups);
  a.own = same ? a.prefix : shared_walk(c, group, own <= 16 ? 16 : rows, 1, c.seqs);
  // Own tokens at the same time as the prefixes cost no launch of their own (6 to 10 us),
  // but have a workgroup on a CU where two or more go: a launch of their own from more of
  // them than CUs.  128 columns, 8 heads, behind 30000 tokens, 200 and 4000 own ones, at the
  // same time and apart: 6 sequences 29 and 37 us, 33 and 39; 32: 47 and 55, 79 and 79;
  // 64: 77 and 77, 153 and 137.
  a.apart = !same && a.own.rows == 16 && (int64_t)c.heads * c.seqs > device_cu_count();
  const size_t n = (size_t)c.rows * q_heads;
  size_t at = 0;
  auto room = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 15) & ~(size_t)15;
    return p;
  };
  auto put = [&](auto *&p, size_t bytes) { p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(room(bytes)); };
  put(a.parts.first, 2 * n * c.dim * sizeof(float));
  put(a.parts.first_ml, 2 * n * sizeof(float2));
  put(a.parts.where, 2 * n * sizeof(int2));
  for (int k = 0; k < 2; ++k) {
    const SharedWalk &w = k ? a.own : a.prefix;
    a.parts.runs[k] = w.runs;
    a.parts.rows[k] = w.rows;
    if (k && same) {
      a.parts.more[k] = a.parts.more[0];
      a.parts.more_ml[k] = a.parts.more_ml[0];
    } else {
      put(a.parts.more[k], (size_t)w.runs * w.rows * c.dim * sizeof(float));
      put(a.parts.more_ml[k], (size_t)w.runs * w.rows * sizeof(float2));
    }
  }
  a.bytes = at;
  return a;
}

size_t attn_shared_workspace_bytes(const KvCacheArgs &c, int groups, int q_heads, int max_q, int max_group) {
  if (!attn_shared_runs(c.heads, c.dim, q_heads, max_q)) return attn_workspace_bytes(c, q_heads, max_q) + 16;      // (never empty)
  return shared_plan(c, groups, q_heads, max_q, max_group).bytes;
}

template <class Walk, class Few>
static void launch_shared_tiles(const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, const SharedPlan &a,
                                hipStream_t st) {
  const unsigned n = (unsigned)a.prefix.runs;
  if (a.own.rows == 16) {
    attn_shared_two_kernel<Walk, Few><<<n, 256, 0, st>>>(c, p, h, a.parts, a.prefix.chunk, a.apart ? 0 : a.own.chunk);
    if (a.apart) attn_shared_kernel<Few><<<(unsigned)a.own.runs, 256, 0, st>>>(c, p, h, a.parts, a.own.chunk, UNITS_OWN);
  } else attn_shared_two_kernel<Walk, Walk><<<n, 256, 0, st>>>(c, p, h, a.parts, a.prefix.chunk, a.own.chunk);
}
template <int SRC, bool FP8, int D>
static void launch_shared_units(const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, const SharedPlan &a,
                                hipStream_t st) {
  using Few = FewWalk<SRC, FP8, D>;
  const bool whole = c.page >= kTile;
  if (a.prefix.rows == 16) 
    attn_shared_kernel<Few><<<(unsigned)a.prefix.runs, 256, 0, st>>>(c, p, h, a.parts, a.prefix.chunk, UNITS_PREFIX | UNITS_OWN);
  else if (a.prefix.rows == 32) {
    if (whole) launch_shared_tiles<TileWalk<SRC, FP8, D, 1, true>, Few>(c, p, h, a, st);
    else launch_shared_tiles<TileWalk<SRC, FP8, D, 1, false>, Few>(c, p, h, a, st);
  } else if constexpr (D <= 128) {
    if (whole) launch_shared_tiles<TileWalk<SRC, FP8, D, 2, true>, Few>(c, p, h, a, st);
    else launch_shared_tiles<TileWalk<SRC, FP8, D, 2, false>, Few>(c, p, h, a, st);
  }
}
template <int SRC, bool FP8, int D>
static hipError_t launch_shared_dim(const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, hipStream_t st) {
  SharedPlan a = shared_plan(c, h.n, p.q_heads, p.max_q, h.most);
  const uintptr_t ws = reinterpret_cast<uintptr_t>(p.ws);
  auto move = [&](auto *&x) { x = reinterpret_cast<std::remove_reference_t<decltype(x)>>(reinterpret_cast<uintptr_t>(x) + ws); };
  move(a.parts.first);
  move(a.parts.first_ml);
  move(a.parts.where);
  for (int k = 0; k < 2; ++k) {
    move(a.parts.more[k]);
    move(a.parts.more_ml[k]);
  }
  launch_shared_units<SRC, FP8, D>(c, p, h, a, st);
  attn_shared_join_kernel<SRC, D><<<(unsigned)c.rows * (unsigned)p.q_heads, 256, 0, st>>>(p, a.parts);
  return hipGetLastError();
}
template <int SRC, bool FP8>
static hipError_t launch_shared_src(const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, hipStream_t st) {
  if (c.dim == 64) return launch_shared_dim<SRC, FP8, 64>(c, p, h, st);
  if (c.dim == 128) return launch_shared_dim<SRC, FP8, 128>(c, p, h, st);
  return launch_shared_dim<SRC, FP8, 256>(c, p, h, st);
}

hipError_t launch_attn_shared(int src, const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, hipStream_t st) {
  if (c.seqs == 0 || c.rows == 0) return hipSuccess;
  if (!attn_shared_runs(c.heads, c.dim, p.q_heads, p.max_q)) return launch_attn(src, c, p, st);
  if (src == SRC_BF16) return c.fp8 ? launch_shared_src<SRC_BF16, true>(c, p, h, st) : launch_shared_src<SRC_BF16, false>(c, p, h, st);
  return c.fp8 ? launch_shared_src<SRC_F16, true>(c, p, h, st) : launch_shared_src<SRC_F16, false>(c, p, h, st);
}

}  // namespace dsl
