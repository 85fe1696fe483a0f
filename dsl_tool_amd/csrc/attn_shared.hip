// Attention where groups of sequences share a prefix, over the paged 8-bit
// cache; attn_core.h has the mathematics and the row order.
//
// A group's sequences hold the same pages for its first E tokens (whole pages).
// Their query rows stand together, so the prefix is the context of one unit with
// all of the group's rows, read once for 16 RB of them instead of once per
// sequence; what lies behind it is each sequence's own.  Both kinds of units
// stand in one line of rounds of 256 tokens, prefixes first, and workgroups take
// equal runs of it, as in attn.hip.  Every row has parts of both; a second
// kernel joins them in their order.  A row sees of the prefix what its length and
// its position allow, so rows of sequences that are shorter than it, or empty, are
// right too.
#include "attn_rows.h"
#include "launch.h"

namespace dsl {

constexpr int kMaxRuns = 512;

// The workspace.  The beginning of a unit is kept by its rows, the first of two
// for each query row and head's prefix and own tokens; what a run holds of a unit
// that began before it (one at most) by the run.
template <int D, int ROWS>
struct SharedParts {
  float *first, *more;           // [row][query head][2][D], [run][ROWS][D]
  float2 *first_ml, *more_ml;    // their maxima and sums
  int2 *where;                   // [row][query head][2]: (run of the beginning, or -1: no part; last run * 64 + row of its block)
  DSL_DEV SharedParts(float *ws, int64_t n, int runs)
      : first(ws), more(first + 2 * n * D), first_ml(reinterpret_cast<float2 *>(more + (int64_t)runs * ROWS * D)),
        more_ml(first_ml + 2 * n), where(reinterpret_cast<int2 *>(more_ml + (int64_t)runs * ROWS)) {}
};

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
  } else {
    const SeqView v = seq_view(c, u - h.n);
    s.rows0 = v.row0;
    s.n = v.n;
    s.off = prefix_behind(c, h, u - h.n);
    s.len = v.len;
  }
  return s;
}

// The line of all units' rounds: by unit, cache head, row block.
template <int ROWS>
struct SharedLine {
  const KvCacheArgs &c;
  const SharedArgs &h;
  const int group, chunk, lane;
  int at, rounds, blocks;        // of this lane's unit
  int before, total, upto;       // the line's length before these 64; theirs; theirs up to and with this lane's
  DSL_DEV SharedLine(const KvCacheArgs &c, const SharedArgs &h, int group, int chunk)
      : c(c), h(h), group(group), chunk(chunk), lane(threadIdx.x & 63), at(-64), before(0), total(0), upto(0) {}
  DSL_DEV void advance() {
    before += total;
    at += 64;
    rounds = blocks = 0;
    const int u = at + lane;
    if (u < c.seqs + h.n) {
      const SharedUnit s = shared_unit(c, h, u);
      const int room = c.width * c.page, len = s.len < room ? s.len : room;
      const int tiles = len > s.off ? (len - s.off + kTile - 1) / kTile : 0;
      rounds = (tiles + chunk - 1) / chunk;
      if (u >= h.n && rounds == 0) rounds = 1;   // of no token: one, for its parts
      blocks = rounds ? (int)(((int64_t)s.n * group + ROWS - 1) / ROWS) : 0;
    }
    upto = lanes_sum(rounds * c.heads * blocks);
    total = __builtin_amdgcn_readlane(upto, 63);
  }
  DSL_DEV int length() {                         // of the whole line; back to its beginning
    while (at + 64 < c.seqs + h.n) advance();
    const int n = before + total;
    if (at > 0) {
      at = -64;
      before = total = 0;
      advance();
    }
    return n;
  }
  // The unit of position x, not before an earlier one; its rounds and row
  // blocks, and x in it.  (-1: none, of groups or starts that do not ascend.)
  DSL_DEV int find(int x, int &ur, int &ub, int &off) {
    while (x >= before + total && at + 64 < c.seqs + h.n) advance();
    const uint64_t past = __ballot(before + upto > x);
    if (!past) return -1;
    const int k = __builtin_ctzll(past);
    ur = __builtin_amdgcn_readlane(rounds, k);
    ub = __builtin_amdgcn_readlane(blocks, k);
    off = x - before - __builtin_amdgcn_readlane(upto, k) + ur * c.heads * ub;
    return at + k;
  }
};

template <int SRC, bool FP8, int D, int RB>
__global__ __launch_bounds__(256, rows_wgs(D, RB)) void attn_shared_kernel(const KvCacheArgs c, const AttnArgs p,
                                                                             const SharedArgs h, const int chunk) {
  constexpr bool F16 = SRC == SRC_F16;
  constexpr int DC = D / 64, ROWS = 16 * RB;
  __shared__ __align__(16) RowsJoin<D> sh;
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const SharedParts<D, ROWS> part(p.ws, (int64_t)c.rows * p.q_heads, gridDim.x);
  SharedLine<ROWS> line(c, h, p.group, chunk);
  const int whole = line.length(), per = (whole + (int)gridDim.x - 1) / (int)gridDim.x;
  int x = (int)blockIdx.x * per;
  const int end = whole - per > x ? x + per : whole;

  while (x < end) {
    int rounds, blocks, off;
    const int u = line.find(x, rounds, blocks, off);
    if (u < 0) return;
    const bool prefix = u < h.n;
    const int unit = off / rounds, r0 = off % rounds, head = unit / blocks, rb = unit % blocks;
    const int left = rounds - r0, count = left < end - x ? left : end - x;
    x += count;
    const SharedUnit s = shared_unit(c, h, u);
    const int rows = s.n * p.group, room = c.width * c.page, seen = s.len < room ? s.len : room;
    // whose table row, from which page on; tokens of it
    int from = u - h.n;
    if (prefix) {
      // the first sequence that is as long as the prefix, else the longest
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
        int most = n;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) most = most > __shfl_xor(most, o) ? most : __shfl_xor(most, o);
        if (most > best) {
          best = most;
          from = b + __builtin_ctzll(__ballot(n == most));
        }
      }
      from = __builtin_amdgcn_readfirstlane(from);
    }
    const Context ctx{c.table + (int64_t)from * c.table_ld + s.off / c.page, c.width - s.off / c.page, s.len - s.off};
    RowsWalk<F16, FP8, D, RB> w;
    int lo = 0x7fffffff, high = 0;               // tokens that every row sees, that some row sees
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      const int r = rb * ROWS + k * 16 + r16, rr = r < rows ? r : rows - 1;
      const int i = rr / p.group, hq = head * p.group + rr % p.group, row = s.rows0 + i;
      const uint16_t *qp = static_cast<const uint16_t *>(p.q) + (int64_t)row * p.q_row + (int64_t)hq * p.q_head;
#pragma unroll
      for (int y = 0; y < DC; ++y)
#pragma unroll
        for (int z = 0; z < 2; ++z)
          w.qf[k][2 * y + z] = *reinterpret_cast<const v4i *>(qp + 64 * y + 16 * g + 8 * z);
      // tokens of its own sequence that the row sees
      int b = u - h.n;
      if (prefix) b = c.starts ? last_upto(c.seqs, row, [&](int j) { return first_row(c, j); }) : row;
      const SeqView v = seq_view(c, b);
      int n = p.causal ? v.first + (row - v.row0) + 1 : v.len;
      n = (n < seen ? n : seen) - s.off;
      w.limit[k] = n > 0 ? n : 0;
      lo = lo < w.limit[k] ? lo : w.limit[k];
      high = high > w.limit[k] ? high : w.limit[k];
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      const int a = __shfl_xor(lo, o), z = __shfl_xor(high, o);
      lo = lo < a ? lo : a;
      high = high > z ? high : z;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int nsee = (__builtin_amdgcn_readfirstlane(high) + kTile - 1) / kTile;
    const int t0 = r0 * chunk, t1 = nsee - t0 > count * chunk ? t0 + count * chunk : nsee;
    w.walk(c, ctx, p.scale, true, head, t0, t1, lo);
    const int last = (int)blockIdx.x + (left - count + per - 1) / per;
    join_rows<D, RB>(sh, w, rows - rb * ROWS, [&](int k, int row, int col, const v4f &v, float mr, float lr) {
      const int r = rb * ROWS + k * 16 + row, i = r / p.group, hq = head * p.group + r % p.group;
      const float2 ml = make_float2(lr == lr ? mr : lr, lr);   // a NaN sum without a maximum stays NaN in the join
      if (r0 == 0) {
        const int64_t rh = (int64_t)(s.rows0 + i) * p.q_heads + hq, at = 2 * rh + (prefix ? 0 : 1);
        *reinterpret_cast<v4f *>(part.first + at * D + col) = v;
        if (col != 0) return;
        part.first_ml[at] = ml;
        part.where[at] = make_int2((int)blockIdx.x, last * 64 + k * 16 + row);
        if (!prefix && s.off == 0) part.where[2 * rh] = make_int2(-1, 0);
      } else {
        const int64_t at = (int64_t)blockIdx.x * ROWS + k * 16 + row;
        *reinterpret_cast<v4f *>(part.more + at * D + col) = v;
        if (col == 0) part.more_ml[at] = ml;
      }
    });
  }
}

// Joins the parts of one query row and head in a workgroup, as attn.hip's does: a
// part per thread for the maximum and the sum, then four columns per thread, the
// parts dealt to 1024 / D threads of each.
template <int SRC, int D, int ROWS>
__global__ __launch_bounds__(256) void attn_shared_join_kernel(const AttnArgs p, const int64_t n, const int runs) {
  constexpr int CG = D / 4, SL = 256 / CG;
  __shared__ float s_f[2 * kMaxRuns], s_red[8];
  __shared__ v4f s_v[SL][CG];
  const int64_t at = blockIdx.x;
  const int tid = threadIdx.x;
  const SharedParts<D, ROWS> part(p.ws, n, runs);
  // (A row of no sequence has what the workspace held: in bounds, and its result
  // is not specified.)
  auto span = [&](const int2 &w) {
    if (w.x < 0 || w.x >= runs) return 0;
    const int many = (w.y >> 6) - w.x + 1, most = runs - w.x;
    return many < 0 ? 0 : many < most ? many : most;
  };
  const int2 wp = part.where[2 * at], wo = part.where[2 * at + 1];
  const int np = span(wp), parts = np + span(wo);
  // part s: a row's beginning, or the run that holds more of it
  auto beginning = [&](int s) { return s == 0 && np > 0 ? 2 * at : s == np ? 2 * at + 1 : (int64_t)-1; };
  auto run_row = [&](int s) {
    const int2 w = s < np ? wp : wo;
    return (int64_t)(w.x + (s < np ? s : s - np)) * ROWS + (w.y & (ROWS - 1));
  };
  auto max_sum = [&](int s) {
    const int64_t b = beginning(s);
    return b >= 0 ? part.first_ml[b] : part.more_ml[run_row(s)];
  };
  float top = -INFINITY, l = 0.f;
  for (int s = tid; s < parts; s += 256) {
    const float m = max_sum(s).x;
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
    l += max_sum(s).y * f;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = l;
  __syncthreads();
  const int cg = tid % CG, sl = tid / CG;
  v4f v = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = sl; s < parts; s += SL) {
    const int64_t b = beginning(s);
    v += *reinterpret_cast<const v4f *>((b >= 0 ? part.first + b * D : part.more + run_row(s) * D) + cg * 4) * s_f[s];
  }
  s_v[sl][cg] = v;
  __syncthreads();
  if (tid >= CG) return;
#pragma unroll
  for (int k = 1; k < SL; ++k) v += s_v[k][cg];
  l = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  const float inv = l > 0.f ? 1.0f / l : 0.f;    // a row that sees nothing is 0
  uint16_t *op = static_cast<uint16_t *>(p.o) + (at / p.q_heads) * p.o_row + (at % p.q_heads) * p.o_head + cg * 4;
  *reinterpret_cast<uint2 *>(op) = make_uint2(narrow2<SRC>(v[0] * inv, v[1] * inv), narrow2<SRC>(v[2] * inv, v[3] * inv));
}

struct SharedPlan {
  int rb, runs, chunk;
};
static SharedPlan shared_plan(const KvCacheArgs &c, int groups, int q_heads, int max_q, int max_group) {
  SharedPlan a{};
  const int64_t group = q_heads / c.heads, rows = (int64_t)max_q * max_group * group;    // of a prefix
  a.rb = rows <= 16 || c.dim > 128 ? 1 : 2;
  a.runs = rows_wgs(c.dim, a.rb) * device_cu_count();
  if (a.runs > kMaxRuns) a.runs = kMaxRuns;
  // rounds of a tile per wave, longer ones where the line's length would pass an int
  const int64_t tiles = ((int64_t)c.width * c.page + kTile - 1) / kTile;
  const int64_t units = c.heads * (2 * ((int64_t)c.rows * group / (16 * a.rb)) + c.seqs + groups);   // at most
  a.chunk = 4;
  while ((tiles + a.chunk - 1) / a.chunk * units > 1 << 30 && a.chunk < tiles) a.chunk *= 2;
  return a;
}

size_t attn_shared_workspace_bytes(const KvCacheArgs &c, int groups, int q_heads, int max_q, int max_group) {
  const SharedPlan a = shared_plan(c, groups, q_heads, max_q, max_group);
  const size_t n = (size_t)c.rows * q_heads, row = (c.dim + 2) * sizeof(float);
  return 2 * n * (row + sizeof(int2)) + (size_t)a.runs * 16 * a.rb * row;
}

template <int SRC, int D, int RB>
static void launch_shared_rows(const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, const SharedPlan &a, hipStream_t st) {
  if (c.fp8) attn_shared_kernel<SRC, true, D, RB><<<(unsigned)a.runs, 256, 0, st>>>(c, p, h, a.chunk);
  else attn_shared_kernel<SRC, false, D, RB><<<(unsigned)a.runs, 256, 0, st>>>(c, p, h, a.chunk);
  attn_shared_join_kernel<SRC, D, 16 * RB><<<(unsigned)c.rows * (unsigned)p.q_heads, 256, 0, st>>>(p, (int64_t)c.rows * p.q_heads, a.runs);
}
template <int SRC, int D>
static hipError_t launch_shared_dim(const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, hipStream_t st) {
  const SharedPlan a = shared_plan(c, h.n, p.q_heads, p.max_q, h.most);
  if (a.rb == 1) launch_shared_rows<SRC, D, 1>(c, p, h, a, st);
  else if constexpr (D <= 128) launch_shared_rows<SRC, D, 2>(c, p, h, a, st);
  return hipGetLastError();
}
template <int SRC>
static hipError_t launch_shared_src(const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, hipStream_t st) {
  if (c.dim == 64) return launch_shared_dim<SRC, 64>(c, p, h, st);
  if (c.dim == 128) return launch_shared_dim<SRC, 128>(c, p, h, st);
  return launch_shared_dim<SRC, 256>(c, p, h, st);
}

hipError_t launch_attn_shared(int src, const KvCacheArgs &c, const AttnArgs &p, const SharedArgs &h, hipStream_t st) {
  if (c.seqs == 0 || c.rows == 0) return hipSuccess;
  return src == SRC_BF16 ? launch_shared_src<SRC_BF16>(c, p, h, st) : launch_shared_src<SRC_F16>(c, p, h, st);
}

}  // namespace dsl
