// Rotary positions: the pairs (x, y) of a head turned by angles of its token,
//   a_i = pos[axis(i)] f_i,  (x, y) -> m (x cos a_i - y sin a_i, y cos a_i + x sin a_i),
// pair i being dimensions (i, i + half) or (2 i, 2 i + 1); what lies behind them
// stays.
//
// A far position's angle has more digits than fp32: the turns pos * f / 2 pi are
// formed in 64 bits and reduced there, and only their fraction goes on in 32.
// A token's cosines and sines serve all its heads, so a workgroup makes them once
// for its tokens, in shared memory, behind the heads' loads.  Bound by the bytes of
// queries and keys, each read and written once (20001 rows of 40 heads of 128: 86 us,
// 4.8 TB/s); a short call by one launch (32 rows: 5.3).
#include "common.h"
#include "generate_args.h"
#include "kv_core.h"
#include "launch.h"

namespace dsl {

constexpr int kTurnBytes = 16384;                // of cosines and sines in a workgroup

template <bool POS64>
DSL_DEV float2 turn_of(const RotaryArgs &p, int row, int i) {
  const int axis = p.axis_of ? p.axis_of[i] : 0;
  double pos = 0.0;                              // of an axis that is none
  if (axis >= 0 && axis < p.axes) {
    const int64_t at = axis * p.pos_ld + row;
    if constexpr (POS64) pos = (double)static_cast<const int64_t *>(p.positions)[at];
    else pos = (double)static_cast<const int32_t *>(p.positions)[at];
  }
  const double turns = pos * (p.freqs[i] * 0.15915494309189533577);
  const float f = (float)(turns - __builtin_rint(turns));
  float s, c;
  sincospif(2.0f * f, &s, &c);
  return make_float2(c * p.magnitude, s * p.magnitude);
}

// V: elements of an access (8: 16 bytes, or 1).  An item is V pairs of a head
// (halves), V / 2 of them (adjacent; 1 at least), or V elements behind them.
template <int V>
DSL_DEV void ld_elems(uint16_t *e, const uint16_t *x) {
  if constexpr (V == 8) {
    const uint4 v = *reinterpret_cast<const uint4 *>(x);
    __builtin_memcpy(e, &v, 16);
  } else {
    e[0] = x[0];
  }
}
template <int V>
DSL_DEV void st_elems(uint16_t *y, const uint16_t *e) {
  if constexpr (V == 8) {
    uint4 v;
    __builtin_memcpy(&v, e, 16);
    *reinterpret_cast<uint4 *>(y) = v;
  } else {
    y[0] = e[0];
  }
}
template <int SRC>
DSL_DEV uint16_t narrow(float v) {
  return (uint16_t)narrow2<SRC>(v, 0.f);
}

// Grid: x groups of `tokens` rows, y slices of a row's items.
template <int SRC, int V, bool ADJ, bool POS64>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs p, const int tokens, const int turned,
                                                     const int rest) {
  __shared__ float2 s_turn[kTurnBytes / 8];
  const int row0 = (int)(blockIdx.x * (int64_t)tokens);
  const int many = p.rows - row0 < tokens ? p.rows - row0 : tokens;
  for (int i = threadIdx.x; i < many * p.half; i += 256) s_turn[i] = turn_of<POS64>(p, row0 + i / p.half, i % p.half);
  __syncthreads();
  const int heads = p.q.heads + p.k.heads, items = heads * (turned + rest);
  const int per = (items + (int)gridDim.y - 1) / (int)gridDim.y, first = (int)blockIdx.y * per;
  const int mine = items - first < per ? items - first : per;
  for (int64_t i = threadIdx.x; i < (int64_t)many * mine; i += 256) {
    const int t = (int)(i / mine), item = first + (int)(i % mine), h = item / (turned + rest), c = item % (turned + rest);
    const bool of_k = h >= p.q.heads;
    const RotaryHeads &r = of_k ? p.k : p.q;
    const int head = of_k ? h - p.q.heads : h;
    const uint16_t *x = static_cast<const uint16_t *>(r.x) + (int64_t)(row0 + t) * r.row + (int64_t)head * r.head;
    uint16_t *y = static_cast<uint16_t *>(r.y) + (int64_t)(row0 + t) * r.yrow + (int64_t)head * r.yhead;
    alignas(16) uint16_t a[V], b[V];
    if (c >= turned) {
      const int d = 2 * p.half + (c - turned) * V;
      ld_elems<V>(a, x + d);
      st_elems<V>(y + d, a);
    } else if constexpr (!ADJ) {
      const int d = c * V;
      ld_elems<V>(a, x + d);
      ld_elems<V>(b, x + d + p.half);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 cs = s_turn[t * p.half + d + e];
        const float u = widen<SRC>(a[e]), w = widen<SRC>(b[e]);
        a[e] = narrow<SRC>(u * cs.x - w * cs.y);
        b[e] = narrow<SRC>(w * cs.x + u * cs.y);
      }
      st_elems<V>(y + d, a);
      st_elems<V>(y + d + p.half, b);
    } else if constexpr (V == 8) {
      const int d = c * V;
      ld_elems<V>(a, x + d);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 cs = s_turn[t * p.half + (d + e) / 2];
        const float u = widen<SRC>(a[e]), w = widen<SRC>(a[e + 1]);
        a[e] = narrow<SRC>(u * cs.x - w * cs.y);
        a[e + 1] = narrow<SRC>(w * cs.x + u * cs.y);
      }
      st_elems<V>(y + d, a);
    } else {
      const int d = 2 * c;
      const float2 cs = s_turn[t * p.half + c];
      const float u = widen<SRC>(x[d]), w = widen<SRC>(x[d + 1]);
      y[d] = narrow<SRC>(u * cs.x - w * cs.y);
      y[d + 1] = narrow<SRC>(w * cs.x + u * cs.y);
    }
  }
}

template <int SRC, int V, bool ADJ>
static hipError_t launch_rotary_form(const RotaryArgs &p, hipStream_t st) {
  const bool in_place = p.q.y == p.q.x && (p.k.heads == 0 || p.k.y == p.k.x);
  const int turned = ADJ && V == 8 ? p.half / 4 : p.half / V;
  const int rest = in_place ? 0 : (p.dim - 2 * p.half) / V;
  const int64_t items = (int64_t)(p.q.heads + p.k.heads) * (turned + rest);
  if (items == 0) return hipSuccess;
  const int cus = device_cu_count();
  int tokens = kTurnBytes / 8 / (p.half > 0 ? p.half : 1);
  tokens = tokens > 8 ? 8 : tokens;
  while (tokens > 1 && (int64_t)(p.rows + tokens - 1) / tokens < 4 * cus) tokens /= 2;
  const int64_t groups = ((int64_t)p.rows + tokens - 1) / tokens;
  int64_t slices = 1;
  while (groups * slices < cus && items * tokens / (2 * slices) >= 64) slices *= 2;
  const dim3 grid((unsigned)groups, (unsigned)slices);
  if (p.pos64) rotary_kernel<SRC, V, ADJ, true><<<grid, 256, 0, st>>>(p, tokens, turned, rest);
  else rotary_kernel<SRC, V, ADJ, false><<<grid, 256, 0, st>>>(p, tokens, turned, rest);
  return hipGetLastError();
}

// 16-byte accesses: rows, heads and the parts of a head begin on one.
static bool rotary_vectors(const RotaryArgs &p) {
  auto fits = [](const RotaryHeads &r) {
    return r.heads == 0 || (r.row % 8 == 0 && r.head % 8 == 0 && r.yrow % 8 == 0 && r.yhead % 8 == 0 &&
                            reinterpret_cast<uintptr_t>(r.x) % 16 == 0 && reinterpret_cast<uintptr_t>(r.y) % 16 == 0);
  };
  return p.dim % 8 == 0 && (p.adjacent ? p.half % 4 == 0 : p.half % 8 == 0) && fits(p.q) && fits(p.k);
}

template <int SRC>
static hipError_t launch_rotary_src(const RotaryArgs &p, hipStream_t st) {
  if (rotary_vectors(p)) {
    return p.adjacent ? launch_rotary_form<SRC, 8, true>(p, st) : launch_rotary_form<SRC, 8, false>(p, st);
  }
  return p.adjacent ? launch_rotary_form<SRC, 1, true>(p, st) : launch_rotary_form<SRC, 1, false>(p, st);
}

hipError_t launch_rotary(int src, const RotaryArgs &p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  return src == SRC_BF16 ? launch_rotary_src<SRC_BF16>(p, st) : launch_rotary_src<SRC_F16>(p, st);
}

}  // namespace dsl
