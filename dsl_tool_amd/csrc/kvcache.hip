// Writing tokens into the paged 8-bit cache, and reading them back.
//
// A page has one scale per head for its keys and one for its values:
//   s = max(scale kept, max|x| / top, 1e-12)   over the page's new tokens,
// the kept scale counting only where older tokens stay in the page.  Where s
// grew, their codes move to it, c' = round(c * s_kept / s) (int8; e4m3
// likewise): one more rounding of at most half a step, and only on growth.
// Every quotient is the IEEE one, so the codes do not depend on how the work
// is split.
//
// One workgroup owns a page and head, so no scale is shared and nothing is
// atomic.  A thread holds four tokens of eight dimensions: a wave's loads then
// cover whole rows, and a value row's four codes are one word, which crosses
// shared memory to leave in 16-byte stores.
#include "kv_core.h"
#include "launch.h"

namespace dsl {

// Word of a value tile in shared memory: row d, 4 tokens from 4 * t4.  Rows of
// `words` words, four more after each eighth row, so that the 64 lanes of a
// wave (16 chunks of dimensions x 4 groups of tokens) write to 64 banks.
DSL_DEV int tile_word(int d, int t4, int words) { return d * words + (d >> 3) * 4 + t4; }

// Division by a scale s.  With r = RN(1 / s), q = RN(x r) is within one ulp of
// x / s, and one step q - (q s - x) r by fused products is then the IEEE
// quotient (Markstein, IBM J. Res. Dev. 34, 1990): three operations for the
// ten of a division.  Where x is so small that its remainder is subnormal the
// quotient may differ, far below half a code.  Scales of which 1 / s would be
// subnormal are brought down with x; an infinite one leaves zeros, and no
// number of an infinity.
struct Divisor {
  float s, r, down;
};
DSL_DEV Divisor divisor_of(float s) {
  Divisor v;
  v.down = s < 0x1p125f ? 1.0f : 0x1p-24f;
  v.s = s * v.down;
  v.r = __fdiv_rn(1.0f, v.s);
  if (v.r == 0.f) v.s = 0.f;
  return v;
}
template <bool FP8>
DSL_DEV uint32_t codes_by(float a, float b, float c, float d, const Divisor &v) {
  auto quotient = [&](float x) __attribute__((always_inline)) {
    x *= v.down;
    const float q = x * v.r;
    return __builtin_fmaf(-__builtin_fmaf(q, v.s, -x), v.r, q);  // -0 stays -0
  };
  return codes_pack<FP8>(quotient(a), quotient(b), quotient(c), quotient(d));
}

// Four codes of scale `kept` moved to another.
template <bool FP8>
DSL_DEV uint32_t codes_moved(uint32_t w, float kept, const Divisor &v) {
  float f[4];
  code_values<FP8>(w, f);
  return codes_by<FP8>(f[0] * kept, f[1] * kept, f[2] * kept, f[3] * kept, v);
}

// Grid: x items (pages a sequence's new tokens touch), y head * 2 + (1:
// values).  HELD: a page's tokens, UN units per thread, stay in registers
// between their maximum and their codes; longer pages go by 64 tokens and read
// them again, from the caches.  A call of few tokens is one chain of loads and
// the fetch of the code itself, so what every call runs is short: one set of
// quotients for keys and values, whose codes are turned by byte permutes (64
// sequences' tokens, 8 heads of 128: 5.6 us; 18 with a copy of the quotients per
// use).  A long call is bound by the bytes: prompts of 8 heads, 34 MB, in
// 9.3 us, where a workgroup per value and key tile that read its tokens twice
// and stored values by words took 14.3.
template <int SRC, bool FP8, int NT, int UN, bool HELD>
__global__ __launch_bounds__(NT) void kv_write_kernel(const KvCacheArgs c, const KvWriteArgs p) {
  __shared__ __attribute__((aligned(16))) uint32_t tile[NT * UN * 9];
  __shared__ float sh[NT / 64 + 1];
  const int tid = threadIdx.x, head = blockIdx.y >> 1;
  const bool vals = blockIdx.y & 1;
  const int P = c.page, plog = __builtin_ctz(P), dlog = __builtin_ctz(c.dim) - 3, D = c.dim;
  int b, item;
  const SeqView s = item_seq(c, blockIdx.x, [&](int row, int q) { return (row >> plog) + 2 * q; }, b, item);
  if (b < 0 || s.n == 0 || s.len == 0) return;
  const int start = s.first > 0 ? s.first : 0;
  const int pg = (start >> plog) + item, base = pg << plog;
  if (item < 0 || base >= s.len || base < 0) return;
  const int lo = start > base ? start - base : 0;
  const int hi = s.len - base < P ? s.len - base : P;        // tokens [lo, hi) of the page are new
  if (pg >= c.width) return;
  const int number = c.table[(int64_t)b * c.table_ld + pg];  // not waited for yet: the tokens come with it
  const uint16_t *x = static_cast<const uint16_t *>(vals ? p.v : p.k) + head * (vals ? p.v_head : p.k_head);
  const int64_t ld = vals ? p.v_row : p.k_row;
  const uint16_t *xr = x + (int64_t)(s.row0 + (base - s.first)) * ld;   // row of the page's token 0
  const int TT = P < 64 ? P : 64, words = TT >> 2;
  uint4 xa[UN][4];
  // rows past the new ones repeat them: no maximum changes, and no code is stored
  auto fetch = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int un = tid + NT * u, t = t0 + ((un >> dlog) << 2), d = (un & ((1 << dlog) - 1)) << 3;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = t + j < lo ? lo : t + j >= hi ? hi - 1 : t + j;
        xa[u][j] = *reinterpret_cast<const uint4 *>(xr + (int64_t)row * ld + d);
      }
    }
  };
  float m = 0.f;
  auto maximum = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[8];
        widen8s<SRC>(xa[u][j], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, __builtin_fabsf(f[e]));
      }
  };
  if (HELD) fetch(0);
  if (number < 0 || number >= c.pages) return;
  const int64_t at = (int64_t)number * c.heads + head;
  float *sp = (vals ? c.v_scale : c.k_scale) + at;
  uint8_t *codes = (vals ? c.v : c.k) + at * P * D;
  const int tb = lo & ~63;                                   // the first tile with new tokens
  if (tid == 0) sh[NT / 64] = lo > 0 ? *sp : 0.f;            // read before any thread stores
  if (HELD) {
    maximum();
  } else {
    for (int t0 = tb; t0 < hi; t0 += 64) {
      fetch(t0);
      maximum();
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) sh[tid >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) m = fmaxf(m, sh[i]);
  const float kept = sh[NT / 64];
  const float sc = fmaxf(kept, kv_scale_of<FP8>(m));
  const Divisor by = divisor_of(sc);
  if (tid == 0) *sp = sc;
  if (lo > 0 && sc > kept) {
    // the older tokens' codes: a key's words are one token's, a value's four tokens'
    const int end = vals ? D * P >> 2 : lo * D >> 2;
#pragma unroll 1
    for (int i = tid; i < end; i += NT) {
      const int ahead = vals ? lo - ((i & ((P >> 2) - 1)) << 2) : 4;   // older tokens of this word, or more
      if (ahead <= 0) continue;
      uint32_t *w = reinterpret_cast<uint32_t *>(codes) + i;
      const uint32_t older = ahead >= 4 ? ~0u : (1u << (8 * ahead)) - 1, old = *w;
      *w = (codes_moved<FP8>(old, kept, by) & older) | (old & ~older);
    }
    __syncthreads();                                         // before bytes of the same words
  }
#pragma unroll 1
  for (int t0 = tb; t0 < hi; t0 += TT) {
    if (!HELD) fetch(t0);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int un = tid + NT * u, t = t0 + ((un >> dlog) << 2), d = (un & ((1 << dlog) - 1)) << 3;
      if (t >= hi || t + 4 <= lo || t >= t0 + TT) continue;
      uint32_t q[4][2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[8];
        widen8s<SRC>(xa[u][j], f);
        q[j][0] = codes_by<FP8>(f[0], f[1], f[2], f[3], by);
        q[j][1] = codes_by<FP8>(f[4], f[5], f[6], f[7], by);
      }
      if (!vals) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (t + j >= lo && t + j < hi)
            *reinterpret_cast<uint2 *>(codes + ((t + j) << (dlog + 3)) + d) = make_uint2(q[j][0], q[j][1]);
        continue;
      }
      uint32_t w[8];                             // four tokens of each dimension
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t a = __builtin_amdgcn_perm(q[1][h], q[0][h], 0x05010400u);
        const uint32_t c2 = __builtin_amdgcn_perm(q[3][h], q[2][h], 0x05010400u);
        const uint32_t e = __builtin_amdgcn_perm(q[1][h], q[0][h], 0x07030602u);
        const uint32_t g = __builtin_amdgcn_perm(q[3][h], q[2][h], 0x07030602u);
        w[4 * h] = __builtin_amdgcn_perm(c2, a, 0x05040100u);
        w[4 * h + 1] = __builtin_amdgcn_perm(c2, a, 0x07060302u);
        w[4 * h + 2] = __builtin_amdgcn_perm(g, e, 0x05040100u);
        w[4 * h + 3] = __builtin_amdgcn_perm(g, e, 0x07060302u);
      }
      const int g0 = t & ~15;                    // 16 new tokens leave as one store, through the tile
      if (g0 >= lo && g0 + 16 <= hi) {
#pragma unroll
        for (int e = 0; e < 8; ++e) tile[tile_word(d + e, (t - t0) >> 2, words)] = w[e];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (t + j < lo || t + j >= hi) continue;
#pragma unroll
          for (int e = 0; e < 8; ++e) codes[(d + e) * P + t + j] = (uint8_t)(w[e] >> (8 * j));
        }
      }
    }
    if (!vals) continue;
    __syncthreads();
    const int clog = __builtin_ctz(TT) - 4;
#pragma unroll 1
    for (int i = tid; i < D << clog; i += NT) {
      const int d = i >> clog, t = (i & ((1 << clog) - 1)) << 4, g = t0 + t;
      if (g >= lo && g + 16 <= hi)
        *reinterpret_cast<uint4 *>(codes + d * P + g) = *reinterpret_cast<const uint4 *>(tile + tile_word(d, t >> 2, words));
    }
    if (!HELD) __syncthreads();                              // the tile's readers
  }
}

template <int SRC, bool FP8>
static void write_by_page(const dim3 &grid, const KvCacheArgs &c, const KvWriteArgs &p, hipStream_t st) {
  // threads by the units of four tokens and eight dimensions in a page, or in 64 tokens of it
  const int units = (c.page < 64 ? c.page : 64) / 4 * (c.dim / 8);
  if (units <= 64) kv_write_kernel<SRC, FP8, 64, 1, true><<<grid, 64, 0, st>>>(c, p);
  else if (units <= 128 && c.page <= 64) kv_write_kernel<SRC, FP8, 128, 1, true><<<grid, 128, 0, st>>>(c, p);
  else if (units <= 256 && c.page <= 64) kv_write_kernel<SRC, FP8, 256, 1, true><<<grid, 256, 0, st>>>(c, p);
  else if (c.page <= 64) kv_write_kernel<SRC, FP8, 256, 2, true><<<grid, 256, 0, st>>>(c, p);
  else if (units <= 256) kv_write_kernel<SRC, FP8, 256, 1, false><<<grid, 256, 0, st>>>(c, p);
  else kv_write_kernel<SRC, FP8, 256, 2, false><<<grid, 256, 0, st>>>(c, p);
}

hipError_t launch_kv_write(int src, const KvCacheArgs &c, const KvWriteArgs &p, hipStream_t st) {
  if (c.seqs == 0 || c.rows == 0) return hipSuccess;
  const dim3 grid((unsigned)(c.starts ? c.rows / c.page + 2 * c.seqs : c.seqs), (unsigned)c.heads * 2);
  if (src == SRC_BF16) {
    if (c.fp8) write_by_page<SRC_BF16, true>(grid, c, p, st);
    else write_by_page<SRC_BF16, false>(grid, c, p, st);
  } else {
    if (c.fp8) write_by_page<SRC_F16, true>(grid, c, p, st);
    else write_by_page<SRC_F16, false>(grid, c, p, st);
  }
  return hipGetLastError();
}

// Rows [starts[b], starts[b+1]) of the result are the sequence's tokens from
// its first on; rows past its length, or of pages that are none, are zeros.
// Grid: x items (64 tokens of a sequence, of one page or several), y head.
// Bound by the bytes: 8 sequences of up to 8192 tokens, pages of 16, 275 MB in
// 58 us; 92 with a workgroup per page and of keys or values, whose
// threads read a word of each value row.
template <int SRC, bool FP8, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvCacheArgs c, const KvReadArgs p) {
  constexpr int DCH = D / 8, UN = D / 128 > 1 ? D / 128 : 1, UNITS = 16 * DCH, CH = D * 4 / 256;
  __shared__ __attribute__((aligned(16))) uint32_t tile[D * 16 + D / 2];
  const int tid = threadIdx.x, head = blockIdx.y;
  int b, item;
  const SeqView s = item_seq(c, blockIdx.x, [](int row, int q) { return (row >> 6) + q; }, b, item);
  const int base = item << 6;
  if (b < 0 || item < 0 || base >= s.n) return;
  const int rows = s.n - base < 64 ? s.n - base : 64, have = s.len - base < rows ? s.len - base : rows;
  const int P = c.page, plog = __builtin_ctz(P), TT = P < 64 ? P : 64, tlog = P < 64 ? plog : 6;
  // a 16-byte chunk of values per turn: those of a page are contiguous, row by row
  uint4 va[CH];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int i = tid + 256 * k, clog = tlog - 4, in = i & ((D << clog) - 1);
    const int d = in >> clog, t = ((i >> (clog + __builtin_ctz(D))) << tlog) + ((in & ((1 << clog) - 1)) << 4);
    const int64_t pid = t < have ? page_of(c, b, (base + t) >> plog) : -1;
    va[k] = make_uint4(0, 0, 0, 0);
    if (pid >= 0)
      va[k] = *reinterpret_cast<const uint4 *>(c.v + ((pid * c.heads + head) * D + d) * P + ((base + t) & (P - 1)));
  }
  uint2 ka[UN][4];
  float ks[UN], vs[UN];
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    const int un = tid + 256 * u, t = (un / DCH) << 2, d = (un % DCH) << 3;
    const int64_t pid = un < UNITS && t < have ? page_of(c, b, (base + t) >> plog) : -1;
    const int64_t at = (pid < 0 ? 0 : pid) * c.heads + head;
    ks[u] = vs[u] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) ka[u][j] = make_uint2(0, 0);
    if (pid >= 0) {
      ks[u] = c.k_scale[at];
      vs[u] = c.v_scale[at];
      const uint8_t *codes = c.k + (at * P + ((base + t) & (P - 1))) * D + d;      // inside the page
#pragma unroll
      for (int j = 0; j < 4; ++j) ka[u][j] = *reinterpret_cast<const uint2 *>(codes + j * D);
    }
  }
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int i = tid + 256 * k, clog = tlog - 4, in = i & ((D << clog) - 1);
    const int d = in >> clog, t = ((i >> (clog + __builtin_ctz(D))) << tlog) + ((in & ((1 << clog) - 1)) << 4);
    *reinterpret_cast<uint4 *>(tile + tile_word(d, t >> 2, 16)) = va[k];
  }
  const int64_t ld = (int64_t)c.heads * D;
  const int64_t out = (int64_t)(s.row0 + base) * ld + (int64_t)head * D;
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    const int un = tid + 256 * u, t = (un / DCH) << 2, d = (un % DCH) << 3;
    if (un >= UNITS) continue;
    uint16_t *o = static_cast<uint16_t *>(p.k) + out + (int64_t)t * ld + d;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (t + j >= rows) break;
      float f[8];
      code_values<FP8>(ka[u][j].x, f);
      code_values<FP8>(ka[u][j].y, f + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = t + j < have ? f[e] * ks[u] : 0.f;
      *reinterpret_cast<uint4 *>(o + (int64_t)j * ld) =
          make_uint4(narrow2<SRC>(f[0], f[1]), narrow2<SRC>(f[2], f[3]), narrow2<SRC>(f[4], f[5]), narrow2<SRC>(f[6], f[7]));
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    const int un = tid + 256 * u, t = (un / DCH) << 2, d = (un % DCH) << 3;
    if (un >= UNITS) continue;
    float f[8][4];
#pragma unroll
    for (int e = 0; e < 8; ++e) code_values<FP8>(tile[tile_word(d + e, t >> 2, 16)], f[e]);
    uint16_t *o = static_cast<uint16_t *>(p.v) + out + (int64_t)t * ld + d;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (t + j >= rows) break;
      float g[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = t + j < have ? f[e][j] * vs[u] : 0.f;
      *reinterpret_cast<uint4 *>(o + (int64_t)j * ld) =
          make_uint4(narrow2<SRC>(g[0], g[1]), narrow2<SRC>(g[2], g[3]), narrow2<SRC>(g[4], g[5]), narrow2<SRC>(g[6], g[7]));
    }
  }
}

template <int SRC, bool FP8>
static void read_by_dim(const KvCacheArgs &c, const KvReadArgs &p, hipStream_t st) {
  const dim3 grid((unsigned)(c.starts ? c.rows / 64 + c.seqs : c.seqs), (unsigned)c.heads);
  if (c.dim == 64) kv_read_kernel<SRC, FP8, 64><<<grid, 256, 0, st>>>(c, p);
  else if (c.dim == 128) kv_read_kernel<SRC, FP8, 128><<<grid, 256, 0, st>>>(c, p);
  else kv_read_kernel<SRC, FP8, 256><<<grid, 256, 0, st>>>(c, p);
}

hipError_t launch_kv_read(int src, const KvCacheArgs &c, const KvReadArgs &p, hipStream_t st) {
  if (c.seqs == 0 || c.rows == 0) return hipSuccess;
  if (src == SRC_BF16) {
    if (c.fp8) read_by_dim<SRC_BF16, true>(c, p, st);
    else read_by_dim<SRC_BF16, false>(c, p, st);
  } else {
    if (c.fp8) read_by_dim<SRC_F16, true>(c, p, st);
    else read_by_dim<SRC_F16, false>(c, p, st);
  }
  return hipGetLastError();
}

}  // namespace dsl
