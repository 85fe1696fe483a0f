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
// atomic.  The new tokens are read twice, the second time from the caches.
#include "kv_core.h"
#include "launch.h"

namespace dsl {

DSL_DEV float block_max256(float v, float *sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();                               // the array's last readers
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}

// blockIdx: x pages from the first touched one on, y head * 2 + (1: values),
// z sequence.
template <int SRC, bool FP8>
__global__ __launch_bounds__(256) void kv_write_kernel(const KvCacheArgs c, const KvWriteArgs p) {
  __shared__ float sh[4];
  const int b = blockIdx.z, head = blockIdx.y >> 1, tid = threadIdx.x;
  const bool vals = blockIdx.y & 1;
  const SeqView s = seq_view(c, b);
  if (s.n == 0 || s.len == 0) return;
  const int start = s.first > 0 ? s.first : 0;
  const int D = c.dim, P = c.page;
  const uint16_t *x = static_cast<const uint16_t *>(vals ? p.v : p.k) + head * (vals ? p.v_head : p.k_head);
  const int64_t ld = vals ? p.v_row : p.k_row;
  const int last = (s.len - 1) / P;
  for (int pg = start / P + blockIdx.x; pg <= last; pg += gridDim.x) {
    const int64_t pid = page_of(c, b, pg);
    if (pid < 0) continue;                       // the whole workgroup
    const int base = pg * P, lo = start > base ? start - base : 0;
    const int hi = s.len - base < P ? s.len - base : P;      // tokens [lo, hi) of the page are new
    const uint16_t *xr = x + (int64_t)(s.row0 + (base - s.first)) * ld;   // row of the page's token 0
    const int dch = D / 8, n8 = (hi - lo) * dch;
    float m = 0.f;
    for (int i = tid; i < n8; i += 256) {
      float f[8];
      widen8s<SRC>(*reinterpret_cast<const uint4 *>(xr + (int64_t)(lo + i / dch) * ld + (i % dch) * 8), f);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, __builtin_fabsf(f[e]));
    }
    m = block_max256(m, sh);
    float *sp = (vals ? c.v_scale : c.k_scale) + pid * c.heads + head;
    const float kept = lo > 0 ? *sp : 0.f;
    const float sc = fmaxf(kept, kv_scale_of<FP8>(m));
    __syncthreads();                             // every thread has the old scale
    if (tid == 0) *sp = sc;
    uint8_t *codes = (vals ? c.v : c.k) + (pid * c.heads + head) * (int64_t)P * D;
    const bool grew = lo > 0 && sc > kept;
    if (!vals) {
      if (grew) {
        for (int i = tid; i < lo * D / 4; i += 256) {
          uint32_t *w = reinterpret_cast<uint32_t *>(codes) + i;
          float f[4];
          code_values<FP8>(*w, f);
          *w = codes_of<FP8>(f[0] * kept, f[1] * kept, f[2] * kept, f[3] * kept, sc);
        }
      }
      for (int i = tid; i < n8; i += 256) {
        const int t = lo + i / dch, d = (i % dch) * 8;
        float f[8];
        widen8s<SRC>(*reinterpret_cast<const uint4 *>(xr + (int64_t)t * ld + d), f);
        *reinterpret_cast<uint2 *>(codes + (int64_t)t * D + d) =
            make_uint2(codes_of<FP8>(f[0], f[1], f[2], f[3], sc), codes_of<FP8>(f[4], f[5], f[6], f[7], sc));
      }
    } else {
      // four tokens of eight rows of dim each: a row's four codes are one word
      const int g0 = grew ? 0 : lo / 4, groups = (hi + 3) / 4 - g0;
      for (int i = tid; i < groups * dch; i += 256) {
        const int t = (g0 + i % groups) * 4, d = (i / groups) * 8;
        float f[4][8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool on = t + j >= lo && t + j < hi;
          const uint4 v = on ? *reinterpret_cast<const uint4 *>(xr + (int64_t)(t + j) * ld + d) : make_uint4(0, 0, 0, 0);
          widen8s<SRC>(v, f[j]);
        }
        uint32_t mask = 0, moved = 0;            // bytes of new tokens, of older ones to move
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (t + j >= lo && t + j < hi) mask |= 0xffu << (8 * j);
          if (grew && t + j < lo) moved |= 0xffu << (8 * j);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint32_t *w = reinterpret_cast<uint32_t *>(codes + (int64_t)(d + e) * P + t);
          uint32_t out = codes_of<FP8>(f[0][e], f[1][e], f[2][e], f[3][e], sc);
          if (mask != 0xffffffffu) {
            const uint32_t old = *w;
            uint32_t again = old;
            if (moved) {
              float o[4];
              code_values<FP8>(old, o);
              again = codes_of<FP8>(o[0] * kept, o[1] * kept, o[2] * kept, o[3] * kept, sc);
            }
            out = (out & mask) | (again & moved) | (old & ~(mask | moved));
          }
          *w = out;
        }
      }
    }
  }
}

hipError_t launch_kv_write(int src, const KvCacheArgs &c, const KvWriteArgs &p, hipStream_t st) {
  if (c.seqs == 0 || c.rows == 0) return hipSuccess;
  int64_t span = (int64_t)(p.max_q + c.page - 2) / c.page + 1;
  if (span > c.width) span = c.width;
  if (span < 1) return hipSuccess;
  const dim3 grid((unsigned)span, (unsigned)c.heads * 2, (unsigned)c.seqs);
  if (src == SRC_BF16) {
    if (c.fp8) kv_write_kernel<SRC_BF16, true><<<grid, 256, 0, st>>>(c, p);
    else kv_write_kernel<SRC_BF16, false><<<grid, 256, 0, st>>>(c, p);
  } else {
    if (c.fp8) kv_write_kernel<SRC_F16, true><<<grid, 256, 0, st>>>(c, p);
    else kv_write_kernel<SRC_F16, false><<<grid, 256, 0, st>>>(c, p);
  }
  return hipGetLastError();
}

// Rows [starts[b], starts[b+1]) of the result are the sequence's tokens from
// its first on; rows past its length, or of pages that are none, are zeros.
// blockIdx as above.
template <int SRC, bool FP8>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvCacheArgs c, const KvReadArgs p) {
  const int b = blockIdx.z, head = blockIdx.y >> 1, tid = threadIdx.x;
  const bool vals = blockIdx.y & 1;
  const SeqView s = seq_view(c, b);
  const int D = c.dim, P = c.page;
  const int64_t ld = (int64_t)c.heads * D;
  uint16_t *out = static_cast<uint16_t *>(vals ? p.v : p.k) + (int64_t)s.row0 * ld + (int64_t)head * D;
  for (int pg = blockIdx.x; (int64_t)pg * P < s.n; pg += gridDim.x) {
    const int base = pg * P;
    const int rows = s.n - base < P ? s.n - base : P;
    const int64_t pid = page_of(c, b, pg);
    int have = s.len - base < rows ? s.len - base : rows;
    if (pid < 0 || have < 0) have = 0;
    const int64_t at = pid < 0 ? 0 : pid * c.heads + head;
    const float sc = have > 0 ? (vals ? c.v_scale : c.k_scale)[at] : 0.f;
    const uint8_t *codes = (vals ? c.v : c.k) + at * P * D;
    uint16_t *o = out + (int64_t)base * ld;
    const int dch = D / 8;
    if (!vals) {
      for (int i = tid; i < rows * dch; i += 256) {
        const int t = i / dch, d = (i % dch) * 8;
        const uint2 w = t < have ? *reinterpret_cast<const uint2 *>(codes + (int64_t)t * D + d) : make_uint2(0, 0);
        float f[8];
        code_values<FP8>(w.x, f);
        code_values<FP8>(w.y, f + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= sc;
        *reinterpret_cast<uint4 *>(o + (int64_t)t * ld + d) =
            make_uint4(narrow2<SRC>(f[0], f[1]), narrow2<SRC>(f[2], f[3]), narrow2<SRC>(f[4], f[5]),
                       narrow2<SRC>(f[6], f[7]));
      }
    } else {
      const int groups = (rows + 3) / 4;
      for (int i = tid; i < groups * dch; i += 256) {
        const int d = (i % dch) * 8, t = (i / dch) * 4;
        float f[8][4];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = t < have ? *reinterpret_cast<const uint32_t *>(codes + (int64_t)(d + e) * P + t) : 0u;
          code_values<FP8>(w, f[e]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (t + j >= rows) break;
          float g[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = t + j < have ? f[e][j] * sc : 0.f;
          *reinterpret_cast<uint4 *>(o + (int64_t)(t + j) * ld + d) =
              make_uint4(narrow2<SRC>(g[0], g[1]), narrow2<SRC>(g[2], g[3]), narrow2<SRC>(g[4], g[5]),
                         narrow2<SRC>(g[6], g[7]));
        }
      }
    }
  }
}

hipError_t launch_kv_read(int src, const KvCacheArgs &c, const KvReadArgs &p, hipStream_t st) {
  if (c.seqs == 0 || c.rows == 0) return hipSuccess;
  // no sequence has more pages than rows, and rows past the table's pages are
  // walked by the same workgroups
  const int64_t span = ((int64_t)c.rows + c.page - 1) / c.page;
  const unsigned gx = (unsigned)(span < c.width ? span : (c.width > 0 ? c.width : 1));
  const dim3 grid(gx, (unsigned)c.heads * 2, (unsigned)c.seqs);
  if (src == SRC_BF16) {
    if (c.fp8) kv_read_kernel<SRC_BF16, true><<<grid, 256, 0, st>>>(c, p);
    else kv_read_kernel<SRC_BF16, false><<<grid, 256, 0, st>>>(c, p);
  } else {
    if (c.fp8) kv_read_kernel<SRC_F16, true><<<grid, 256, 0, st>>>(c, p);
    else kv_read_kernel<SRC_F16, false><<<grid, 256, 0, st>>>(c, p);
  }
  return hipGetLastError();
}

}  // namespace dsl
