// Row quantizers: the residual's addition, the RMS norm and an 8-bit result in
// one pass, and int8 codes of plain rows.
//
//   h = x + r,   y = h / sqrt(mean(h^2) + eps) * w,
//   s = max(max|y| / top, 1e-12) over a row, or over each 128 columns,
//   q = round(y / s) (int8, top 127) or e4m3(y / s) (top 448).
//
// One workgroup holds a row in registers, eight elements per thread and
// chunk, so x, r and w are read once and h, q and the scales written once:
// 3 * 2 + 1 bytes per element, which bounds a long call.  h is stored in the
// source's type; norm and codes come from the sum before that rounding, and y
// is not rounded before it is quantized (bf16 holds 8 bits: codes of a rounded
// y would sit on ties and differ in a quarter of their upper half).  The
// quotients y / s take one Markstein step from v_rcp_f32 (common.h, quot): y
// carries the rounding of its own products, so no IEEE quotient is owed.  The
// codes of plain rows are those of the IEEE quotient.
//
// A row takes as many threads as it has chunks, up to 512, and 1024 for few rows
// (then two and four chunks each): with few rows a call is one load latency, one reduction
// for the sum and one for the maximum.  With many, workgroups walk rows, the next
// row's loads behind this one's reductions, and the weights stay in registers.
#include "launch.h"
#include "quant_core.h"
#include "serve_args.h"

namespace dsl {

template <int SRC>
DSL_DEV void widen8(const uint4 &v, float *f) {
  if constexpr (SRC == SRC_BF16) {
    unpack8(v, f);
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
      f[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
    }
  }
}

template <int SRC>
DSL_DEV uint4 narrow8(const float *f) {
  if constexpr (SRC == SRC_BF16) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i]) |
             (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * i + 1]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

DSL_DEV uint32_t int8_pack4(float a, float b, float c, float d) {
  const uint32_t ia = (uint32_t)(int)__builtin_rintf(a), ib = (uint32_t)(int)__builtin_rintf(b);
  const uint32_t ic = (uint32_t)(int)__builtin_rintf(c), id = (uint32_t)(int)__builtin_rintf(d);
  const uint32_t lo = __builtin_amdgcn_perm(ib, ia, 0x0c0c0400u), hi = __builtin_amdgcn_perm(id, ic, 0x04000c0cu);
  return lo | hi;
}

template <bool MAX>
DSL_DEV float join(float a, float b) {
  if constexpr (MAX) return fmaxf(a, b);
  else return a + b;
}

// Sum or maximum over the workgroup; every thread gets it.  One barrier: each
// reduction has an array of its own.
template <int NT, bool MAX>
DSL_DEV float reduce(float v, float *sh) {
  v = join<MAX>(v, dpp_f<0xb1>(v));
  v = join<MAX>(v, dpp_f<0x4e>(v));
  v = join<MAX>(v, dpp_f<0x141>(v));
  v = join<MAX>(v, dpp_f<0x140>(v));
  v = join<MAX>(v, __shfl_xor(v, 16));
  v = join<MAX>(v, __shfl_xor(v, 32));
  constexpr int NW = NT / 64;
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v = join<MAX>(v, sh[i]);
  }
  return v;
}

// Waves of a CU that walk the rows.  3001x7168 fp16: 37 us with 16, 38 with 24, 40
// with 32 and 50 with 64; with a workgroup per row, its loads, reductions and stores
// one after another, 62.
constexpr int kResident = 16;

template <int SRC, int FMT, bool NORM, bool W32, int NT, int CPL>
__global__ __launch_bounds__(NT) void row_quant_kernel(const RowQuantArgs p) {
  __shared__ float sh_sum[2][NT / 64], sh_max[2][NT / 64];   // by turns: a row's readers may still be at theirs
  constexpr int ESZ = SRC == SRC_F32 ? 4 : 2, V = ESZ / 2;   // 16-byte words per chunk
  const int tid = threadIdx.x, nch = p.cols >> 3;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 xa[CPL][V], ra[CPL], wa[CPL][W32 ? 2 : 1];
  auto load = [&](int64_t row) __attribute__((always_inline)) {
    const uint4 *xr = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(p.x) + row * p.ldx * ESZ);
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const int c = tid + NT * j;
#pragma unroll
      for (int h = 0; h < V; ++h) xa[j][h] = c < nch ? xr[V * c + h] : zero;
    }
    if constexpr (NORM) {
      const uint4 *rr = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(p.r) + row * p.ldr * ESZ);
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const int c = tid + NT * j;
        ra[j] = p.r && c < nch ? rr[c] : zero;
      }
    }
  };
  load(blockIdx.x);
  if constexpr (NORM) {
    // the weights with the first row: their latency hides behind it
    const uint4 *w4 = static_cast<const uint4 *>(p.w);
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const int c = tid + NT * j;
#pragma unroll
      for (int h = 0; h < (W32 ? 2 : 1); ++h) wa[j][h] = c < nch ? w4[W32 ? 2 * c + h : c] : zero;
    }
  }
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    float f[CPL][8];
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      if constexpr (SRC == SRC_F32) {
        const uint32_t b[8] = {xa[j][0].x, xa[j][0].y, xa[j][0].z, xa[j][0].w,
                               xa[j][V - 1].x, xa[j][V - 1].y, xa[j][V - 1].z, xa[j][V - 1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) f[j][e] = u2f(b[e]);
      } else {
        widen8<SRC>(xa[j][0], f[j]);
      }
    }
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        const int c = tid + NT * j;
        float r[8];
        widen8<SRC>(ra[j], r);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[j][e] += r[e];
          ss += f[j][e] * f[j][e];
        }
        if (p.h && c < nch)
          reinterpret_cast<uint4 *>(static_cast<uint8_t *>(p.h) + row * p.cols * 2)[c] = narrow8<SRC>(f[j]);
      }
      if (row + gridDim.x < p.rows) load(row + gridDim.x);     // the next row, behind this one's reductions
      ss = reduce<NT, false>(ss, sh_sum[turn]);
      const float rinv = 1.0f / __builtin_sqrtf(ss / (float)p.cols + p.eps);
#pragma unroll
      for (int j = 0; j < CPL; ++j) {
        float w[8];
        if constexpr (W32) {
          const uint32_t b[8] = {wa[j][0].x, wa[j][0].y, wa[j][0].z, wa[j][0].w,
                                 wa[j][1].x, wa[j][1].y, wa[j][1].z, wa[j][1].w};
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = u2f(b[e]);
        } else {
          unpack8(wa[j][0], w);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[j][e] = (f[j][e] * rinv) * w[e];
      }
    }
    if constexpr (!NORM) {
      if (row + gridDim.x < p.rows) load(row + gridDim.x);
    }
    constexpr float TOP = FMT == RQ_INT8 ? 127.0f : kE4M3Max;
    float s = 0.f;
    if constexpr (FMT != RQ_FP8_G128) {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < CPL; ++j) m = fmaxf(m, amax8(f[j]));
      m = reduce<NT, true>(m, sh_max[turn]);
      s = fmaxf(__fdiv_rn(m, TOP), kScaleFloor);
      if (tid == 0) p.scales[row] = s;
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
      const int c = tid + NT * j;
      if constexpr (FMT == RQ_FP8_G128) {
        s = fmaxf(__fdiv_rn(team_max<16>(amax8(f[j])), TOP), kScaleFloor);
        if ((tid & 15) == 0 && c < nch) p.scales[row * ((p.cols + 127) / 128) + (c >> 4)] = s;
      }
      if (c >= nch) continue;
      uint2 code;
      if constexpr (FMT != RQ_INT8) {
        code = e4m3_quot8(f[j], s, rcp_approx(s));
      } else {
        float v[8];
        const float r = rcp_approx(s);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = NORM ? quot(f[j][e], s, r) : __fdiv_rn(f[j][e], s);
        code = make_uint2(int8_pack4(v[0], v[1], v[2], v[3]), int8_pack4(v[4], v[5], v[6], v[7]));
      }
      reinterpret_cast<uint2 *>(p.q + row * p.cols)[c] = code;
    }
  }
}

template <int SRC, int FMT, bool NORM, bool W32 = false>
static hipError_t launch_rows(const RowQuantArgs &p, hipStream_t st) {
  const int nch = p.cols / 8;
  if (p.rows == 0) return hipSuccess;
  // Up to 1024 chunks of few rows by 1024 threads: 7168 columns, fp32 weights, 16 / 400
  // / 512 / 3001 rows 7.4 / 11.5 / 11.8 / 39.3 us, by 512 of two chunks 7.4 / 13.3 / 13.5
  // / 36.6.
  const int few = 2 * device_cu_count();
  // workgroups that are resident together, each walking its rows
  const int waves = nch <= 64 ? 1 : nch <= 128 ? 2 : nch <= 256 ? 4 : nch <= 512 ? 8 : nch <= 1024 && p.rows > few ? 8 : 16;
  const int64_t most = (int64_t)device_cu_count() * (kResident / waves);
  const unsigned grid = (unsigned)(p.rows < most ? p.rows : most);
  if (nch <= 64) row_quant_kernel<SRC, FMT, NORM, W32, 64, 1><<<grid, 64, 0, st>>>(p);
  else if (nch <= 128) row_quant_kernel<SRC, FMT, NORM, W32, 128, 1><<<grid, 128, 0, st>>>(p);
  else if (nch <= 256) row_quant_kernel<SRC, FMT, NORM, W32, 256, 1><<<grid, 256, 0, st>>>(p);
  else if (nch <= 512) row_quant_kernel<SRC, FMT, NORM, W32, 512, 1><<<grid, 512, 0, st>>>(p);
  else if (nch <= 1024 && p.rows > few) row_quant_kernel<SRC, FMT, NORM, W32, 512, 2><<<grid, 512, 0, st>>>(p);
  else if (nch <= 1024) row_quant_kernel<SRC, FMT, NORM, W32, 1024, 1><<<grid, 1024, 0, st>>>(p);
  else if (nch <= 2048) row_quant_kernel<SRC, FMT, NORM, W32, 1024, 2><<<grid, 1024, 0, st>>>(p);
  else row_quant_kernel<SRC, FMT, NORM, W32, 1024, 4><<<grid, 1024, 0, st>>>(p);
  return hipGetLastError();
}

hipError_t launch_row_quant(int src, const RowQuantArgs &p, hipStream_t st) {
  if (src == SRC_BF16) return launch_rows<SRC_BF16, RQ_INT8, false>(p, st);
  if (src == SRC_F16) return launch_rows<SRC_F16, RQ_INT8, false>(p, st);
  return launch_rows<SRC_F32, RQ_INT8, false>(p, st);
}

template <int SRC, bool W32>
static hipError_t launch_norm(int fmt, const RowQuantArgs &p, hipStream_t st) {
  if (fmt == RQ_INT8) return launch_rows<SRC, RQ_INT8, true, W32>(p, st);
  if (fmt == RQ_FP8) return launch_rows<SRC, RQ_FP8, true, W32>(p, st);
  return launch_rows<SRC, RQ_FP8_G128, true, W32>(p, st);
}

hipError_t launch_add_rmsnorm_quant(int src, int fmt, const RowQuantArgs &p, hipStream_t st) {
  if (src == SRC_BF16) return p.w_f32 ? launch_norm<SRC_BF16, true>(fmt, p, st) : launch_norm<SRC_BF16, false>(fmt, p, st);
  return p.w_f32 ? launch_norm<SRC_F16, true>(fmt, p, st) : launch_norm<SRC_F16, false>(fmt, p, st);
}

}  // namespace dsl
