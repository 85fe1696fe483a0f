// Log probabilities of given tokens, the entropy and the largest logits of a
// row, in one pass over its logits.
//
// With m = max x, d = (x - m) scale log2(e) in powers of two, S = sum 2^d and T = sum d 2^d:
//   logp(t) = (x_t - m) scale - ln S,  H = (log2 S - T / S) ln 2.
// Every thread keeps m, S and T of its elements in fp32 (S and T join in 64 bits).  m is a
// logit, not a product, so that d is 0 at the maximum whatever the logits' size: the
// difference is formed first, of halves (x / 2 - m / 2 is one fused product and does not
// overflow), and its error is relative to it.
// A masked token, x = -inf, has no part in either sum; a row of nothing else gives
// entropy 0 and -inf for every token; NaN or +inf give NaN.
//
// The largest: by value, then by lowest index, as 64-bit keys (the value's order,
// then the index turned round) that no two elements share.  In the pass a thread
// only notes which of its 16-byte words holds its largest value.  Of these, one
// element per thread, the `top`-th largest is a bound that no element of the
// result lies below, and only threads whose own largest reaches it can hold any: as many
// threads as `top`, so their words are read once more and everything else is not.
// Keys are sorted 64 to a wave, and sorted runs are merged, best 64 kept.
//
// Bound by the logits' bytes: 3001 rows of 100003 in bf16 take 127 us, 4.7 TB/s (with 512
// threads to a workgroup, which wait for the sorts longer, 150 where 256 took 131; 128: 140).
// Few rows are split over workgroups, and a second launch joins the parts: 16 rows of 131071 in
// fp32 take 9.7 and 4.5 us, latency of launches, sums and sorts; the bytes would take 1.6.
#include "common.h"
#include "generate_args.h"
#include "kv_core.h"
#include "launch.h"

namespace dsl {

constexpr int kLogThreads = 256, kLogWaves = kLogThreads / 64;
constexpr double kLog2eD = 1.44269504088896341;
constexpr double kLn2 = 0.693147180559945309417;

// ------------------------------------------------------------------- keys --
DSL_DEV uint64_t key_of(float v, int index) {
  v = v == v ? v + 0.f : -INFINITY;              // -0 is 0; NaN is no candidate before the others
  const uint32_t u = f2u(v);
  return (uint64_t)(u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u)) << 32 | (uint32_t)~(uint32_t)index;
}
DSL_DEV int index_of(uint64_t key) { return (int)~(uint32_t)key; }
DSL_DEV float value_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return u2f(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}

// One step of a bitonic network over the wave: lane l and l ^ J, `larger` to keep the
// larger key.  In registers: data-parallel moves up to 16 lanes, swaps of rows beyond (by
// shuffles 16 rows' 20 best of 131071 took 24 us, so 19).
template <int J>
DSL_DEV uint64_t exchange(uint64_t k, bool larger) {
  const uint32_t lo = (uint32_t)k, hi = (uint32_t)(k >> 32);
  if constexpr (J >= 16) {
    uint64_t a, b;                               // the pair's, in both lanes
    if constexpr (J == 16) {
      const auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
      const auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
      a = (uint64_t)h[0] << 32 | l[0];
      b = (uint64_t)h[1] << 32 | l[1];
    } else {
      const auto l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
      const auto h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
      a = (uint64_t)h[0] << 32 | l[0];
      b = (uint64_t)h[1] << 32 | l[1];
    }
    return (a > b) == larger ? a : b;
  } else {
    auto other = [](uint32_t v) {
      if constexpr (J == 1) return __builtin_amdgcn_update_dpp(v, v, 0xb1, 0xf, 0xf, false);
      if constexpr (J == 2) return __builtin_amdgcn_update_dpp(v, v, 0x4e, 0xf, 0xf, false);
      if constexpr (J == 4) {                    // ^ 7, ^ 3
        v = __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, false);
        return __builtin_amdgcn_update_dpp(v, v, 0x1b, 0xf, 0xf, false);
      }
      if constexpr (J == 8) return __builtin_amdgcn_update_dpp(v, v, 0x128, 0xf, 0xf, false);
    };
    const uint64_t o = (uint64_t)(uint32_t)other(hi) << 32 | (uint32_t)other(lo);
    return (o > k) == larger ? o : k;
  }
}
// Steps J, J / 2 .. 1 of runs of N lanes, falling and rising in turn (N 64: falling).
template <int N, int J>
DSL_DEV uint64_t exchanges(uint64_t k) {
  const int lane = threadIdx.x & 63;
  k = exchange<J>(k, ((lane & J) == 0) == ((lane & N) == 0));
  if constexpr (J > 1) k = exchanges<N, J / 2>(k);
  return k;
}
// The wave's keys in falling order.
DSL_DEV uint64_t sort_wave(uint64_t k) {
  k = exchanges<2, 1>(k);
  k = exchanges<4, 2>(k);
  k = exchanges<8, 4>(k);
  k = exchanges<16, 8>(k);
  k = exchanges<32, 16>(k);
  return exchanges<64, 32>(k);
}
// The best 64 of two runs in falling order, in falling order; b reversed: lane l
// holds b[63 - l].
DSL_DEV uint64_t merge_reversed(uint64_t a, uint64_t b) { return exchanges<64, 32>(a > b ? a : b); }
DSL_DEV uint64_t merge_wave(uint64_t a, uint64_t b) {
  return merge_reversed(a, __shfl((unsigned long long)b, 63 - (int)(threadIdx.x & 63)));
}
// The best 64 of all waves' runs, in runs[0 .. 63] and in wave 0's lanes.
template <int NW>
DSL_DEV uint64_t merge_waves(uint64_t k, uint64_t *runs) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();                               // the last readers of runs
  runs[wave * 64 + lane] = k;
#pragma unroll
  for (int half = NW / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (wave < half) {
      k = merge_reversed(k, runs[(wave + half) * 64 + 63 - lane]);
      runs[wave * 64 + lane] = k;
    }
  }
  __syncthreads();
  return k;
}

// ------------------------------------------------------------------- sums --
struct Sums {
  float m;
  double s, t;
};
// What the halves' differences are multiplied by.
DSL_DEV float twice_scale(const LogprobArgs &p) { return (float)(2.0 * p.scale * kLog2eD); }
DSL_DEV float below(float x, float half_m, float c2) { return __builtin_fmaf(x, 0.5f, -half_m) * c2; }
DSL_DEV Sums join_sums(const Sums &a, const Sums &b, float c2) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  // of a part without a maximum: no sums, or nothing but NaN
  const float da = a.m == -INFINITY ? 0.f : below(a.m, 0.5f * r.m, c2), db = b.m == -INFINITY ? 0.f : below(b.m, 0.5f * r.m, c2);
  const double fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  r.s = a.s * fa + b.s * fb;
  // (a difference past every exponent leaves nothing, and times a sum of 0 no NaN)
  r.t = (a.t + (double)fmaxf(da, -1000.f) * a.s) * fa + (b.t + (double)fmaxf(db, -1000.f) * b.s) * fb;
  return r;
}
DSL_DEV Sums sums_of_wave(Sums v, float c2) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    Sums u;
    u.m = __shfl_xor(v.m, o);
    u.s = __shfl_xor(v.s, o);
    u.t = __shfl_xor(v.t, o);
    v = join_sums(v, u, c2);
  }
  return v;
}
template <int NW>
DSL_DEV Sums sums_of_group(Sums v, Sums *sh, float c2) {
  v = sums_of_wave(v, c2);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) v = join_sums(v, sh[w], c2);
  return v;
}

template <int SRC>
DSL_DEV float logit(const void *x, int64_t at) {
  if constexpr (SRC == SRC_F32) return static_cast<const float *>(x)[at];
  else return widen<SRC>(static_cast<const uint16_t *>(x)[at]);
}
template <int SRC>
constexpr int kWord = SRC == SRC_F32 ? 4 : 8;    // logits of 16 bytes
template <int SRC>
DSL_DEV void widen_word(const uint4 &v, float *f) {
  if constexpr (SRC == SRC_F32) {
    f[0] = u2f(v.x);
    f[1] = u2f(v.y);
    f[2] = u2f(v.z);
    f[3] = u2f(v.w);
  } else {
    widen8s<SRC>(v, f);
  }
}

// What a row's results are made of.
template <int SRC>
DSL_DEV void write_row(const LogprobArgs &p, int row, const Sums &v, uint64_t key, int tid, int threads) {
  const bool none = v.s == 0.0;                  // no token has a probability
  const double ls = none ? 0.0 : log(v.s);
  auto logp = [&](float x) {
    if (none || x == -INFINITY) return v.s == v.s ? -INFINITY : __builtin_nanf("");
    return (float)(((double)x - (double)v.m) * (double)p.scale - ls);
  };
  for (int i = tid; i < p.n_ids; i += threads) {
    const int id = p.ids[(int64_t)row * p.ids_ld + i];
    p.logp[(int64_t)row * p.n_ids + i] =
        logp(id >= 0 && id < p.vocab ? logit<SRC>(p.x, (int64_t)row * p.ld + id) : -INFINITY);
  }
  if (tid == 0) {
    const double h = none ? 0.0 : ls - v.t / v.s * kLn2;
    p.entropy[row] = (float)(h < 0.0 ? 0.0 : h);
  }
  if (tid < p.top) {
    p.top_logp[(int64_t)row * p.top + tid] = logp(value_of(key));
    p.top_ids[(int64_t)row * p.top + tid] = index_of(key);
  }
}

// Parts of split rows: [part] sums, then [part][top] keys.
struct LogParts {
  Sums *sums;
  uint64_t *keys;
  DSL_HD LogParts(void *ws, int64_t parts) : sums(static_cast<Sums *>(ws)), keys(reinterpret_cast<uint64_t *>(sums + parts)) {}
};

template <int SRC, bool TOP>
__global__ __launch_bounds__(kLogThreads) void logprob_kernel(const LogprobArgs p, const int splits) {
  constexpr int E = kWord<SRC>, NT = kLogThreads, U = 4;
  __shared__ Sums s_sums[kLogWaves];
  __shared__ uint64_t s_runs[TOP ? NT : 1], s_cand[TOP ? NT * E + 64 : 1];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = (int)(blockIdx.x / (unsigned)splits), split = (int)(blockIdx.x % (unsigned)splits);
  constexpr int B = SRC == SRC_F32 ? 4 : 2;
  const uint8_t *x = static_cast<const uint8_t *>(p.x) + (int64_t)row * p.ld * B;
  // the row: elements up to the first whole word, words, elements behind them
  int head = (int)((-reinterpret_cast<uintptr_t>(x) & 15) / B);
  head = head < p.vocab ? head : p.vocab;
  const int words = (p.vocab - head) / E, tail = head + words * E;
  const int w0 = (int)((int64_t)words * split / splits), w1 = (int)((int64_t)words * (split + 1) / splits);
  const uint4 *xw = reinterpret_cast<const uint4 *>(x + (int64_t)head * B);
  const float c2 = twice_scale(p);

  float m = -INFINITY, s = 0.f, t = 0.f, best = -INFINITY;
  int bestw = w0 + tid < w1 ? w0 + tid : -1;
  // m to what `top` makes of it, the sums with it; half of m, 0 while there is none.  (No
  // branch: a round's words are computed among each other, 3001 rows of 100003 in bf16 130 us with one, 127 without.)
  auto raise = [&](float top) __attribute__((always_inline)) {
    const float now = fmaxf(m, top), half_m = now == -INFINITY ? 0.f : 0.5f * now;
    const float d = below(m, half_m, c2);        // 0, but -inf at first
    const float f = __builtin_amdgcn_exp2f(d);
    t = (t + fmaxf(d, -1000.f) * s) * f;
    s *= f;
    m = now;
    return half_m;
  };
  auto take = [&](float v, float half_m) __attribute__((always_inline)) {
    const float d = below(v, half_m, c2);
    const float e = __builtin_amdgcn_exp2f(d);
    s += e;
    t = __builtin_fmaf(e, fmaxf(d, -1000.f), t);
  };
  auto word = [&](const uint4 &raw, int w) __attribute__((always_inline)) {
    float f[E], top;
    widen_word<SRC>(raw, f);
    top = f[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, f[e]);
    if (TOP && top > best) {
      best = top;
      bestw = w;
    }
    const float half_m = raise(top);
#pragma unroll
    for (int e = 0; e < E; ++e) take(f[e], half_m);
  };
  int w = w0 + tid;
  for (; w + (U - 1) * NT < w1; w += U * NT) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = xw[w + u * NT];
#pragma unroll
    for (int u = 0; u < U; ++u) word(v[u], w + u * NT);
  }
  if (w < w1) {                                  // the rest, its loads together too
    uint4 v[U - 1];
#pragma unroll
    for (int u = 0; u < U - 1; ++u) v[u] = xw[w + u * NT < w1 ? w + u * NT : w];
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (w + u * NT < w1) word(v[u], w + u * NT);
  }
  // the elements of no whole word: a thread each
  int edge = -1;
  if (split == 0 && tid < head) edge = tid;
  if (split == splits - 1 && tid >= 64 && tail + tid - 64 < p.vocab) edge = tail + tid - 64;
  float edgev = 0.f;
  if (edge >= 0) {
    edgev = logit<SRC>(x, edge);
    take(edgev, raise(edgev));
  }
  const Sums all = sums_of_group<kLogWaves>(Sums{m, s, t}, s_sums, c2);

  uint64_t kept = 0;                             // the wave's best, falling
  if constexpr (TOP) {
    auto read = [&](int at, float *f) __attribute__((always_inline)) {
      widen_word<SRC>(xw[at], f);
    };
    uint64_t mine = 0;
    if (bestw >= 0) {
      float f[E];
      read(bestw, f);
#pragma unroll
      for (int e = E - 1; e >= 0; --e) {
        const uint64_t k = key_of(f[e], head + bestw * E + e);
        mine = k > mine ? k : mine;
      }
    }
    merge_waves<kLogWaves>(sort_wave(mine), s_runs);
    const uint64_t bound = s_runs[p.top - 1];
    int held = 0;                                // threads that can hold one: s_runs[0 .. held)
    for (int i = 0; i < p.top; ++i) held += s_runs[i] != 0;
    const int each = (w1 - w0 + NT - 1) / NT;    // words of a thread
    const int items = held * each;
    for (int i0 = 0; i0 < items || i0 == 0; i0 += NT) {
      if (tid == 0) s_count = 0;
      __syncthreads();
      auto offer = [&](uint64_t k) __attribute__((always_inline)) {
        if (k >= bound) s_cand[atomicAdd(&s_count, 1)] = k;
      };
      if (i0 == 0 && edge >= 0) offer(key_of(edgev, edge));
      const int i = i0 + tid;
      if (i < items) {
        const int owner = ((index_of(s_runs[i / each]) - head) / E - w0) % NT, at = w0 + owner + i % each * NT;
        if (at < w1) {
          float f[E];
          read(at, f);
#pragma unroll
          for (int e = 0; e < E; ++e) offer(key_of(f[e], head + at * E + e));
        }
      }
      __syncthreads();
      const int n = s_count;
      for (int j = wave * 64; j < n; j += NT) kept = merge_wave(kept, sort_wave(j + lane < n ? s_cand[j + lane] : 0));
      __syncthreads();                           // s_count's readers
    }
    kept = merge_waves<kLogWaves>(kept, s_runs);
  }
  if (splits > 1) {
    const LogParts part(p.ws, (int64_t)p.rows * splits);
    if (tid == 0) part.sums[blockIdx.x] = all;
    if (TOP && tid < p.top) part.keys[(int64_t)blockIdx.x * p.top + tid] = kept;
  } else {
    write_row<SRC>(p, row, all, kept, tid, NT);
  }
}

// A workgroup per row: its parts' sums and keys, each part's already in falling order.
template <int SRC>
__global__ __launch_bounds__(kLogThreads) void logprob_join_kernel(const LogprobArgs p, const int splits) {
  __shared__ Sums s_sums[kLogWaves];
  __shared__ uint64_t s_runs[kLogThreads];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const LogParts part(p.ws, (int64_t)p.rows * splits);
  const uint64_t *keys = part.keys + (int64_t)row * splits * p.top;
  const int back = 63 - lane;
  uint64_t kept = p.top && wave < splits && lane < p.top ? keys[wave * p.top + lane] : 0;
  uint64_t next = p.top && wave + kLogWaves < splits && back < p.top ? keys[(wave + kLogWaves) * p.top + back] : 0;
  const float c2 = twice_scale(p);
  Sums v{-INFINITY, 0.0, 0.0};
  for (int i = tid; i < splits; i += kLogThreads) v = join_sums(v, part.sums[(int64_t)row * splits + i], c2);
  v = sums_of_group<kLogWaves>(v, s_sums, c2);
  if (p.top) {
    for (int k = wave + kLogWaves; k < splits; k += kLogWaves) {
      const uint64_t now = next;
      if (k + kLogWaves < splits && back < p.top) next = keys[(k + kLogWaves) * p.top + back];
      kept = merge_reversed(kept, now);
    }
    kept = merge_waves<kLogWaves>(kept, s_runs);
  }
  write_row<SRC>(p, row, v, kept, tid, kLogThreads);
}

// Parts of a row: a workgroup per CU, of two words for each thread at least.  (16 rows of
// 131071 in fp32: 13.2 us, two workgroups per CU 15.1; 64: 16.9 and 16.4, 128: 25.7 and 21.4, 256:
// 34.3 and 33, 400: 41.6 and 51.5; of 100003 in bf16 16: 13.6 and 15, 128: 16.5 and 17.3, 400: 27.7 and 30.9.)
static int logprob_splits(int src, int rows, int vocab) {
  const int words = vocab / (src == SRC_F32 ? 4 : 8);
  int64_t s = ((int64_t)device_cu_count() + rows - 1) / (rows > 0 ? rows : 1);
  const int64_t most = words / (2 * kLogThreads);
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > 256 ? 256 : s));
}
size_t logprob_workspace_bytes(int src, int rows, int vocab, int top) {
  const int splits = logprob_splits(src, rows, vocab);
  return splits > 1 ? (size_t)rows * splits * (sizeof(Sums) + top * sizeof(uint64_t)) : 0;
}

template <int SRC>
static hipError_t launch_logprobs_src(const LogprobArgs &p, hipStream_t st) {
  const int splits = logprob_splits(SRC, p.rows, p.vocab);
  const unsigned grid = (unsigned)p.rows * (unsigned)splits;
  if (p.top) logprob_kernel<SRC, true><<<grid, kLogThreads, 0, st>>>(p, splits);
  else logprob_kernel<SRC, false><<<grid, kLogThreads, 0, st>>>(p, splits);
  if (splits > 1) logprob_join_kernel<SRC><<<(unsigned)p.rows, kLogThreads, 0, st>>>(p, splits);
  return hipGetLastError();
}
hipError_t launch_logprobs(int src, const LogprobArgs &p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  if (src == SRC_BF16) return launch_logprobs_src<SRC_BF16>(p, st);
  if (src == SRC_F16) return launch_logprobs_src<SRC_F16>(p, st);
  return launch_logprobs_src<SRC_F32>(p, st);
}

}  // namespace dsl
