// The pages of the paged 8-bit cache between steps: sequences that fork, are
// dropped or grow, and live pages moved to the cache's front.
//
// refs[p] counts the table entries that hold page p (and whatever else keeps
// it); pages without one are free.  A step is a function of its inputs: lengths,
// table and counts are written anew, and of the cache only pages change that no
// sequence of the new step held before.
//
// The bookkeeping is a few thousand integers and bound by latency, so one
// workgroup does all of it up to kSmallWork entries, a barrier between the phases;
// larger tables take a launch per phase, and only the search for free pages
// stays with one workgroup.  Values that other threads change by atomics are read
// past the first-level cache.  Copies are bound by bytes: 16 KB pieces of all
// pages, dealt to as many workgroups as there may be pieces.  (16 sequences of 4001 tokens
// forked into 256, 25000 entries and pages: 18 us, and 8 for 240 copies of 128 KB; 8 beams: 9 and 3.
// 1 GB compacted: 13, and 107 for 2000 pages, 5.0 TB/s.)
#include "common.h"
#include "generate_args.h"
#include "launch.h"

namespace dsl {

constexpr int kBook = 1024;                      // threads of the bookkeeping workgroup
// Table entries (old and new) and pages up to which one workgroup keeps the books; past
// them a launch per phase.  The whole call, tables and counts in the caches: 8000 of them 15.6
// and 18.9 us, 24000 23.8 and 22.3, 63000 39 and 22; not in them: 20.7 and 27.2, 30 and
// 36.6, 35000 33 and 35.6, 45000 40 and 36, 63000 47 and 35.
constexpr int64_t kSmallWork = 1 << 15;
constexpr int kPiece = 16384;                    // bytes of a copy's piece

DSL_DEV int ld_shared(const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DSL_DEV void st_shared(int32_t *p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DSL_DEV void add_shared(int32_t *p, int v) { __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DSL_DEV void min_shared(int32_t *p, int v) { __hip_atomic_fetch_min(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Phase boundary of one workgroup: every access of it has reached L2.
DSL_DEV void phase_end() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}

// The exclusive sum over a workgroup of kBook threads; `total` is that of all.
template <class T>
DSL_DEV T scan_book(T v, T &total, T *sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T u = __shfl_up(s, o);
    if (lane >= o) s += u;
  }
  __syncthreads();                               // the last scan's readers
  if (lane == 63) sh[wave] = s;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kBook / 64; ++w) {
    if (w < wave) before += sh[w];
    all += sh[w];
  }
  total = all;
  return before + s - v;
}

// ------------------------------------------------------------------- fork --
// The workspace: children of a sequence, the first of them; per child its first
// fresh page's rank and its copies' rank; free pages; the copies.
struct ForkSpace {
  int32_t *count, *first, *off, *list, *from, *to, *copies;
  DSL_HD ForkSpace(const ForkArgs &p)
      : count(p.ws), first(count + p.seqs), off(first + p.seqs), list(off + p.children + 1), from(list + p.pages),
        to(from + p.children), copies(to + p.children) {}
};
size_t fork_workspace_bytes(int seqs, int width, int children, int pages) {
  return ((size_t)2 * seqs + 3 * (size_t)children + 1 + pages + 1) * sizeof(int32_t);
}

// A child: its parent (-1: none), that one's tokens, the entries held whole, the
// page that is partly filled (-1: none), and the fresh entries begin .. end.
struct Child {
  int parent, len, more, full, part, begin;
  int64_t end;
};
DSL_DEV int valid_page(const ForkArgs &p, int a, int i) {
  const int v = p.table[(int64_t)a * p.table_ld + i];
  return v >= 0 && v < p.pages ? v : -1;
}
DSL_DEV Child child_of(const ForkArgs &p, int a, int c) {
  Child k;
  k.parent = a >= 0 && a < p.seqs ? a : -1;
  const int n = k.parent < 0 ? 0 : p.lens[k.parent];
  k.len = n > 0 ? n : 0;
  const int m = p.more ? p.more[c] : p.more_all;
  k.more = m > 0 ? m : 0;
  const int whole = k.len / p.page;
  k.full = whole < p.width ? whole : p.width;
  k.part = k.len % p.page != 0 && whole < p.width ? valid_page(p, k.parent, whole) : -1;
  k.begin = (int)(((int64_t)k.len + p.page - 1) / p.page);
  k.end = ((int64_t)k.len + k.more + p.page - 1) / p.page;
  return k;
}

DSL_DEV void fork_clear(const ForkArgs &p, int64_t tid, int64_t n) {
  const ForkSpace s(p);
  for (int64_t i = tid; i < p.pages; i += n) st_shared(p.out_refs + i, p.refs[i]);
  for (int64_t i = tid; i < p.seqs; i += n) {
    st_shared(s.count + i, 0);
    st_shared(s.first + i, 0x7fffffff);
  }
}
DSL_DEV void fork_count(const ForkArgs &p, int64_t tid, int64_t n) {
  const ForkSpace s(p);
  for (int64_t c = tid; c < p.children; c += n) {
    const int a = p.parents[c];
    if (a < 0 || a >= p.seqs) continue;
    add_shared(s.count + a, 1);
    min_shared(s.first + a, (int)c);
  }
}
// A wave per row: the counts of the old entries, then the children's held entries.
DSL_DEV void fork_rows(const ForkArgs &p, int64_t wave, int64_t waves) {
  const ForkSpace s(p);
  const int lane = threadIdx.x & 63;
  for (int64_t a = wave; a < p.seqs; a += waves) {
    const int kids = ld_shared(s.count + a);
    const int len = p.lens[a] > 0 ? p.lens[a] : 0, whole = len / p.page;
    for (int i = lane; i < p.width; i += 64) {
      const int v = valid_page(p, (int)a, i);
      if (v < 0) continue;
      const int now = i < whole ? kids : (i == whole && len % p.page != 0 && kids > 0 ? 1 : 0);
      if (now != 1) add_shared(p.out_refs + v, now - 1);
    }
  }
  for (int64_t c = wave; c < p.children; c += waves) {
    const Child k = child_of(p, p.parents[c], (int)c);
    const bool keeps = k.part >= 0 && ld_shared(s.first + k.parent) == (int)c;
    for (int i = lane; i < p.width; i += 64) {
      int v = -1;
      if (i < k.full) v = valid_page(p, k.parent, i);
      else if (i == k.full && keeps) v = k.part;
      p.out_table[c * p.width + i] = v;
    }
    if (lane == 0) {
      const int64_t len = (int64_t)k.len + k.more;
      p.out_lens[c] = (int)(len < 0x7fffffff ? len : 0x7fffffff);
    }
  }
}
// The k-th fresh entry that is asked for (by child, a copy before the new tokens')
// gets the k-th free page.
// (`kids` has the children, `keeper(a)` the first child of a sequence, `off` room for
// children + 1 ranks.)
template <class Kids, class Keeper>
DSL_DEV void fork_give(const ForkArgs &p, const Kids &kids, const Keeper &keeper, int32_t *off) {
  __shared__ int64_t sh[kBook / 64];
  const ForkSpace s(p);
  const int tid = threadIdx.x;
  int64_t asked = 0, beyond = 0, copies = 0;
  for (int64_t c0 = 0; c0 < p.children; c0 += kBook) {
    const int64_t c = c0 + tid;
    int64_t mine = 0;
    bool copied = false;
    int part = -1;
    if (c < p.children) {
      const Child k = kids((int)c);
      const int64_t e = k.end < p.width ? k.end : p.width;
      part = k.part;
      copied = part >= 0 && keeper(k.parent) != (int)c;
      const int64_t fresh = e > k.begin ? e - k.begin : 0;
      mine = fresh + copied;
      beyond += (k.end > k.begin ? k.end - k.begin : 0) - fresh;
    }
    int64_t all;                                 // both ranks in one sum: copies of 1024 children below
    const int64_t both = scan_book(mine * (2 * kBook) + copied, all, sh);
    const int64_t rank = asked + both / (2 * kBook), cr = copies + both % (2 * kBook);
    if (c < p.children) off[c] = (int)(rank < p.pages ? rank : p.pages);
    asked += all / (2 * kBook);
    if (copied) {
      s.from[cr] = part;
      s.to[cr] = (int)(rank < p.pages ? rank : p.pages);   // its fresh page's rank, for now
    }
    copies += all % (2 * kBook);
  }
  {
    int64_t all;
    scan_book(beyond, all, sh);
    beyond = all;
  }
  const int need = (int)(asked < p.pages ? asked : p.pages);
  if (tid == 0) off[p.children] = need;
  int found = 0;
  for (int64_t p0 = 0; p0 < p.pages && found < need; p0 += 4 * kBook) {
    int at[4], zeros = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = p0 + 4 * tid + j;
      at[j] = i < p.pages ? ld_shared(p.out_refs + i) : 1;
      zeros += at[j] == 0;
    }
    int64_t all;
    int rank = found + (int)scan_book((int64_t)zeros, all, sh);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at[j] == 0) {
        if (rank < need) s.list[rank] = (int)(p0 + 4 * tid + j);
        ++rank;
      }
    found += (int)all;
  }
  const int given = found < need ? found : need;
  __syncthreads();
  for (int k = tid; k < given; k += kBook) {
    int lo = 0, hi = p.children;                 // off[lo] <= k < off[hi]
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (off[mid] <= k) lo = mid;
      else hi = mid;
    }
    const Child c = kids(lo);
    const bool copied = c.part >= 0 && keeper(c.parent) != lo;
    const int j = k - off[lo], page = s.list[k];
    p.out_table[(int64_t)lo * p.width + (copied && j == 0 ? c.full : c.begin + j - copied)] = page;
    st_shared(p.out_refs + page, 1);
  }
  for (int64_t i = tid; i < copies; i += kBook) s.to[i] = s.to[i] < given ? s.list[s.to[i]] : -1;
  if (tid == 0) {
    *s.copies = (int)copies;
    const int64_t lacks = asked + beyond - given;
    *p.lacking = (int)(lacks < 0x7fffffff ? lacks : 0x7fffffff);
  }
}

// All of it by one workgroup, for kBook sequences and children at most: what a child and a
// sequence are in shared memory, a thread per table entry, four or eight loads at a time.
__global__ __launch_bounds__(kBook) void fork_book_kernel(const ForkArgs p) {
  __shared__ int s_count[kBook], s_first[kBook], s_whole[kBook], s_off[kBook + 1];
  __shared__ Child s_child[kBook];
  const int tid = threadIdx.x;
  for (int i0 = tid; i0 < p.pages; i0 += 8 * kBook) {
    int v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i0 + u * kBook < p.pages ? p.refs[i0 + u * kBook] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u * kBook < p.pages) st_shared(p.out_refs + i0 + u * kBook, v[u]);
  }
  s_count[tid] = 0;
  s_first[tid] = 0x7fffffff;
  const int n = tid < p.seqs && p.lens[tid] > 0 ? p.lens[tid] : 0;
  s_whole[tid] = n / p.page * 2 + (n % p.page != 0);           // whole pages, and whether there is a part of one
  __syncthreads();
  if (tid < p.children) {
    const Child k = child_of(p, p.parents[tid], tid);
    s_child[tid] = k;
    if (k.parent >= 0) {
      atomicAdd(&s_count[k.parent], 1);
      atomicMin(&s_first[k.parent], tid);
    }
    const int64_t len = (int64_t)k.len + k.more;
    p.out_lens[tid] = (int)(len < 0x7fffffff ? len : 0x7fffffff);
  }
  phase_end();
  constexpr int U = 8;
  const int old = p.seqs * p.width, held = p.children * p.width;
  const float inv = 1.0f / (float)p.width;       // (e + 0.5) inv is within e 2^-22 / width of its value, so right below 2^21
  for (int e0 = tid; e0 < old; e0 += U * kBook) {
    int v[U], row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kBook;
      row[u] = (int)(((float)e + 0.5f) * inv);
      v[u] = e < old ? valid_page(p, row[u], e - row[u] * p.width) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v[u] < 0) continue;
      const int i = e0 + u * kBook - row[u] * p.width, has = s_whole[row[u]], whole = has >> 1, kids = s_count[row[u]];
      const int now = i < whole ? kids : (i == whole && (has & 1) && kids > 0 ? 1 : 0);
      if (now != 1) add_shared(p.out_refs + v[u], now - 1);
    }
  }
  for (int e0 = tid; e0 < held; e0 += U * kBook) {
    int v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kBook, c = e < held ? (int)(((float)e + 0.5f) * inv) : 0, i = e - c * p.width;
      const Child &k = s_child[c];
      v[u] = -1;
      if (e >= held) continue;
      if (i < k.full) v[u] = valid_page(p, k.parent, i);
      else if (i == k.full && k.part >= 0 && s_first[k.parent] == c) v[u] = k.part;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (e0 + u * kBook < held) p.out_table[e0 + u * kBook] = v[u];
  }
  phase_end();
  fork_give(p, [&](int c) { return s_child[c]; }, [&](int a) { return s_first[a]; }, s_off);
}
__global__ __launch_bounds__(256) void fork_clear_kernel(const ForkArgs p) {
  fork_clear(p, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}
__global__ __launch_bounds__(256) void fork_count_kernel(const ForkArgs p) {
  fork_count(p, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}
__global__ __launch_bounds__(256) void fork_rows_kernel(const ForkArgs p) {
  fork_rows(p, (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), (int64_t)gridDim.x * 4);
}
__global__ __launch_bounds__(kBook) void fork_give_kernel(const ForkArgs p) {
  const ForkSpace s(p);
  fork_give(p, [&](int c) { return child_of(p, p.parents[c], c); }, [&](int a) { return ld_shared(s.first + a); }, s.off);
}

// ----------------------------------------------------------------- copies --
// Piece `at` of a page: keys, then values; scales with the first.
DSL_DEV void copy_piece(const PageArgs &c, int from, int to, int64_t at) {
  const int64_t half = (c.bytes + kPiece - 1) / kPiece;
  const bool vals = at >= half;
  const int64_t begin = (vals ? at - half : at) * kPiece;
  const int64_t n = c.bytes - begin < kPiece ? c.bytes - begin : kPiece;
  uint8_t *base = (vals ? c.v : c.k) + begin;
  const v4i *x = reinterpret_cast<const v4i *>(base + (int64_t)from * c.bytes);
  v4i *y = reinterpret_cast<v4i *>(base + (int64_t)to * c.bytes);
  const int words = (int)(n >> 4);
  constexpr int U = kPiece / 16 / 256;
  const int tid = threadIdx.x;
  if (words == U * 256) {
    v4i v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = x[tid + 256 * u];
#pragma unroll
    for (int u = 0; u < U; ++u) y[tid + 256 * u] = v[u];
  } else {
    for (int i = tid; i < words; i += 256) y[i] = x[i];
  }
  if (at == 0)
    for (int i = threadIdx.x; i < c.heads; i += 256) {
      c.k_scale[(int64_t)to * c.heads + i] = c.k_scale[(int64_t)from * c.heads + i];
      c.v_scale[(int64_t)to * c.heads + i] = c.v_scale[(int64_t)from * c.heads + i];
    }
}
static int64_t pieces_of(const PageArgs &c) { return 2 * ((c.bytes + kPiece - 1) / kPiece); }

__global__ __launch_bounds__(256) void copy_pages_kernel(const PageArgs c, const int32_t *from, const int32_t *to,
                                                         const int32_t *count, const int64_t pieces) {
  const int64_t n = *count * pieces;
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
    const int k = (int)(i / pieces), t = to[k];
    if (t >= 0) copy_piece(c, from[k], t, i % pieces);
  }
}

static unsigned blocks_for(int64_t items, int64_t each, int64_t most) {
  const int64_t n = (items + each - 1) / each;
  return (unsigned)(n < 1 ? 1 : (n < most ? n : most));
}

hipError_t launch_fork(const PageArgs &c, const ForkArgs &p, hipStream_t st) {
  const int64_t entries = (int64_t)(p.seqs + p.children) * p.width, most = 8 * (int64_t)device_cu_count();
  if (entries + p.pages <= kSmallWork && p.seqs <= kBook && p.children <= kBook) {
    fork_book_kernel<<<1, kBook, 0, st>>>(p);
  } else {
    const int64_t flat = p.pages > p.seqs ? p.pages : p.seqs;
    fork_clear_kernel<<<blocks_for(flat, 256, most), 256, 0, st>>>(p);
    fork_count_kernel<<<blocks_for(p.children, 256, most), 256, 0, st>>>(p);
    fork_rows_kernel<<<blocks_for((int64_t)p.seqs + p.children, 4, most), 256, 0, st>>>(p);
    fork_give_kernel<<<1, kBook, 0, st>>>(p);
  }
  const ForkSpace s(p);
  const int64_t pieces = pieces_of(c);
  if (p.children > 0 && p.pages > 0)
    copy_pages_kernel<<<blocks_for((int64_t)p.children * pieces, 1, most), 256, 0, st>>>(c, s.from, s.to, s.copies, pieces);
  return hipGetLastError();
}

// ---------------------------------------------------------------- compact --
struct CompactSpace {
  int32_t *from, *to, *count;
  DSL_HD CompactSpace(const CompactArgs &p) : from(p.ws), to(from + p.pages / 2 + 1), count(to + p.pages / 2 + 1) {}
};
size_t compact_workspace_bytes(int pages) { return ((size_t)2 * (pages / 2 + 1) + 1) * sizeof(int32_t); }

// n live pages; the k-th live page from n on goes to the k-th free one before n.
__global__ __launch_bounds__(kBook) void compact_book_kernel(const CompactArgs p) {
  __shared__ int64_t sh[kBook / 64];
  const CompactSpace s(p);
  const int tid = threadIdx.x;
  int mine = 0;
#pragma unroll 4
  for (int64_t i = tid; i < p.pages; i += kBook) mine += p.refs[i] > 0;
  int64_t n;
  scan_book((int64_t)mine, n, sh);
  int64_t before = 0;                            // movers, and holes << 32
  for (int64_t p0 = 0; p0 < p.pages; p0 += 4 * kBook) {
    int at[4];
    int64_t add = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = p0 + 4 * tid + j;
      at[j] = i < p.pages ? p.refs[i] : 0;
      if (i < p.pages) add += i < n ? (int64_t)(at[j] <= 0) << 32 : (int64_t)(at[j] > 0);
    }
    int64_t all;
    int64_t rank = before + scan_book(add, all, sh);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = p0 + 4 * tid + j;
      if (i >= p.pages) break;
      const bool live = at[j] > 0;
      if (i < n) {
        p.moved[i] = live ? (int)i : -1;
        if (live) p.out_refs[i] = at[j];
        else {
          s.to[rank >> 32] = (int)i;
          rank += (int64_t)1 << 32;
        }
      } else {
        p.out_refs[i] = 0;
        if (live) {
          s.from[(uint32_t)rank] = (int)i;
          ++rank;
        } else {
          p.moved[i] = -1;
        }
      }
    }
    before += all;
  }
  const int movers = (int)(uint32_t)before;
  __syncthreads();
  for (int k = tid; k < movers; k += kBook) {
    const int from = s.from[k], to = s.to[k];
    p.moved[from] = to;
    p.out_refs[to] = p.refs[from];
  }
  if (tid == 0) {
    *s.count = movers;
    *p.live = (int)n;
  }
}
__global__ __launch_bounds__(256) void compact_move_kernel(const PageArgs c, const CompactArgs p, const int64_t pieces,
                                                           const int rows) {
  if ((int)blockIdx.x < rows) {                  // the table's rows
    for (int64_t b = blockIdx.x; b < p.seqs; b += rows)
      for (int i = threadIdx.x; i < p.width; i += 256) {
        const int v = p.table[b * p.table_ld + i];
        p.out_table[b * p.width + i] = v >= 0 && v < p.pages ? p.moved[v] : -1;
      }
    return;
  }
  const CompactSpace s(p);
  const int64_t n = *s.count * pieces;
  for (int64_t i = blockIdx.x - rows; i < n; i += gridDim.x - rows) {
    const int k = (int)(i / pieces);
    copy_piece(c, s.from[k], s.to[k], i % pieces);
  }
}

hipError_t launch_compact(const PageArgs &c, const CompactArgs &p, hipStream_t st) {
  compact_book_kernel<<<1, kBook, 0, st>>>(p);
  const int64_t pieces = pieces_of(c), most = 8 * (int64_t)device_cu_count();
  const unsigned rows = p.seqs > 0 && p.width > 0 ? blocks_for(p.seqs, 1, most) : 0;
  const unsigned copies = p.pages > 1 ? blocks_for(p.pages / 2 * pieces, 1, most) : 0;
  if (rows + copies) compact_move_kernel<<<rows + copies, 256, 0, st>>>(c, p, pieces, (int)rows);
  return hipGetLastError();
}

}  // namespace dsl
