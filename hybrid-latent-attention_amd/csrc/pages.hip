// A pool of cache pages: requests that share, drop and take pages, the compaction of the pages in use, and page copies.
//
// tables [R, cols]: the pages of request r, -1 behind its last; lengths [R]: its rows; refs [N]: how many requests hold a page;
// free: bit p % 32 of word p / 32 is set where refs[p] == 0. Every result is a function of the pool and the arguments alone
// (free pages are taken lowest first, in the order of requests and of their columns), whatever the order of the atomics.
// The bookkeeping is a few KB to a MB of scattered words: latency, not bytes. One workgroup takes what needs an order (the
// bit per page makes 200,000 pages 25 KB of it); drops and forks go a workgroup per request.
#include "common.h"

namespace hla {
namespace {

constexpr int kPoolThreads = 1024, kPoolWaves = kPoolThreads / 64;
constexpr int kMaxRequests = 8192;

struct Pool {
  int32_t* tables;
  int64_t t_st;
  int R, cols;
  int32_t* lengths;
  int32_t* refs;
  int N;
  uint32_t* free;
  int block;
};

__device__ __forceinline__ int pages_of(const Pool& p, int64_t rows) { return (int)((rows + p.block - 1) / p.block); }
__device__ __forceinline__ int rows_of(const Pool& p, int32_t length) {  // a length that the table can hold
  return (int)min((int64_t)max(length, 0), min((int64_t)p.cols * p.block, (int64_t)INT32_MAX));
}
__device__ __forceinline__ bool is_page(const Pool& p, int32_t page) { return page >= 0 && page < p.N; }

__device__ __forceinline__ void drop_page(const Pool& p, int32_t page) {
  if (is_page(p, page) && atomicSub(&p.refs[page], 1) == 1) atomicOr(&p.free[page >> 5], 1u << (page & 31));
}

// ---- release -----------------------------------------------------------------------------------------------------
// Request requests[i] keeps its first to[i] rows (none without `to`). The lengths are lowered atomically: a request named
// twice drops each of its columns once, in whatever order.
__global__ __launch_bounds__(256) void pool_release_kernel(Pool p, const int32_t* requests, const int32_t* to) {
  __shared__ int32_t before;
  const int r = requests[blockIdx.x];
  if (r < 0 || r >= p.R) return;
  const int left = to ? max(to[blockIdx.x], 0) : 0;
  if (threadIdx.x == 0) before = atomicMin(&p.lengths[r], left);
  __syncthreads();
  const int had = pages_of(p, rows_of(p, before));
  for (int c = pages_of(p, left) + threadIdx.x; c < had; c += 256) {
    int32_t* entry = p.tables + r * p.t_st + c;
    drop_page(p, *entry);
    *entry = -1;
  }
}

// ---- fork --------------------------------------------------------------------------------------------------------
// Request children[i] takes over the pages and the length of parents[i]. Refused: numbers outside the pool, children with rows,
// children named before, parents that the list names as children (what they hold would depend on the order).
__global__ __launch_bounds__(256) void pool_fork_kernel(Pool p, const int32_t* parents, const int32_t* children, int n,
                                                        uint8_t* ok) {
  const int i = blockIdx.x;
  const int parent = parents[i], child = children[i];
  bool bad = parent < 0 || parent >= p.R || child < 0 || child >= p.R;
  if (!bad)
    for (int j = threadIdx.x; j < n; j += 256) {
      const int c = children[j];
      bad = bad || c == parent || (c == child && j < i);
    }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) ok[i] = 0;
    return;
  }
  const int had = p.lengths[child];   // (written by this workgroup alone, below)
  const int32_t length = p.lengths[parent];
  __syncthreads();
  if (threadIdx.x == 0) {
    ok[i] = had <= 0;
    if (had <= 0) p.lengths[child] = length;
  }
  if (had > 0) return;
  const int held = pages_of(p, rows_of(p, length));
  for (int c = threadIdx.x; c < held; c += 256) {
    const int32_t page = p.tables[parent * p.t_st + c];
    p.tables[child * p.t_st + c] = page;
    if (is_page(p, page)) atomicAdd(&p.refs[page], 1);
  }
}

// ---- scans of a workgroup ------------------------------------------------------------------------------------------
// Exclusive prefix sum over the workgroup's threads; `total` is their sum. `sums` holds kPoolWaves + 1 entries.
__device__ __forceinline__ int64_t pool_scan(int64_t v, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t x = v;
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();   // sums may still be read from a call before
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  int64_t at = 0;
  total = 0;
  for (int w = 0; w < kPoolWaves; ++w) {
    if (w == wave) at = total;
    total += sums[w];
  }
  return at + x - v;
}

// Set bits of word w of the pool's bitmap that are pages
__device__ __forceinline__ uint32_t page_bits(const Pool& p, int w) {
  const int words = (p.N + 31) / 32;
  if (w >= words) return 0;
  const int last = p.N & 31;
  return w == words - 1 && last ? (1u << last) - 1 : ~0u;
}

// ---- extend ------------------------------------------------------------------------------------------------------
// Room for the rows [from, to) of every request: columns behind its last get a free page each, columns that hold a shared page
// a free page that the caller fills with a copy of it (the pairs source, target). Requests are served in order as long as what
// they and those before them ask for is there; the others stay as they are. So the pages that served requests get are ranks
// 0, 1, .. of the free pages, and a request's first rank is what those before it ask for.
struct ExtendParams {
  Pool p;
  const int32_t* to;
  const int32_t* from;  // null: the lengths
  uint8_t* ok;
  int32_t *source, *target;
  int32_t* ids;    // with `from`: [R * cols] the pages that are handed out
  int32_t* start;  // with `from`: [R] what a request asks for, then its first rank, -1 where it has to wait
};

__device__ __forceinline__ int64_t count_free(const Pool& p, int64_t* sums) {
  const int words = (p.N + 31) / 32;
  int n = 0;
  for (int w = threadIdx.x; w < words; w += kPoolThreads) n += __popc(p.free[w] & page_bits(p, w));
  int64_t have;
  pool_scan(n, sums, have);
  return have;
}

// The `given` lowest free pages, which are free no longer: 32 * kPoolThreads pages of the pool at a time, place(base, n, page0) with
// the pages of ranks base .. base + n - 1 in `found`, less page0.
constexpr int kAtOnce = 32 * kPoolThreads;

template <typename Place>
__device__ __forceinline__ void hand_out(const Pool& p, int given, int64_t* sums, uint16_t* found, Place place) {
  for (int w0 = 0, base = 0; base < given; w0 += kPoolThreads) {   // (given is no more than there are)
    const int w = w0 + threadIdx.x;
    const uint32_t all = w < (p.N + 31) / 32 ? p.free[w] : 0u;
    uint32_t bits = all & page_bits(p, w);
    const uint32_t others = all ^ bits;
    int64_t total;
    int at = (int)pool_scan(__popc(bits), sums, total);
    const int n = min((int)total, given - base), end = min(n, at + __popc(bits));
    for (; at < end; ++at, bits &= bits - 1) found[at] = (uint16_t)(threadIdx.x * 32 + __ffs((int)bits) - 1);
    const uint32_t kept = others | bits;
    if (kept != all) p.free[w] = kept;
    __syncthreads();
    place(base, n, w0 * 32);
    __syncthreads();
    base += n;
  }
}

// from = lengths[r]: at most one column of a request, its last, is shared, and lists have an entry per request. A call of few
// pages is a chain of loads and barriers; one of many is bound by the instructions of its one workgroup (80,000 of 143,619 pages 31 us: for every
// 32,768 pages of the pool 0.8 in the scan, 2.1 in `found`, 3.4 in tables and counts, whose stores are what they wait for: barriers
// that leave them in flight gain nothing), so a wave places the pages of a request 64 at a time, in consecutive columns, and only
// requests of up to kFew pages are left to their threads. (A wave per 64 pages of the pool in `found`: 42.)
constexpr int kFew = 4;

__global__ __launch_bounds__(kPoolThreads) void pool_extend_kernel(ExtendParams a) {
  __shared__ int64_t sums[kPoolWaves + 1];
  __shared__ int start[kMaxRequests + 1];   // first rank of a request's pages
  __shared__ int column[kMaxRequests];      // where the first of them goes; negative: ~column, in place of a shared page
  __shared__ uint16_t found[kAtOnce];
  __shared__ int given;                     // ranks handed out
  const Pool& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63;

  int64_t asked = 0, have = 0;
  if (tid == 0) given = 0;
  for (int r0 = 0; r0 < p.R; r0 += kPoolThreads) {
    const int r = r0 + tid;
    int need = 0, first = 0, want = 0, length = 0;
    bool fits = true;
    if (r < p.R) {
      length = rows_of(p, p.lengths[r]);
      want = max(a.to[r], length);
      fits = want <= (int64_t)p.cols * p.block;
      if (fits && want > length) {
        const int held = pages_of(p, length), last = length / p.block;
        first = held;
        if (last < held) {   // rows go into the last page
          const int32_t page = p.tables[r * p.t_st + last];
          if (is_page(p, page) && p.refs[page] > 1) first = ~last;
        }
        need = pages_of(p, want) - held + (first < 0);
      }
    }
    if (r0 == 0) have = count_free(p, sums);
    int64_t total;
    const int64_t before = asked + pool_scan(need, sums, total);
    asked += total;
    const bool served = need == 0 || before + need <= have;
    if (r < p.R) {
      start[r] = (int)min(before, have);
      column[r] = first;
      a.source[r] = -1;
      a.target[r] = -1;
      a.ok[r] = fits && served;
      if (served && need) atomicMax(&given, (int)(before + need));
      if (fits && served && want > length) p.lengths[r] = want;
    }
  }
  if (tid == 0) start[p.R] = (int)min(asked, have);
  __syncthreads();
  const int pages = given;   // (the request that is not served first, and all behind it, start at `pages` or later)
  hand_out(p, pages, sums, found, [&](int base, int n, int page0) {
    for (int r0 = 0; r0 < p.R; r0 += kPoolThreads) {
      const int r = r0 + lane * kPoolWaves + (tid >> 6);   // (neighbours with different waves)
      int lo = 0, hi = 0;
      int64_t entry = 0;   // that of rank k is entry + k
      if (r < p.R) {
        const int first_rank = start[r], c = column[r];
        lo = max(first_rank, base);
        hi = min(start[r + 1], base + n);
        entry = r * p.t_st + (c < 0 ? ~c : c) - first_rank;
        if (c < 0 && lo == first_rank && lo < hi) {
          a.source[r] = p.tables[entry + lo];
          a.target[r] = page0 + found[lo - base];
        }
      }
      auto place = [&](int32_t* entries, int k) {
        const int page = page0 + found[k - base];
        entries[k] = page;
        p.refs[page] = 1;
      };
      if (hi - lo <= kFew)
        for (int k = lo; k < hi; ++k) place(p.tables + entry, k);
      for (uint64_t many = __ballot(hi - lo > kFew); many; many &= many - 1) {
        const int from = __ffsll((unsigned long long)many) - 1, end = __builtin_amdgcn_readlane(hi, from);
        int32_t* entries = p.tables + uniform64(__shfl(entry, from));
#pragma unroll 2
        for (int k = __builtin_amdgcn_readlane(lo, from) + lane; k < end; k += 64) place(entries, k);
      }
    }
  });
  // the pages that were copied from lose a holder, after all free bits have been read
  for (int r = tid; r < p.R; r += kPoolThreads)
    if (column[r] < 0 && a.source[r] >= 0) drop_page(p, a.source[r]);
}

// from = write_from[r]: any column may be shared, and lists have an entry per table entry. In three launches: a workgroup per
// request finds what it asks for (`source` has the shared pages), one plans, and a workgroup per request fills its columns: 27 us for
// the 32,640 shared pages of 64 requests of 8160 rows, 19 of them in the one that hands the new ones out (bound by the instructions of
// its one workgroup), 10 where none is shared. (One workgroup for all three: 243, and 59.)
struct Columns {   // columns [c0, c1) have rows to write, those from `held` on no page yet
  int length, want, held, c0, c1;
  bool fits;
};

__device__ __forceinline__ Columns columns_of(const ExtendParams& a, int r) {
  const Pool& p = a.p;
  Columns c;
  c.length = rows_of(p, p.lengths[r]);
  c.want = max(a.to[r], c.length);
  c.held = pages_of(p, c.length);
  c.fits = c.want <= (int64_t)p.cols * p.block;
  const int from = min(max(a.from[r], 0), c.length);
  c.c0 = from / p.block;
  c.c1 = c.fits && c.want > from ? pages_of(p, c.want) : c.c0;
  return c;
}

__global__ __launch_bounds__(256) void pool_need_kernel(ExtendParams a) {
  __shared__ int need;
  const Pool& p = a.p;
  const int r = blockIdx.x;
  const Columns c = columns_of(a, r);
  if (threadIdx.x == 0) need = max(0, c.c1 - max(c.c0, c.held));
  __syncthreads();
  for (int at = threadIdx.x; at < p.cols; at += 256) {
    int32_t shared = -1;
    if (at >= c.c0 && at < min(c.c1, c.held)) {
      const int32_t page = p.tables[r * p.t_st + at];
      if (is_page(p, page) && p.refs[page] > 1) {
        shared = page;
        atomicAdd(&need, 1);
      }
    }
    a.source[(int64_t)r * p.cols + at] = shared;
  }
  __syncthreads();
  if (threadIdx.x == 0) a.start[r] = need;
}

__global__ __launch_bounds__(kPoolThreads) void pool_plan_kernel(ExtendParams a) {
  __shared__ int64_t sums[kPoolWaves + 1];
  __shared__ uint16_t found[kAtOnce];
  __shared__ int given;
  const Pool& p = a.p;
  const int tid = threadIdx.x;
  if (tid == 0) given = 0;
  const int64_t have = count_free(p, sums);
  int64_t asked = 0;
  for (int r0 = 0; r0 < p.R; r0 += kPoolThreads) {
    const int r = r0 + tid;
    const int need = r < p.R ? a.start[r] : 0;
    int64_t total;
    const int64_t before = asked + pool_scan(need, sums, total);
    asked += total;
    if (r < p.R) {
      const bool served = need == 0 || before + need <= have;
      a.start[r] = served ? (int)min(before, have) : -1;
      a.ok[r] = served && columns_of(a, r).fits;
      if (served && need) atomicMax(&given, (int)(before + need));
    }
  }
  __syncthreads();
  hand_out(p, given, sums, found, [&](int base, int n, int page0) {
    for (int i = tid; i < n; i += kPoolThreads) {
      a.ids[base + i] = page0 + found[i];
      p.refs[page0 + found[i]] = 1;
    }
  });
}

__global__ __launch_bounds__(256) void pool_fill_kernel(ExtendParams a) {
  __shared__ int sums[4];
  const Pool& p = a.p;
  const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Columns c = columns_of(a, r);
  int k = a.start[r];
  const bool served = k >= 0;
  for (int c0 = 0; c0 < p.cols; c0 += 256) {
    const int at = c0 + threadIdx.x;
    const int64_t i = (int64_t)r * p.cols + at;
    const int32_t from = at < p.cols && served ? a.source[i] : -1;
    const bool takes = served && at >= c.c0 && at < c.c1 && (at >= c.held || from >= 0);
    const uint64_t mask = __ballot(takes);
    if (lane == 0) sums[wave] = __popcll(mask);
    __syncthreads();
    int before = k;
    for (int w = 0; w < 4; ++w) {
      before += w < wave ? sums[w] : 0;
      k += sums[w];
    }
    int32_t page = -1;
    if (takes) {
      page = a.ids[before + __popcll(mask & ((1ull << lane) - 1))];
      p.tables[r * p.t_st + at] = page;
    }
    if (at < p.cols) {
      a.source[i] = from;
      a.target[i] = from >= 0 ? page : -1;
    }
    if (from >= 0) drop_page(p, from);
    __syncthreads();
  }
  if (threadIdx.x == 0 && served && c.fits && c.want > c.length) p.lengths[r] = c.want;
}

// ---- compaction --------------------------------------------------------------------------------------------------
// With U pages in use, the i-th page in use at or behind U moves to the i-th free place before it. pool_pairs_kernel finds the
// pairs, place[page] for the pages that move, place[N] = U and place[N + 1] = their number; pool_compact_kernel then rewrites
// tables, counts and bits, and ends the lists.
__global__ __launch_bounds__(kPoolThreads) void pool_pairs_kernel(Pool p, int32_t* source, int32_t* target, int32_t* place) {
  __shared__ int64_t sums[kPoolWaves + 1];
  const int tid = threadIdx.x, words = (p.N + 31) / 32;
  const int used = p.N - (int)count_free(p, sums);
  int64_t total;
  int moved = 0;
  for (int pass = 0; pass < 2; ++pass) {   // holes, then movers
    const int first = pass ? used / 32 : 0, end = pass ? words : (used + 31) / 32;
    int base = 0;
    for (int w0 = first; w0 < end; w0 += kPoolThreads) {
      const int w = w0 + tid;
      uint32_t bits = 0;
      if (w < end) {
        bits = p.free[w];
        const int cut = used - 32 * w;   // pages of this word before U
        const uint32_t below = cut >= 32 ? ~0u : cut <= 0 ? 0u : (1u << cut) - 1;
        bits = pass ? ~bits & ~below & page_bits(p, w) : bits & below;
      }
      int rank = base + (int)pool_scan(__popc(bits), sums, total);
      base += (int)total;
      for (; bits; bits &= bits - 1, ++rank) {
        const int page = w * 32 + __ffs((int)bits) - 1;
        (pass ? source : target)[rank] = page;
      }
    }
    moved = base;
    __syncthreads();
  }
  for (int i = tid; i < moved; i += kPoolThreads) place[source[i]] = target[i];
  if (tid == 0) {
    place[p.N] = used;
    place[p.N + 1] = moved;
  }
}

__global__ __launch_bounds__(256) void pool_compact_kernel(Pool p, int32_t* source, int32_t* target, const int32_t* place,
                                                           int words) {
  const int used = place[p.N], moved = place[p.N + 1];
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t i = i0; i < (int64_t)p.R * p.cols; i += step) {
    const int r = (int)(i / p.cols), c = (int)(i % p.cols);
    if (c >= pages_of(p, rows_of(p, p.lengths[r]))) continue;
    int32_t* entry = p.tables + r * p.t_st + c;
    const int32_t page = *entry;
    if (page >= used && page < p.N) *entry = place[page];
  }
  for (int64_t i = i0; i < moved; i += step) {
    p.refs[target[i]] = p.refs[source[i]];
    p.refs[source[i]] = 0;
  }
  for (int64_t i = moved + i0; i < p.N / 2; i += step) source[i] = target[i] = -1;
  for (int64_t w = i0; w < words; w += step) {
    const int64_t cut = used - 32 * w;
    const uint32_t below = cut >= 32 ? ~0u : cut <= 0 ? 0u : (1u << cut) - 1;
    p.free[w] = ~below & page_bits(p, (int)w);
  }
}

// ---- copies ------------------------------------------------------------------------------------------------------
// Page target[i] of every cache becomes page source[i], in units of 16 bytes (or single ones). A workgroup takes kPiece bytes
// of a page, of `per` list entries one after the other (64 of a list that may be mostly -1: a look at 64 at a time). Bound by
// HBM: 1.5 GB both ways of 4 caches in 314 us, 4.8 TB/s (pieces of 8 KB: 13 us more, of 32 KB 23). Stores go past the caches,
// loads do not: the pages that forks copy have one source in common (256 pages of 16 sources in 8 caches: 13.3 us; with loads
// past the caches 21, with plain stores 16).
constexpr int kMaxCaches = 128;
constexpr int kPiece = 16384;

struct CopyParams {
  uint8_t* caches[kMaxCaches];
  int64_t page_stride, page_bytes, num_pages;
  const int32_t *source, *target;
  int64_t count;
  int per, pieces;
};

template <typename Unit>
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyParams a) {
  constexpr int U = kPiece / sizeof(Unit) / 256;
  const int lane = threadIdx.x & 63;
  uint8_t* cache = a.caches[blockIdx.y];
  const int64_t at = (int64_t)(blockIdx.x % a.pieces) * kPiece;
  const int64_t units = min((int64_t)kPiece, a.page_bytes - at) / (int64_t)sizeof(Unit);
  const int64_t e0 = (int64_t)(blockIdx.x / a.pieces) * a.per;
  int32_t s = -1, d = -1;
  if (lane < a.per && e0 + lane < a.count) {
    s = a.source[e0 + lane];
    d = a.target[e0 + lane];
  }
  const bool valid = s >= 0 && s < a.num_pages && d >= 0 && d < a.num_pages && s != d;
  for (uint64_t left = __ballot(valid); left; left &= left - 1) {
    const int i = __ffsll((unsigned long long)left) - 1;
    const Unit* from = reinterpret_cast<const Unit*>(cache + (int64_t)__shfl(s, i) * a.page_stride + at);
    Unit* to = reinterpret_cast<Unit*>(cache + (int64_t)__shfl(d, i) * a.page_stride + at);
    if constexpr (sizeof(Unit) == 16) {
      Unit v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (threadIdx.x + 256 * u < units) v[u] = from[threadIdx.x + 256 * u];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (threadIdx.x + 256 * u < units) __builtin_nontemporal_store(v[u], to + threadIdx.x + 256 * u);
    } else {
      for (int64_t u = threadIdx.x; u < units; u += 256) to[u] = from[u];
    }
  }
}

int check_pool(const char* what, const int32_t* tables, int64_t t_st, int R, int cols, const int32_t* lengths,
               const int32_t* refs, int64_t N, const void* free, int block) {
  HLA_REQUIRE(R >= 0 && R <= kMaxRequests && cols >= 0 && N >= 0 && N <= INT32_MAX - 64 && block >= 1, HLA_S6_EINVAL,
              "%s: bad request count (0..%d), table width, page count or block size", what, kMaxRequests);
  HLA_REQUIRE(R == 0 || lengths, HLA_S6_EINVAL, "%s: null lengths", what);
  HLA_REQUIRE(R == 0 || cols == 0 || tables, HLA_S6_EINVAL, "%s: null tables", what);
  HLA_REQUIRE(N == 0 || (refs && free), HLA_S6_EINVAL, "%s: null page state", what);
  HLA_REQUIRE(t_st >= cols || R <= 1, HLA_S6_EINVAL, "%s: table rows overlap", what);
  return HLA_S6_OK;
}

}  // namespace
}  // namespace hla

#define HLA_POOL(what)                                                                                       \
  int rc = check_pool(what, tables, t_st, num_reqs, cols, lengths, refs, num_pages, free_bits, block_size);  \
  if (rc != HLA_S6_OK) return rc;                                                                            \
  const Pool p = {tables, t_st, num_reqs, cols, lengths, refs, (int)num_pages, free_bits, block_size}

extern "C" int hla_s6_pool_release(int32_t* tables, int64_t t_st, int32_t num_reqs, int32_t cols, int32_t* lengths,
                                   int32_t* refs, int64_t num_pages, uint32_t* free_bits, int32_t block_size,
                                   const int32_t* requests, const int32_t* to, int32_t count, void* stream) {
  using namespace hla;
  HLA_POOL("pool_release");
  HLA_REQUIRE(count >= 0 && (count == 0 || requests), HLA_S6_EINVAL, "pool_release: bad list");
  HLA_REQUIRE(launchable(count, 256), HLA_S6_EINVAL, "pool_release: list too long");
  if (count == 0 || num_reqs == 0) return HLA_S6_OK;
  hipLaunchKernelGGL(pool_release_kernel, dim3((unsigned)count), dim3(256), 0, as_stream(stream), p, requests, to);
  return check_launch("pool_release");
}

extern "C" int hla_s6_pool_fork(int32_t* tables, int64_t t_st, int32_t num_reqs, int32_t cols, int32_t* lengths,
                                int32_t* refs, int64_t num_pages, uint32_t* free_bits, int32_t block_size,
                                const int32_t* parents, const int32_t* children, int32_t count, uint8_t* ok, void* stream) {
  using namespace hla;
  HLA_POOL("pool_fork");
  HLA_REQUIRE(count >= 0 && count <= kMaxRequests && (count == 0 || (parents && children && ok)), HLA_S6_EINVAL,
              "pool_fork: bad lists (at most %d entries)", kMaxRequests);
  if (count == 0) return HLA_S6_OK;
  hipLaunchKernelGGL(pool_fork_kernel, dim3((unsigned)count), dim3(256), 0, as_stream(stream), p, parents, children, count, ok);
  return check_launch("pool_fork");
}

extern "C" int hla_s6_pool_extend(int32_t* tables, int64_t t_st, int32_t num_reqs, int32_t cols, int32_t* lengths,
                                  int32_t* refs, int64_t num_pages, uint32_t* free_bits, int32_t block_size,
                                  const int32_t* to, const int32_t* from, uint8_t* ok, int32_t* source, int32_t* target,
                                  int32_t* scratch, void* stream) {
  using namespace hla;
  HLA_POOL("pool_extend");
  if (num_reqs == 0) return HLA_S6_OK;
  HLA_REQUIRE(to && ok && ((source && target) || (from && cols == 0)) && (!from || scratch), HLA_S6_EINVAL,
              "pool_extend: null pointer argument");
  HLA_REQUIRE(!from || (int64_t)num_reqs * cols <= INT32_MAX, HLA_S6_EINVAL, "pool_extend: too many table entries");
  const hipStream_t st = as_stream(stream);
  const ExtendParams a = {p, to, from, ok, source, target, scratch, from ? scratch + (int64_t)num_reqs * cols : nullptr};
  if (from) {
    hipLaunchKernelGGL(pool_need_kernel, dim3((unsigned)num_reqs), dim3(256), 0, st, a);
    hipLaunchKernelGGL(pool_plan_kernel, dim3(1), dim3(kPoolThreads), 0, st, a);
    hipLaunchKernelGGL(pool_fill_kernel, dim3((unsigned)num_reqs), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL(pool_extend_kernel, dim3(1), dim3(kPoolThreads), 0, st, a);
  }
  return check_launch("pool_extend");
}

extern "C" int hla_s6_pool_compact(int32_t* tables, int64_t t_st, int32_t num_reqs, int32_t cols, int32_t* lengths,
                                   int32_t* refs, int64_t num_pages, uint32_t* free_bits, int32_t block_size,
                                   int32_t* source, int32_t* target, int32_t* scratch, void* stream) {
  using namespace hla;
  HLA_POOL("pool_compact");
  if (num_pages == 0) return HLA_S6_OK;
  HLA_REQUIRE(scratch && (num_pages < 2 || (source && target)), HLA_S6_EINVAL, "pool_compact: null pointer argument");
  const hipStream_t st = as_stream(stream);
  hipLaunchKernelGGL(pool_pairs_kernel, dim3(1), dim3(kPoolThreads), 0, st, p, source, target, scratch);
  const int words = (int)((num_pages + 31) / 32);
  const int64_t most = (int64_t)num_reqs * cols > num_pages ? (int64_t)num_reqs * cols : num_pages;
  const unsigned grid = (unsigned)((most + 1023) / 1024 < 1024 ? (most + 1023) / 1024 : 1024);
  hipLaunchKernelGGL(pool_compact_kernel, dim3(grid), dim3(256), 0, st, p, source, target, scratch, words);
  return check_launch("pool_compact");
}

extern "C" int hla_s6_copy_pages(void* const* caches, int32_t num_caches, int64_t page_stride, int64_t page_bytes,
                                 int64_t num_pages, const int32_t* source, const int32_t* target, int64_t count,
                                 void* stream) {
  using namespace hla;
  HLA_REQUIRE(num_caches >= 0 && page_bytes >= 0 && num_pages >= 0 && count >= 0, HLA_S6_EINVAL, "copy_pages: negative size");
  HLA_REQUIRE(page_stride >= page_bytes || num_pages <= 1, HLA_S6_EINVAL, "copy_pages: pages overlap");
  if (num_caches == 0 || page_bytes == 0 || count == 0 || num_pages == 0) return HLA_S6_OK;
  HLA_REQUIRE(caches && source && target, HLA_S6_EINVAL, "copy_pages: null pointer argument");
  const hipStream_t st = as_stream(stream);
  CopyParams a = {};
  a.page_stride = page_stride;
  a.page_bytes = page_bytes;
  a.num_pages = num_pages;
  a.source = source;
  a.target = target;
  a.count = count;
  const int64_t pieces = (page_bytes - 1) / kPiece + 1;
  a.per = count > 4096 ? 64 : 1;
  const int64_t groups = (count - 1) / a.per + 1;
  HLA_REQUIRE(pieces <= INT32_MAX && groups <= INT32_MAX && launchable(groups * pieces, 256), HLA_S6_EINVAL,
              "copy_pages: lists or pages too long");
  a.pieces = (int)pieces;
  for (int c0 = 0; c0 < num_caches; c0 += kMaxCaches) {
    const int n = num_caches - c0 < kMaxCaches ? num_caches - c0 : kMaxCaches;
    bool vec = page_stride % 16 == 0 && page_bytes % 16 == 0;
    for (int c = 0; c < n; ++c) {
      HLA_REQUIRE(caches[c0 + c], HLA_S6_EINVAL, "copy_pages: null cache");
      a.caches[c] = static_cast<uint8_t*>(caches[c0 + c]);
      vec = vec && (reinterpret_cast<uintptr_t>(caches[c0 + c]) & 15u) == 0;
    }
    const dim3 grid((unsigned)(groups * pieces), (unsigned)n);
    if (vec) hipLaunchKernelGGL(copy_pages_kernel<u32x4>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(copy_pages_kernel<uint8_t>, grid, dim3(256), 0, st, a);
  }
  return check_launch("copy_pages");
}
