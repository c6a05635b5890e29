// The pages of a paged cache: who holds them (extend, free, fork, compact) and their contents (copy, fork,
// compact). All state is on the device and nothing is read back, so a step can be captured.
//
// Measured: 201 pages of 32 KB in 16 caches copied in 37 us (5.7 TB/s read and written, 0.87 of the copy rate; 32.6 alone, behind a
// flushed L2); half a gigabyte moved by a compaction in 86 and its plan in 4; a step that frees 32 rows, extends 16 and forks 16
// in 14, which is the host's time for the three calls.
//
// The bookkeeping is a few thousand integers and bound by latency: one CTA of 1024 threads plans a request
// (requests that name a row twice, a prefix sum of the pages that they need, the lowest free pages by a
// prefix sum over the reference counts up to the last one needed), the order of every result is that of the
// request and not of the atomics. The contents are bound by HBM: a warp copies pieces of 4 KB, eight 16-byte
// loads in flight per lane, all caches of all layers in one launch.
//
// Every kernel may be scheduled while the one before it on the stream still runs, and waits for its end before it
// touches anything: its launch is hidden. What it reads may have been written during its own life, so that no
// load here is of the read-only kind.
#include <algorithm>
#include <climits>

#include "common.cuh"

namespace {

constexpr int PLAN = 1024;                 // threads of a planning CTA
constexpr int PER = 16;                    // reference counts per thread and step
constexpr int COPY_WARPS = 8, COPY_CTAS = 16;   // and CTAs for an SM, three of them at a time
constexpr int PIECE = 4096;                // bytes of a warp's piece
constexpr int MAX_CACHES = 64;             // per launch
constexpr int TILE = 4096;                 // pages per CTA of a compaction's plan

// Inclusive prefix sum over the CTA; `total` is the sum. s: 33 values of shared memory.
template <class T>
__device__ __forceinline__ T block_scan(T x, T* s, T& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const T up = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += up;
  }
  __syncthreads();                         // the last scan's values have been read
  if (lane == 31) s[w] = x;
  __syncthreads();
  if (w == 0) {
    T y = lane < warps ? s[lane] : T(0);
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const T up = __shfl_up_sync(0xffffffffu, y, off);
      if (lane >= off) y += up;
    }
    s[lane] = y;
  }
  __syncthreads();
  total = s[warps - 1];
  return w ? x + s[w - 1] : x;
}

// A set of integers >= 0 in shared memory, with the lowest index that came with each: open addressing, at most
// half full.
template <int SIZE>
struct SmallMap {
  int key[SIZE], least[SIZE];
  __device__ void clear() {                // by the whole CTA, a barrier behind it
    for (int i = threadIdx.x; i < SIZE; i += blockDim.x) key[i] = -1, least[i] = INT_MAX;
    __syncthreads();
  }
  static constexpr int BITS = 11;
  static_assert(SIZE == 1 << BITS, "the top bits of a product are the place");
  static __device__ __forceinline__ unsigned place(int k) { return ((unsigned)k * 2654435761u) >> (32 - BITS); }
  __device__ bool add(int k, int index) {  // false: it was there
    for (unsigned at = place(k);; ++at) {
      const int old = atomicCAS(&key[at % SIZE], -1, k);
      if (old != -1 && old != k) continue;
      atomicMin(&least[at % SIZE], index);
      return old == -1;
    }
  }
  __device__ int find(int k) const {       // its lowest index, -1: not there. Behind a barrier.
    for (unsigned at = place(k);; ++at) {
      if (key[at % SIZE] == k) return least[at % SIZE];
      if (key[at % SIZE] == -1) return -1;
    }
  }
};
constexpr int MAP = 2 * PLAN;              // for lists of up to PLAN entries

// The first entry of a list that names `row` gets it: shared memory for a list that fits, claim[num_rows] (with any
// values before) for others. Called by the whole CTA; then mine(i, row) says whether entry i does.
struct Claims {
  SmallMap<MAP>& map;
  int32_t* claim;
  bool small;
  __device__ Claims(SmallMap<MAP>& m, const int32_t* list, int n, int rows, int32_t* c) : map(m), claim(c), small(n <= PLAN) {
    if (small) {
      const int i = threadIdx.x, row = i < n ? list[i] : -1;
      map.clear();
      if ((unsigned)row < (unsigned)rows) map.add(row, i);
      __syncthreads();
      return;
    }
    for (int i = threadIdx.x; i < n; i += blockDim.x)
      if ((unsigned)list[i] < (unsigned)rows) claim[list[i]] = i;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x)
      if ((unsigned)list[i] < (unsigned)rows) atomicMin(claim + list[i], i);
    __syncthreads();
  }
  __device__ __forceinline__ bool mine(int i, int row) const { return (small ? map.find(row) : claim[row]) == i; }
};

// The lowest free pages, in ascending order: the first NEAR of them in shared memory, the others in far[].
constexpr int NEAR = 2048;
struct Fresh {
  int* near;
  int32_t* far;
  __device__ __forceinline__ int operator[](int i) const { return i < NEAR ? near[i] : far[i]; }
  __device__ __forceinline__ void set(int i, int page) const { (i < NEAR ? near : far)[i] = page; }
};
// Which of a thread's PER pages from p0 on are free.
__device__ __forceinline__ unsigned free_of(const int32_t* refs, int pages, int p0) {
  unsigned mask = 0;
  if (p0 + PER <= pages && ((uintptr_t)refs & 15) == 0) {
#pragma unroll
    for (int j = 0; j < PER; j += 4) {
      const int4 r = *reinterpret_cast<const int4*>(refs + p0 + j);
      mask |= ((r.x == 0) | (r.y == 0) << 1 | (r.z == 0) << 2 | (r.w == 0) << 3) << j;
    }
    return mask;
  }
  for (int j = 0; j < PER && p0 + j < pages; ++j) mask |= (refs[p0 + j] == 0) << j;
  return mask;
}
// Finds the first `wanted` free pages and returns how many there are, at most `wanted`. `mask`: free_of() of the
// first step, asked for before so that it is there by now. Called by the whole CTA.
__device__ int lowest_free(const int32_t* refs, int pages, int wanted, unsigned mask, const Fresh& fresh, int* s_scan) {
  int found = 0;
  for (int base = 0; base < pages && found < wanted; base += PLAN * PER) {
    const int p0 = base + threadIdx.x * PER;
    if (base) mask = free_of(refs, pages, p0);
    int total;
    int at = found + block_scan(__popc(mask), s_scan, total) - __popc(mask);
    for (; mask && at < wanted; mask &= mask - 1, ++at) fresh.set(at, p0 + __ffs(mask) - 1);
    found += total;
  }
  __syncthreads();                         // fresh is complete
  return min(found, wanted);
}

__device__ __forceinline__ int pages_of(int64_t tokens, int page_size) { return (int)((tokens + page_size - 1) / page_size); }

struct Grow {
  int32_t* table;
  int32_t* lens;
  int32_t* refs;
  const int32_t* rows;
  const int32_t* add;
  uint8_t* ok;
  int32_t* claim;    // [num_rows]
  int4* request;     // [n] row, length before, length after, pages set aside before it or -1: it is not valid
  int32_t* fresh;    // [num_pages]
  int n, num_rows, max_pages, num_pages, page_size;
};

__global__ void __launch_bounds__(PLAN) extend_kernel(const Grow g) {
  __shared__ int s_scan[33];
  __shared__ long long s_scan64[33];
  __shared__ SmallMap<MAP> s_map;
  __shared__ int s_near[NEAR];
  __shared__ int4 s_request[PLAN];
  ako::pdl_trigger();
  ako::pdl_wait();
  const unsigned mask = free_of(g.refs, g.num_pages, threadIdx.x * PER);
  const Claims claims(s_map, g.rows, g.n, g.num_rows, g.claim);
  const Fresh fresh = {s_near, g.fresh};
  int4* requests = g.n <= PLAN ? s_request : g.request;
  long long taken = 0;
  for (int base = 0; base < g.n; base += PLAN) {
    const int i = base + threadIdx.x;
    long long need = 0;
    int4 r = make_int4(0, 0, 0, -1);
    if (i < g.n) {
      const int row = g.rows[i], add = g.add[i];
      if ((unsigned)row < (unsigned)g.num_rows && add >= 0 && claims.mine(i, row)) {
        const int64_t len = max(0, g.lens[row]), now = len + add;
        if (now <= (int64_t)g.max_pages * g.page_size && now <= INT_MAX) {
          need = pages_of(now, g.page_size) - pages_of(len, g.page_size);
          r = make_int4(row, (int)len, (int)now, 0);
        }
      }
    }
    long long total;
    const long long before = taken + block_scan(need, s_scan64, total) - need;
    if (r.w == 0) r.w = (int)min(before, (long long)INT_MAX);
    if (i < g.n) requests[i] = r;
    taken += total;
  }
  const int have = lowest_free(g.refs, g.num_pages, (int)min(taken, (long long)g.num_pages), mask, fresh, s_scan);
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < g.n; i += PLAN / 32) {   // a warp per request
    const int4 r = requests[i];
    const int held = pages_of(r.y, g.page_size), need = pages_of(r.z, g.page_size) - held;
    const bool ok = r.w >= 0 && (need == 0 || (int64_t)r.w + need <= have);
    if (ok) {
      for (int j = lane; j < need; j += 32) {
        const int page = fresh[r.w + j];
        g.table[(int64_t)r.x * g.max_pages + held + j] = page;
        g.refs[page] = 1;
      }
      if (lane == 0) g.lens[r.x] = r.z;
    }
    if (lane == 0) g.ok[i] = ok;
  }
}

// A warp per row. The exchange gives a row that is listed twice to one of the two; which one makes no difference.
__global__ void __launch_bounds__(256) free_kernel(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* rows, int n,
                                                   int num_rows, int max_pages, int num_pages, int page_size) {
  ako::pdl_trigger();
  ako::pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (i >= n) return;
  const int row = rows[i];
  if ((unsigned)row >= (unsigned)num_rows) return;
  int len = 0;
  if (lane == 0) len = atomicExch(lens + row, 0);
  len = __shfl_sync(0xffffffffu, len, 0);
  if (len <= 0) return;
  const int held = min(pages_of(len, page_size), max_pages);
  int32_t* mine = table + (int64_t)row * max_pages;
  for (int j = lane; j < held; j += 32) {
    const int page = mine[j];
    if ((unsigned)page < (unsigned)num_pages) atomicSub(refs + page, 1);
    mine[j] = -1;
  }
}

// ---- contents -----------------------------------------------------------------------------------

struct Caches {
  unsigned char* data[MAX_CACHES];
  int64_t stride[MAX_CACHES], bytes[MAX_CACHES];
  int32_t first_piece[MAX_CACHES + 1];     // pieces of a page in the caches before
  uint8_t width[MAX_CACHES];               // bytes per access: 16, 4 or 1
  int count;
};

template <class V>
__device__ __forceinline__ void copy_piece(const unsigned char* from, unsigned char* to, int bytes, int lane) {
  const V* f = reinterpret_cast<const V*>(from);
  V* t = reinterpret_cast<V*>(to);
  const int n = bytes / (int)sizeof(V);
  constexpr int U = 8;
  for (int i = lane; i < n; i += 32 * U) {
    V x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + 32 * u < n) x[u] = __ldcs(f + i + 32 * u);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + 32 * u < n) __stcs(t + i + 32 * u, x[u]);
  }
}

// One piece of one page.
__device__ __forceinline__ void copy_unit(const Caches& c, int src, int dst, int piece, int lane) {
  int lo = 0, hi = c.count;                // the cache: first_piece[lo] <= piece < first_piece[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c.first_piece[mid] <= piece) lo = mid;
    else hi = mid;
  }
  const int64_t at = (int64_t)(piece - c.first_piece[lo]) * PIECE;
  const int bytes = (int)min((int64_t)PIECE, c.bytes[lo] - at);
  const unsigned char* from = c.data[lo] + src * c.stride[lo] + at;
  unsigned char* to = c.data[lo] + dst * c.stride[lo] + at;
  if (c.width[lo] == 16) copy_piece<uint4>(from, to, bytes, lane);
  else if (c.width[lo] == 4) copy_piece<uint32_t>(from, to, bytes, lane);
  else copy_piece<uint8_t>(from, to, bytes, lane);
}

__device__ __forceinline__ int quotient(int64_t u, unsigned by) {   // in 32 bits where that will do
    return u <= 0xffffffffLL ? (int)((unsigned)u / by) : (int)(u / by);
}
struct Warps {
  int lane;
  int64_t first, step;
};
__device__ __forceinline__ Warps grid_warps() {
  return {(int)(threadIdx.x & 31), (int64_t)blockIdx.x * COPY_WARPS + (threadIdx.x >> 5), (int64_t)gridDim.x * COPY_WARPS};
}

// owner[page] for the pages of the list: an index of a pair that has it as its destination. What owner[] holds for
// others is not known, so an entry counts only if the pair that it names says so too.
__device__ __forceinline__ bool pair_counts(int s, int d, int pages) {
  return s != d && (unsigned)s < (unsigned)pages && (unsigned)d < (unsigned)pages;
}
__global__ void __launch_bounds__(PLAN) copy_plan_kernel(const int32_t* src, const int32_t* dst, int n, int pages, int32_t* owner,
                                                         uint8_t* ok, int32_t* go) {
  ako::pdl_trigger();
  ako::pdl_wait();
  for (int i = threadIdx.x; i < n; i += PLAN)
    if (pair_counts(src[i], dst[i], pages)) owner[dst[i]] = i;
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += PLAN) {
    const int s = src[i], d = dst[i];
    if (!pair_counts(s, d, pages)) continue;
    bad |= owner[d] != i;
    const int o = owner[s];
    bad |= (unsigned)o < (unsigned)n && dst[o] == s && pair_counts(src[o], s, pages);
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) {
    *ok = !bad;
    *go = !bad;
  }
}
__global__ void __launch_bounds__(COPY_WARPS * 32, 3) copy_kernel(const Caches c, const int32_t* src, const int32_t* dst, int n, int pages,
                                                               const int32_t* go) {
  ako::pdl_wait();
  if (!*go) return;
  const Warps w = grid_warps();
  const int pieces = c.first_piece[c.count];
  for (int64_t u = w.first; u < (int64_t)n * pieces; u += w.step) {
    const int i = quotient(u, pieces);
    if (pair_counts(src[i], dst[i], pages)) copy_unit(c, src[i], dst[i], (int)(u - (int64_t)i * pieces), w.lane);
  }
}

// Lists of up to PAIRS pairs: every CTA checks the list for itself, in shared memory, instead of a launch before (200 pages of
// four caches of 2 KB 4.0 -> 3.4 us; 600 pages 4.9 -> 6.3, 1 000 6.2 -> 16).
constexpr int PAIRS = 256;
__global__ void __launch_bounds__(COPY_WARPS * 32, 3) copy_short_kernel(const Caches c, const int32_t* src, const int32_t* dst, int n, int pages,
                                                                     uint8_t* ok) {
  __shared__ SmallMap<8 * PAIRS> s_map;
  __shared__ int2 s_pair[PAIRS];
  ako::pdl_trigger();
  ako::pdl_wait();
  for (int i = threadIdx.x; i < n; i += COPY_WARPS * 32) s_pair[i] = make_int2(src[i], dst[i]);
  s_map.clear();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += COPY_WARPS * 32)
    if (pair_counts(s_pair[i].x, s_pair[i].y, pages)) bad |= !s_map.add(s_pair[i].y, i);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += COPY_WARPS * 32)
    if (pair_counts(s_pair[i].x, s_pair[i].y, pages)) bad |= s_map.find(s_pair[i].x) >= 0;
  bad = __syncthreads_or(bad);
  if (blockIdx.x == 0 && threadIdx.x == 0) *ok = !bad;
  if (bad) return;
  const Warps w = grid_warps();
  const unsigned pieces = c.first_piece[c.count];
  for (int64_t u = w.first; u < (int64_t)n * pieces; u += w.step) {
    const int i = quotient(u, pieces);
    const int2 p = s_pair[i];
    if (pair_counts(p.x, p.y, pages)) copy_unit(c, p.x, p.y, (int)(u - (int64_t)i * pieces), w.lane);
  }
}

struct Fork {
  int32_t* table;
  int32_t* lens;
  int32_t* refs;
  const int32_t* parents;
  const int32_t* children;
  uint8_t* ok;
  int32_t* claim;    // [num_rows]
  int2* plan;        // [n]: {pages set aside before; then the fresh page or -1, length or -1 where not ok}
  int32_t* fresh;    // [num_pages]
  int n, num_rows, max_pages, num_pages, page_size;
};

__global__ void __launch_bounds__(PLAN) fork_plan_kernel(const Fork f) {
  __shared__ int s_scan[33];
  __shared__ SmallMap<MAP> s_map;
  __shared__ int s_near[NEAR];
  __shared__ int2 s_plan[PLAN];
  ako::pdl_trigger();
  ako::pdl_wait();
  int2* plan = f.n <= PLAN ? s_plan : f.plan;
  const unsigned mask = free_of(f.refs, f.num_pages, threadIdx.x * PER);
  const Claims claims(s_map, f.children, f.n, f.num_rows, f.claim);
  const Fresh fresh = {s_near, f.fresh};
  int taken = 0;
  for (int base = 0; base < f.n; base += PLAN) {
    const int i = base + threadIdx.x;
    int need = 0, len = -1;
    if (i < f.n) {
      const int parent = f.parents[i], child = f.children[i];
      if ((unsigned)parent < (unsigned)f.num_rows && (unsigned)child < (unsigned)f.num_rows && claims.mine(i, child) && f.lens[child] == 0) {
        len = max(0, f.lens[parent]);
        if (len > (int64_t)f.max_pages * f.page_size) len = -1;
        else need = len % f.page_size != 0;
      }
    }
    int total;
    const int before = taken + block_scan(need, s_scan, total) - need;
    if (i < f.n) plan[i] = make_int2(need ? before : -1, len);
    taken += total;
  }
  // all lengths have been read before the first one is written: the scans below are barriers, and so is this
  const int have = lowest_free(f.refs, f.num_pages, min(taken, f.num_pages), mask, fresh, s_scan);
  for (int i = threadIdx.x; i < f.n; i += PLAN) {
    int2 p = plan[i];
    const bool ok = p.y >= 0 && p.x < have;   // p.x = -1: no page needed
    if (ok) {
      if (p.x >= 0) {
        p.x = fresh[p.x];
        f.refs[p.x] = 1;
      }
      f.lens[f.children[i]] = p.y;
    } else {
      p = make_int2(-1, -1);
    }
    f.plan[i] = p;
    f.ok[i] = ok;
  }
}
// Units: a row of the table per warp (in the first launch of a call), then the pieces of the copied pages.
__global__ void __launch_bounds__(COPY_WARPS * 32, 3) fork_kernel(const Caches c, const Fork f, bool rows) {
  ako::pdl_trigger();
  ako::pdl_wait();
  const Warps w = grid_warps();
  const int pieces = c.first_piece[c.count], row_units = rows ? f.n : 0;
  for (int64_t u = w.first; u < row_units + (int64_t)f.n * pieces; u += w.step) {
    const bool row = u < row_units;
    const int i = row ? (int)u : quotient(u - row_units, pieces);
    const int2 p = f.plan[i];
    if (p.y < 0) continue;
    const int32_t* from = f.table + (int64_t)f.parents[i] * f.max_pages;
    const int full = p.y / f.page_size;
    if (row) {
      int32_t* to = f.table + (int64_t)f.children[i] * f.max_pages;
      for (int j = w.lane; j < full; j += 32) {
        const int page = from[j];
        to[j] = page;
        if ((unsigned)page < (unsigned)f.num_pages) atomicAdd(f.refs + page, 1);
      }
      if (w.lane == 0 && p.x >= 0) to[full] = p.x;
    } else if (p.x >= 0) {
      const int page = from[full];
      if ((unsigned)page < (unsigned)f.num_pages)
        copy_unit(c, page, p.x, (int)(u - row_units - (int64_t)i * pieces), w.lane);
    }
  }
}

// ---- compaction ---------------------------------------------------------------------------------

// used[] before each tile of pages, and all of them behind the last one
__global__ void __launch_bounds__(PLAN) compact_count_kernel(const int32_t* refs, int pages, int32_t* counts) {
  ako::pdl_trigger();
  ako::pdl_wait();
  const int p0 = blockIdx.x * TILE + threadIdx.x * (TILE / PLAN);
  int used = 0;
#pragma unroll
  for (int j = 0; j < TILE / PLAN; ++j) used += p0 + j < pages && refs[p0 + j] > 0;
  __shared__ int s_scan[33];
  int total;
  block_scan(used, s_scan, total);
  if (threadIdx.x == 0) counts[blockIdx.x] = total;
}
// With u pages in use and U(p) of them in front of p: page p >= u in use is the (u - 1 - U(p))-th from the top, place
// p < u that is free the (p - U(p))-th from the bottom, and they meet. code[p]: the place of a page that stays, -2 -
// its number of a page that moves, -1 of a free one.
__global__ void __launch_bounds__(PLAN) compact_plan_kernel(const int32_t* refs, int pages, const int32_t* counts, int tiles,
                                                            int32_t* code, int32_t* src, int32_t* dst, int32_t* moves) {
  __shared__ int s_scan[33];
  ako::pdl_trigger();
  ako::pdl_wait();
  const int p0 = blockIdx.x * TILE + threadIdx.x * (TILE / PLAN);
  int used[TILE / PLAN], mine = 0;
#pragma unroll
  for (int j = 0; j < TILE / PLAN; ++j) {
    used[j] = p0 + j < pages && refs[p0 + j] > 0;
    mine += used[j];
  }
  int total;
  int at = block_scan(mine, s_scan, total) - mine, all = total;
  if (tiles > 1) {                         // with one tile there was no count
    int before = 0, u = 0, front;
    for (int t = threadIdx.x; t < tiles; t += PLAN) {
      u += counts[t];
      if (t < (int)blockIdx.x) before += counts[t];
    }
    block_scan(u, s_scan, all);
    block_scan(before, s_scan, front);
    at += front;
  }
  if (all == pages && blockIdx.x == 0 && threadIdx.x == 0) *moves = 0;
#pragma unroll
  for (int j = 0; j < TILE / PLAN; ++j) {
    const int p = p0 + j;
    if (p < pages) {
      if (p == all) *moves = all - at;     // the places in front that are free
      int c = -1;
      if (used[j]) {
        c = p < all ? p : -2 - (all - 1 - at);
        if (p >= all) src[all - 1 - at] = p;
      } else if (p < all) {
        dst[p - at] = p;
      }
      code[p] = c;
    }
    at += used[j];
  }
}

struct Compact {
  int32_t* table;
  int32_t* refs;
  int32_t* page_map;
  const int32_t* code;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* moves;
  int64_t entries;   // of the table
  int pages;
};
__global__ void __launch_bounds__(COPY_WARPS * 32, 3) compact_kernel(const Caches c, const Compact k, bool tables) {
  ako::pdl_trigger();
  ako::pdl_wait();
  const Warps w = grid_warps();
  const int pieces = c.first_piece[c.count], moves = *k.moves;
  if (tables) {
    const int64_t threads = (int64_t)gridDim.x * blockDim.x, me = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (int64_t i = me; i < k.pages; i += threads) {
      const int x = k.code[i];
      k.page_map[i] = x < -1 ? k.dst[-2 - x] : x;
    }
    for (int64_t i = me; i < k.entries; i += threads) {
      const int page = k.table[i];
      if ((unsigned)page >= (unsigned)k.pages) continue;
      const int x = k.code[page];
      if (x < -1) k.table[i] = k.dst[-2 - x];
    }
    for (int64_t i = me; i < moves; i += threads) {
      k.refs[k.dst[i]] = k.refs[k.src[i]];
      k.refs[k.src[i]] = 0;
    }
  }
  for (int64_t u = w.first; u < (int64_t)moves * pieces; u += w.step) {
    const int i = quotient(u, pieces);
    copy_unit(c, k.src[i], k.dst[i], (int)(u - (int64_t)i * pieces), w.lane);
  }
}

// ---- host ---------------------------------------------------------------------------------------

bool counts_ok(int64_t n, int64_t num_rows, int64_t max_pages, int64_t num_pages, int64_t page_size) {
  const int64_t most = 0x7fffffffLL - 65536;   // loops step past their end by a CTA's work at most
  return n >= 0 && n <= most && num_rows >= 0 && num_rows <= most && max_pages >= 0 && max_pages <= most && num_pages >= 0 &&
         num_pages <= most && page_size >= 1 && page_size <= most;
}
bool int_ptr(const void* p) { return p && ((uintptr_t)p & 3) == 0; }

// The caches of one launch; false where they are not usable.
bool take(Caches& c, void* const* data, const int64_t* bytes, const int64_t* strides, int64_t from, int64_t to) {
  c.count = (int)(to - from);
  int64_t pieces = 0;
  for (int64_t i = from; i < to; ++i) {
    const int k = (int)(i - from);
    if (!data[i] || bytes[i] <= 0 || strides[i] < bytes[i]) return false;
    c.data[k] = (unsigned char*)data[i];
    c.bytes[k] = bytes[i];
    c.stride[k] = strides[i];
    const uint64_t all = (uintptr_t)data[i] | (uint64_t)bytes[i] | (uint64_t)strides[i];
    c.width[k] = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    c.first_piece[k] = (int32_t)pieces;
    pieces += ako::cdiv(bytes[i], (int64_t)PIECE);
    if (pieces > 0x7fffffffLL) return false;
  }
  c.first_piece[c.count] = (int32_t)pieces;
  return true;
}
bool caches_ok(void* const* data, const int64_t* bytes, const int64_t* strides, int64_t n) {
  if (n < 0 || (n > 0 && (!data || !bytes || !strides))) return false;
  Caches c;
  for (int64_t at = 0; at < n; at += MAX_CACHES)
    if (!take(c, data, bytes, strides, at, std::min(n, at + MAX_CACHES))) return false;
  return true;
}
// Calls launch(caches, whether it is the first) for every MAX_CACHES caches, once at least.
template <class F>
int for_caches(void* const* data, const int64_t* bytes, const int64_t* strides, int64_t n, F launch) {
  for (int64_t at = 0; at == 0 || at < n; at += MAX_CACHES) {
    Caches c = {};
    take(c, data, bytes, strides, at, std::min(n, at + MAX_CACHES));
    if (launch(c, at == 0) != cudaSuccess) return AKO4X_ELAUNCH;
  }
  return AKO4X_OK;
}
unsigned copy_grid(int64_t units) {
  const int64_t most = (int64_t)ako::sm_count() * COPY_CTAS;
  return (unsigned)std::max<int64_t>(1, std::min(most, ako::cdiv(units, (int64_t)COPY_WARPS)));
}

size_t up(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace

extern "C" size_t ako4x_kv_pages_extend_workspace_bytes(int64_t n, int64_t num_rows, int64_t num_pages) {
  if (n <= 0 || num_rows < 0 || num_pages < 0) return 0;
  return up(4 * num_rows) + up(16 * n) + up(4 * num_pages);
}

extern "C" int ako4x_kv_pages_extend(int32_t* block_table, int32_t* seq_lens, int32_t* ref_counts, const int32_t* rows,
                                     const int32_t* add, uint8_t* ok, int64_t n, int64_t num_rows, int64_t max_pages,
                                     int64_t num_pages, int64_t page_size, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (!counts_ok(n, num_rows, max_pages, num_pages, page_size)) return AKO4X_EINVAL;
  if (n == 0) return AKO4X_OK;
  if (!int_ptr(rows) || !int_ptr(add) || !ok) return AKO4X_EINVAL;
  if (num_rows > 0 && (!int_ptr(seq_lens) || (max_pages > 0 && !int_ptr(block_table)))) return AKO4X_EINVAL;
  if (num_pages > 0 && !int_ptr(ref_counts)) return AKO4X_EINVAL;
  if (!workspace || workspace_bytes < ako4x_kv_pages_extend_workspace_bytes(n, num_rows, num_pages)) return AKO4X_EWORKSPACE;
  if ((uintptr_t)workspace & 15) return AKO4X_EINVAL;
  unsigned char* ws = (unsigned char*)workspace;
  Grow g = {block_table, seq_lens, ref_counts, rows, add, ok, (int32_t*)ws, (int4*)(ws + up(4 * num_rows)),
            (int32_t*)(ws + up(4 * num_rows) + up(16 * n)), (int)n, (int)num_rows, (int)max_pages, (int)num_pages, (int)page_size};
  return ako::launch_pdl(true, extend_kernel, dim3(1), dim3(PLAN), 0, (cudaStream_t)stream, g) == cudaSuccess ? AKO4X_OK : AKO4X_ELAUNCH;
}

extern "C" int ako4x_kv_pages_free(int32_t* block_table, int32_t* seq_lens, int32_t* ref_counts, const int32_t* rows, int64_t n,
                                   int64_t num_rows, int64_t max_pages, int64_t num_pages, int64_t page_size, void* stream) {
  if (!counts_ok(n, num_rows, max_pages, num_pages, page_size)) return AKO4X_EINVAL;
  if (n == 0 || num_rows == 0) return AKO4X_OK;
  if (!int_ptr(rows) || !int_ptr(seq_lens) || (max_pages > 0 && !int_ptr(block_table)) || (num_pages > 0 && !int_ptr(ref_counts)))
    return AKO4X_EINVAL;
  return ako::launch_pdl(true, free_kernel, dim3((unsigned)ako::cdiv(n, (int64_t)8)), dim3(256), 0, (cudaStream_t)stream, block_table, seq_lens,
                         ref_counts, rows, (int)n, (int)num_rows, (int)max_pages, (int)num_pages, (int)page_size) == cudaSuccess
             ? AKO4X_OK
             : AKO4X_ELAUNCH;
}

extern "C" size_t ako4x_kv_pages_fork_workspace_bytes(int64_t n, int64_t num_rows, int64_t num_pages) {
  if (n <= 0 || num_rows < 0 || num_pages < 0) return 0;
  return up(4 * num_rows) + up(8 * n) + up(4 * num_pages);
}

extern "C" int ako4x_kv_pages_fork(void* const* caches, const int64_t* page_bytes, const int64_t* page_strides, int64_t num_caches,
                                   int32_t* block_table, int32_t* seq_lens, int32_t* ref_counts, const int32_t* parents,
                                   const int32_t* children, uint8_t* ok, int64_t n, int64_t num_rows, int64_t max_pages,
                                   int64_t num_pages, int64_t page_size, void* workspace, size_t workspace_bytes, void* stream) {
  if (!counts_ok(n, num_rows, max_pages, num_pages, page_size)) return AKO4X_EINVAL;
  if (!caches_ok(caches, page_bytes, page_strides, num_caches)) return AKO4X_EINVAL;
  if (n == 0) return AKO4X_OK;
  if (!int_ptr(parents) || !int_ptr(children) || !ok) return AKO4X_EINVAL;
  if (num_rows > 0 && (!int_ptr(seq_lens) || (max_pages > 0 && !int_ptr(block_table)))) return AKO4X_EINVAL;
  if (num_pages > 0 && !int_ptr(ref_counts)) return AKO4X_EINVAL;
  if (!workspace || workspace_bytes < ako4x_kv_pages_fork_workspace_bytes(n, num_rows, num_pages)) return AKO4X_EWORKSPACE;
  if ((uintptr_t)workspace & 15) return AKO4X_EINVAL;
  unsigned char* ws = (unsigned char*)workspace;
  cudaStream_t st = (cudaStream_t)stream;
  Fork f = {block_table, seq_lens, ref_counts, parents, children, ok, (int32_t*)ws, (int2*)(ws + up(4 * num_rows)),
            (int32_t*)(ws + up(4 * num_rows) + up(8 * n)), (int)n, (int)num_rows, (int)max_pages, (int)num_pages, (int)page_size};
  if (ako::launch_pdl(true, fork_plan_kernel, dim3(1), dim3(PLAN), 0, st, f) != cudaSuccess) return AKO4X_ELAUNCH;
  return for_caches(caches, page_bytes, page_strides, num_caches, [&](const Caches& c, bool first) {
    const int64_t units = (first ? n : 0) + n * c.first_piece[c.count];
    return ako::launch_pdl(first, fork_kernel, dim3(copy_grid(units)), dim3(COPY_WARPS * 32), 0, st, c, f, first);
  });
}

extern "C" size_t ako4x_kv_pages_copy_workspace_bytes(int64_t n, int64_t num_pages) {
  if (n <= PAIRS || num_pages < 0) return 0;
  return 256 + up(4 * num_pages);
}

extern "C" int ako4x_kv_pages_copy(void* const* caches, const int64_t* page_bytes, const int64_t* page_strides, int64_t num_caches,
                                   const int32_t* src, const int32_t* dst, uint8_t* ok, int64_t n, int64_t num_pages,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (!counts_ok(n, 0, 0, num_pages, 1) || !caches_ok(caches, page_bytes, page_strides, num_caches) || !ok) return AKO4X_EINVAL;
  cudaStream_t st = (cudaStream_t)stream;
  if (n > 0 && (!int_ptr(src) || !int_ptr(dst))) return AKO4X_EINVAL;
  if (n > PAIRS && (!workspace || workspace_bytes < ako4x_kv_pages_copy_workspace_bytes(n, num_pages))) return AKO4X_EWORKSPACE;
  if ((uintptr_t)workspace & 15) return AKO4X_EINVAL;
  if (n == 0) return cudaMemsetAsync(ok, 1, 1, st) == cudaSuccess ? AKO4X_OK : AKO4X_ELAUNCH;
  if (n <= PAIRS)
    return for_caches(caches, page_bytes, page_strides, num_caches, [&](const Caches& c, bool) {
      return ako::launch_pdl(true, copy_short_kernel, dim3(copy_grid(n * c.first_piece[c.count])), dim3(COPY_WARPS * 32), 0, st, c, src, dst,
                             (int)n, (int)num_pages, ok);
    });
  int32_t* go = (int32_t*)workspace;
  if (ako::launch_pdl(true, copy_plan_kernel, dim3(1), dim3(PLAN), 0, st, src, dst, (int)n, (int)num_pages, go + 64, ok, go) != cudaSuccess)
    return AKO4X_ELAUNCH;
  return for_caches(caches, page_bytes, page_strides, num_caches, [&](const Caches& c, bool first) {
    return ako::launch_pdl(first, copy_kernel, dim3(copy_grid(n * c.first_piece[c.count])), dim3(COPY_WARPS * 32), 0, st, c, src, dst,
                           (int)n, (int)num_pages, (const int32_t*)go);
  });
}

extern "C" size_t ako4x_kv_pages_compact_workspace_bytes(int64_t num_pages) {
  if (num_pages <= 0) return 0;
  return 256 + up(4 * ako::cdiv(num_pages, (int64_t)TILE)) + 3 * up(4 * num_pages);
}

extern "C" int ako4x_kv_pages_compact(void* const* caches, const int64_t* page_bytes, const int64_t* page_strides,
                                      int64_t num_caches, int32_t* block_table, int32_t* ref_counts, int32_t* page_map,
                                      int64_t num_rows, int64_t max_pages, int64_t num_pages, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  if (!counts_ok(0, num_rows, max_pages, num_pages, 1) || !caches_ok(caches, page_bytes, page_strides, num_caches)) return AKO4X_EINVAL;
  if (num_pages == 0) return AKO4X_OK;
  if (!int_ptr(ref_counts) || !int_ptr(page_map) || (num_rows * max_pages > 0 && !int_ptr(block_table))) return AKO4X_EINVAL;
  if (!workspace || workspace_bytes < ako4x_kv_pages_compact_workspace_bytes(num_pages)) return AKO4X_EWORKSPACE;
  if ((uintptr_t)workspace & 15) return AKO4X_EINVAL;
  cudaStream_t st = (cudaStream_t)stream;
  const int tiles = (int)ako::cdiv(num_pages, (int64_t)TILE);
  unsigned char* ws = (unsigned char*)workspace;
  int32_t* moves = (int32_t*)ws;
  int32_t* counts = (int32_t*)(ws + 256);
  int32_t* code = (int32_t*)(ws + 256 + up(4 * (size_t)tiles));
  int32_t* src = (int32_t*)((unsigned char*)code + up(4 * num_pages));
  int32_t* dst = (int32_t*)((unsigned char*)src + up(4 * num_pages));
  if (tiles > 1) {
    if (ako::launch_pdl(true, compact_count_kernel, dim3(tiles), dim3(PLAN), 0, st, (const int32_t*)ref_counts, (int)num_pages, counts) != cudaSuccess)
      return AKO4X_ELAUNCH;
  }
  if (ako::launch_pdl(true, compact_plan_kernel, dim3(tiles), dim3(PLAN), 0, st, (const int32_t*)ref_counts, (int)num_pages,
                      (const int32_t*)counts, tiles, code, src, dst, moves) != cudaSuccess)
    return AKO4X_ELAUNCH;
  Compact k = {block_table, ref_counts, page_map, code, src, dst, moves, num_rows * max_pages, (int)num_pages};
  return for_caches(caches, page_bytes, page_strides, num_caches, [&](const Caches& c, bool first) {
    // how many pages move is known on the device only
    const int64_t units = std::max<int64_t>(num_pages / 2 * c.first_piece[c.count], ako::cdiv(num_rows * max_pages, (int64_t)128));
    return ako::launch_pdl(first, compact_kernel, dim3(copy_grid(units)), dim3(COPY_WARPS * 32), 0, st, c, k, first);
  });
}
