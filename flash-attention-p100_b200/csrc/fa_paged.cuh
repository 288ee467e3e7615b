// fa_paged.cuh -- the paged key-value cache: pages handed to requests and taken
// back, new keys and values written to their slots, and the attention of one
// new token per request over its pages. No counterpart in the reference, which
// has no cache.
//
// A cache is (P, Hkv, page, D): P pages of `page` tokens (a multiple of 16). A
// block table (B, W) lists every request's pages, a token's slot is
// page_id * page + offset, and the free pages are the first free_count entries
// of a stack. Every page id and slot read from device memory is checked against
// the pool before it addresses anything; the host cannot see them.
#pragma once
#include <cmath>
#include <cstdint>

#include "sm100.cuh"

namespace fab {

// ---------------------------------------------------------------------------
// block tables
// ---------------------------------------------------------------------------
// Both calls are two running sums over the requests, by one block, and then
// writes that need only their results. The sums are latency: a load, two scans,
// a store. The writes go by the same block where the host knows that they are
// few, else by a second launch that fills the GPU and whose start overlaps the
// first (kExtendWide, kReleaseWide). Bound by latency throughout: 64 decoding
// requests take 2.4 us, 1024 prompts with 1.03 M tokens 11.3 us (4.7 MB read and
// written), the return of 262 k pages of 2048 requests 7.9 us.
constexpr int kTableThreads = 1024;
// Slots (extend), and runs of kReleaseRun table entries of all requests (release),
// above which the second launch pays. Measured, one block against two launches, in
// us: 4096 slots of 128 requests 4.4 / 5.1, 8192 6.0 / 5.0; 64 requests of up to 512
// pages (128 runs) 3.8 / 4.2 when every eighth ends, 9.2 / 5.4 when all do, and 2 us of
// host time less; 256 requests of up to 256 pages (256 runs) 5.2 / 5.2 and 19.2 / 5.4.
constexpr int kExtendWide = 4096, kReleaseWide = 128;
// Up to this many tokens a request's own thread writes them (a decoding step);
// a page holds 16 or more, so they take at most one new page.
constexpr int kSlotsByRow = 4;

// What the writes need of a request.
struct alignas(16) TableRow {
  int tok;    // first token of the request in the call's packed tokens (extend)
  int page;   // first page of the request in the call's pages
  int len;    // length before the call
  int count;  // tokens granted (extend) or pages given back (release)
};
struct alignas(16) TableHead {
  int pages;    // pages the call takes or gives back
  int free;     // free pages before the call
  int by_rows;  // the requests' own threads have written every slot (extend)
  int pad;
};

__device__ __forceinline__ int clamp_count(int n, int P) { return min(max(n, 0), P); }

__device__ __forceinline__ int clip_int(long long x) {
  return x > 0x7fffffffll ? 0x7fffffff : static_cast<int>(x);
}

// Blocks until the launch before this one has ended and its writes are seen
// (programmatic dependent launch).
__device__ __forceinline__ void wait_for_prior_launch() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Inclusive sum over the block of one value per thread; *total is the block's.
// `sums` holds 32 values of shared memory. 64 bits: lengths add up past 2^31.
__device__ __forceinline__ long long block_sum(long long x, long long* sums, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // `sums` of the previous call is read
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  long long s = lane < static_cast<int>(blockDim.x >> 5) ? sums[lane] : 0;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, s, d);
    if (lane >= d) s += y;
  }
  *total = __shfl_sync(0xffffffffu, s, 31);
  const long long before = __shfl_sync(0xffffffffu, s, max(warp - 1, 0));
  return x + (warp ? before : 0);
}

// Last row r of [0, B) with start(r) <= x; start does not fall, start(0) is 0.
template <typename Start>
__device__ __forceinline__ int last_at_most(const Start& start, int B, int x) {
  int lo = 0, hi = B;  // start(lo) <= x < start(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start(mid) <= x) lo = mid; else hi = mid;
  }
  return lo;
}

struct ExtendArgs {
  const int *new_lens, *lens, *free_pages, *free_count;
  int *table, *slots, *granted, *lens_out, *free_out;
  long long table_stride;
  TableHead* head;
  TableRow* rows;
  int B, W, P, page, T;
};

__device__ __forceinline__ int slot_of(int id, int off, const ExtendArgs& a) {
  return static_cast<unsigned>(id) < static_cast<unsigned>(a.P) ? id * a.page + off : -1;
}

// Which requests are served and where their tokens and pages start:
//   e = sum of new tokens (served or not): the packed position of the tokens
//   c = sum of new pages of the requests that fit their row and the call
// A request is served if it needs no page or c <= free. A request of few tokens
// is finished here, with the entry of its last page loaded ahead of the sums.
// Returns whether a longer one is left to extend_fill.
__device__ __forceinline__ bool extend_rows(const ExtendArgs& a) {
  __shared__ long long sums[32];
  __shared__ int most;
  if (threadIdx.x == 0) most = 0;
  const int free = clamp_count(*a.free_count, a.P);
  const long long cap = static_cast<long long>(a.W) * a.page;
  long long tok0 = 0, page0 = 0;
  int taken = 0;
  bool longer = false;
  for (int r0 = 0; r0 < a.B; r0 += static_cast<int>(blockDim.x)) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    const int n = r < a.B ? max(a.new_lens[r], 0) : 0;
    const int len = r < a.B ? a.lens[r] : 0;
    const bool room = n > 0 && len >= 0 && static_cast<long long>(len) + n <= cap;
    const int p0 = room ? (len + a.page - 1) / a.page : 0;
    int* row = a.table + static_cast<long long>(r) * a.table_stride;
    const int last = room && n <= kSlotsByRow && p0 * a.page > len ? row[p0 - 1] : -1;
    long long all;
    const long long e = tok0 + block_sum(n, sums, &all);
    tok0 += all;
    const bool fits = room && e <= a.T;
    const int want = fits ? (len + n + a.page - 1) / a.page - p0 : 0;
    const long long c = page0 + block_sum(want, sums, &all);
    page0 += all;
    const bool ok = fits && (want == 0 || c <= free);
    if (ok && want) taken = static_cast<int>(c);
    if (r < a.B) {
      a.rows[r] = TableRow{clip_int(e - n), clip_int(c - want), len, ok ? n : 0};
      a.granted[r] = ok ? n : 0;
      a.lens_out[r] = len + (ok ? n : 0);
    }
    if (n > kSlotsByRow) {
      longer = true;
    } else if (n) {
      int fresh = -1;
      if (ok && want) row[p0] = fresh = a.free_pages[free - static_cast<int>(c)];
#pragma unroll
      for (int i = 0; i < kSlotsByRow; ++i) {
        const long long t = e - n + i;
        if (i >= n || t >= a.T) break;
        const int pos = len + i, in_new = pos - p0 * a.page;
        a.slots[t] = !ok ? -1 : in_new >= 0 ? slot_of(fresh, in_new, a) : slot_of(last, in_new + a.page, a);
      }
    }
  }
  // pages taken: c of the last served request that takes any
  taken = __reduce_max_sync(0xffffffffu, taken);
  if ((threadIdx.x & 31) == 0) atomicMax(&most, taken);
  longer = __syncthreads_or(longer);
  // no token behind the last; extend_fill writes these too
  if (!longer)
    for (long long t = tok0 + threadIdx.x; t < a.T; t += blockDim.x) a.slots[t] = -1;
  if (threadIdx.x == 0) {
    *a.head = TableHead{most, free, longer ? 0 : 1, 0};
    *a.free_out = free - most;
  }
  return longer;
}

// The slots of the call's tokens and the new entries of the block table, by
// threads `first`, `first + step`, ... of the launch. New entries lie behind
// the entries that this reads (a request's pages so far), so the order of the
// threads does not matter. A thread takes kSlotRun tokens in a row: one search
// and, inside a request, at most two pages (a page holds 16 or more). A run that meets
// a request's end steps over the requests behind it one by one: 5001 tokens of one
// request take 5.2 us alone, 9.1 ahead of 63 requests without new tokens, 20 of 255 and
// 122 of 2047.
constexpr int kSlotRun = 8;
constexpr int kRowsShared = 2048;  // rows whose first tokens and pages are searched in shared memory

// Page of position j * page ... of a row, given its TableRow.
__device__ __forceinline__ int page_id(const ExtendArgs& a, const TableRow& row, int r, int j, int free) {
  const int fresh = j - (row.len + a.page - 1) / a.page;  // >= 0: a page of this call
  return fresh >= 0 ? a.free_pages[free - 1 - row.page - fresh] : a.table[r * a.table_stride + j];
}

template <typename Tok, typename Page>
__device__ __forceinline__ void extend_fill(const ExtendArgs& a, const Tok& tok, const Page& page_of,
                                            long long first, long long step) {
  const int free = a.head->free, pages = a.head->pages;
  const bool vec = (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0;
  for (long long t0 = first * kSlotRun; t0 < a.T; t0 += step * kSlotRun) {
    const int t = static_cast<int>(t0);
    int r = last_at_most(tok, a.B, t);
    TableRow row = a.rows[r];
    int slot[kSlotRun];
    const int in = t - row.tok;
    if (row.count - in >= kSlotRun) {   // one request
      const int pos = row.len + in, j = pos / a.page, off = pos - j * a.page;
      const int id0 = page_id(a, row, r, j, free);
      const int id1 = off + kSlotRun > a.page ? page_id(a, row, r, j + 1, free) : -1;
#pragma unroll
      for (int i = 0; i < kSlotRun; ++i)
        slot[i] = off + i < a.page ? slot_of(id0, off + i, a) : slot_of(id1, off + i - a.page, a);
    } else {
      for (int i = 0; i < kSlotRun; ++i) {
        const long long ti = t0 + i;
        while (r + 1 < a.B && tok(r + 1) <= ti) row = a.rows[++r];
        const long long at = ti - row.tok;
        int x = -1;
        if (at < row.count) {
          const int pos = row.len + static_cast<int>(at), j = pos / a.page;
          x = slot_of(page_id(a, row, r, j, free), pos - j * a.page, a);
        }
        if (ti < a.T) a.slots[ti] = x;
      }
      continue;
    }
    if (vec) {
      int4* out = reinterpret_cast<int4*>(a.slots + t0);
      out[0] = make_int4(slot[0], slot[1], slot[2], slot[3]);
      out[1] = make_int4(slot[4], slot[5], slot[6], slot[7]);
    } else {
#pragma unroll
      for (int i = 0; i < kSlotRun; ++i) a.slots[t0 + i] = slot[i];
    }
  }
  for (long long k = first; k < pages; k += step) {
    const int r = last_at_most(page_of, a.B, static_cast<int>(k));
    const TableRow row = a.rows[r];
    const int j = (row.len + a.page - 1) / a.page + static_cast<int>(k) - row.page;
    a.table[r * a.table_stride + j] = a.free_pages[free - 1 - k];
  }
}

// The block's searches: in shared memory where the rows fit, so that a search
// costs one round trip to L2 and not one per step.
__device__ __forceinline__ void extend_fill_block(const ExtendArgs& a, long long first, long long step) {
  __shared__ int s_tok[kRowsShared], s_page[kRowsShared];
  if (a.B <= kRowsShared) {
    for (int r = threadIdx.x; r < a.B; r += blockDim.x) {
      const int2 x = *reinterpret_cast<const int2*>(a.rows + r);
      s_tok[r] = x.x;
      s_page[r] = x.y;
    }
    __syncthreads();
    extend_fill(a, [&](int r) { return s_tok[r]; }, [&](int r) { return s_page[r]; }, first, step);
  } else {
    extend_fill(a, [&](int r) { return a.rows[r].tok; }, [&](int r) { return a.rows[r].page; }, first, step);
  }
}

__global__ void __launch_bounds__(kTableThreads) extend_kernel(const ExtendArgs a, int fill) {
  wait_for_prior_launch();
  const bool longer = extend_rows(a);
  if (!fill || !longer) return;
  __syncthreads();
  extend_fill_block(a, threadIdx.x, blockDim.x);
}

__global__ void __launch_bounds__(256) extend_fill_kernel(const ExtendArgs a) {
  wait_for_prior_launch();
  if (a.head->by_rows) return;
  extend_fill_block(a, blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll);
}

struct ReleaseArgs {
  const unsigned char* finished;
  const int *lens, *table, *free_count;
  int *free_pages, *lens_out, *free_out;
  long long table_stride;
  TableHead* head;
  TableRow* rows;
  int B, W, P, page;
};

// Entries of a row that a warp copies at a time.
constexpr int kReleaseRun = 256;

// Entries [j0, j0 + kReleaseRun) of row r onto the stack, by one warp. `row` has
// the row's count and first page, `pages` is where the call's pages end.
__device__ __forceinline__ void release_run(const ReleaseArgs& a, const TableRow& row, int r, int j0, int free,
                                            int pages) {
  // a clipped first page is behind the stack's end
  const long long end = min(min(static_cast<long long>(row.count), static_cast<long long>(j0) + kReleaseRun),
                            static_cast<long long>(pages) - row.page);
  const int* from = a.table + r * a.table_stride;
  int* to = a.free_pages + free + row.page;
#pragma unroll 8
  for (long long j = j0 + static_cast<int>(threadIdx.x & 31); j < end; j += 32) to[j] = from[j];
}

// Which requests give pages back and where those start. With FILL the block also
// copies them, the finished requests of kTableThreads rows at a time from a list
// in shared memory; else `rows` and `head` tell release_fill_kernel.
template <bool FILL>
__global__ void __launch_bounds__(kTableThreads) release_kernel(const ReleaseArgs a) {
  __shared__ long long sums[32];
  __shared__ TableRow s_row[FILL ? kTableThreads : 1];
  __shared__ int s_index[FILL ? kTableThreads : 1];
  wait_for_prior_launch();
  const int free = clamp_count(*a.free_count, a.P), room = a.P - free;
  // more pages than the stack has room for cannot come from one pool: the rest
  // are dropped
  long long page0 = 0;
  for (int r0 = 0; r0 < a.B; r0 += static_cast<int>(blockDim.x)) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    const bool done = r < a.B && a.finished[r] != 0;
    const int len = r < a.B ? a.lens[r] : 0;
    const int n = done ? (min(max(len, 0), a.W * a.page) + a.page - 1) / a.page : 0;
    // two sums in one: pages below bit 48, requests that have any above it
    constexpr int kCount = 48;
    long long all;
    const long long sum = block_sum(n + (static_cast<long long>(n > 0) << kCount), sums, &all);
    const long long c = page0 + (sum & ((1ll << kCount) - 1));
    const TableRow row{0, clip_int(c - n), len, n};
    if (r < a.B) {
      if (!FILL) a.rows[r] = row;
      a.lens_out[r] = done ? 0 : len;
    }
    if (FILL) {
      if (n > 0) {
        s_row[(sum >> kCount) - 1] = row;
        s_index[(sum >> kCount) - 1] = r;
      }
      __syncthreads();
      const int listed = static_cast<int>(all >> kCount), runs = (a.W + kReleaseRun - 1) / kReleaseRun;
      const long long items = static_cast<long long>(listed) * runs;
      for (long long i = threadIdx.x >> 5; i < items; i += blockDim.x >> 5) {
        const int at = static_cast<int>(i / runs);
        release_run(a, s_row[at], s_index[at], static_cast<int>(i - static_cast<long long>(at) * runs) * kReleaseRun,
                    free, room);
      }
    }
    page0 += all & ((1ll << kCount) - 1);
  }
  if (threadIdx.x == 0) {
    const int back = static_cast<int>(min(page0, static_cast<long long>(room)));
    if (!FILL) *a.head = TableHead{back, free, 0, 0};
    *a.free_out = free + back;
  }
}

__global__ void __launch_bounds__(256) release_fill_kernel(const ReleaseArgs a) {
  wait_for_prior_launch();
  const int free = a.head->free, pages = a.head->pages;
  const int runs = (a.W + kReleaseRun - 1) / kReleaseRun;
  const long long items = static_cast<long long>(a.B) * runs;
  for (long long i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < items; i += gridDim.x * 8ll) {
    const int r = static_cast<int>(i / runs), j0 = static_cast<int>(i - static_cast<long long>(r) * runs) * kReleaseRun;
    const TableRow row = a.rows[r];
    if (j0 < row.count) release_run(a, row, r, j0, free, pages);
  }
}

// ---------------------------------------------------------------------------
// append: rows of k and v to their slots
// ---------------------------------------------------------------------------
struct AppendArgs {
  const uint16_t *k, *v;
  uint16_t *k_cache, *v_cache;
  Strides sk, sv, skc, svc;  // rows: h head, n token; caches: b page, h head, n token
  const int* slots;
  int T, Hkv, P, page;
};

// A 16-byte piece of k and of v per thread; the pieces of a row are neighbouring
// threads. The loads are finished ahead of the test of the slot, so that no copy
// waits for two loads in turn. Bound by HBM: 65536 tokens of 8 heads of 128 take
// 81 us, 6.6 TB/s read and written (84 us with the test first; several rows a
// thread are no faster there and slower below).
template <int D>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  wait_for_prior_launch();
  constexpr int CH = D / 8;
  const long long row = static_cast<long long>(blockIdx.x) * (256 / CH) + threadIdx.x / CH;
  const int c = static_cast<int>(threadIdx.x) % CH * 8;
  uint4 k, v;
  int slot = -1, h = 0;
  if (row < static_cast<long long>(a.T) * a.Hkv) {
    const int t = static_cast<int>(row / a.Hkv);
    h = static_cast<int>(row - static_cast<long long>(t) * a.Hkv);
    slot = a.slots[t];
    k = *reinterpret_cast<const uint4*>(a.k + a.sk.at(0, h, t) + c);
    v = *reinterpret_cast<const uint4*>(a.v + a.sv.at(0, h, t) + c);
  }
  if (slot >= 0 && slot < a.P * a.page) {
    const int id = slot / a.page, off = slot - id * a.page;
    *reinterpret_cast<uint4*>(a.k_cache + a.skc.at(id, h, off) + c) = k;
    *reinterpret_cast<uint4*>(a.v_cache + a.svc.at(id, h, off) + c) = v;
  }
}

// ---------------------------------------------------------------------------
// attention of one new token per request
// ---------------------------------------------------------------------------
// o_h = sum_j softmax_j(q_h . k_j / sqrt(D)) v_j over a request's cached tokens.
// Every cached byte is read once for Hq/Hkv query heads: 1 FLOP per byte and
// head, so HBM is the bound, and the matrix instruction only has to keep up
// with the loads. That is why this is mma.sync and not tcgen05: a group of 1 to
// 16 heads fills one m16 fragment (a tcgen05 tile would be 128 rows), operands
// come straight out of the loaded tile, and no accumulator leaves registers.
//
// A unit is one request's kv head and a tile of up to ROWS of its query heads;
// its keys are taken in steps of STEP. The steps are cut along the keys in one
// of two ways:
//   * the line (CLUSTER false): all units in order form one line of steps that
//     is divided evenly over the blocks of the launch. A block walks its stretch
//     through unit after unit; a unit that lies within one stretch is finished
//     there, one cut by a border is left as partial results (o, max, sum in
//     fp32) that paged_join_kernel adds up in the order of the keys. So one long
//     request and a thousand ragged ones both keep every SM loading;
//   * clusters (CLUSTER true): the blocks of a cluster share one unit and meet in
//     distributed shared memory. No sums over the requests ahead, no second
//     launch: for few and short units, where those are most of the time.
// Either way the result does not depend on timing.
//
// Inside a block each warp takes KEYS of a step's keys into a ring of its own
// (cp.async, 16 bytes a lane), three steps deep, across unit borders too: the
// loads never drain, and warps meet only where a unit ends.
//
// Measured: 64 ragged requests of 32/8 heads of 128 (1.0 GB of cache) 154 to 158 us,
// 6.3 to 6.5 TB/s or 97 to 99% of the measured copy, DRAM traffic equal to the cache's
// bytes, a fifth of the tensor pipe; one request of 131001 tokens 85 us, 6.3 TB/s; one
// of 1000 tokens 6.0 us, a chain of dependent loads (length, page, keys). 16 heads
// for 32 sequences of 4096 tokens, 0.27 GB: 54 us, 5.0 TB/s. Wider groups'
// line is paged_wide_kernel's: two fragments' products at 8 warps an SM are bound by
// their latency, 85 us at 32 heads. Clusters take them here, up to 32 heads a tile.

// Blocks of a cluster for `units` units whose table rows hold up to `most` steps
// (32 KB of cache each), 0 where the line is used. Clusters need all their blocks
// at once: two blocks an SM, one for clusters of 16, which fill a GPC. The line
// keeps every SM busy whatever the lengths, but adds them up first and joins in a
// second launch. A cluster has up to `max_cluster` blocks, which the device can place.
// Device time of a call, clusters / line, in us (bf16):
//   8 kv heads, D=128, 1 request:    512 tokens 4.6 / 7.1, 2048 6.7 / 7.8, 8192 12.3 / 10.7
//   32 requests of 512 tokens 11.0 / 14.7, of 1 to 512 10.3 / 13.2, of 1 to 1024 16.2 / 18.5
//   20 requests (160 blocks) of 512 tokens 10.7 / 12.7, of 1024 17.4 / 16.5
//   40 requests (two blocks a unit, in waves) of 256 tokens 14.9 / 12.9
//   1 kv head, D=64, 1 request: 2048 tokens 5.1 / 6.6, 8192 7.7 / 7.0, 16000 13.2 / 8.4
//   256 units (a block each), D=64, 2048 tokens 25.1 / 28.8, of 1 to 2048 19.2 / 16.8
//   64 units (four blocks each), D=64, 2048 tokens 8.2 / 11.6, 8192 25.7 / 28.7, of 1 to
//   8192 19.3 / 15.7; D=128, 2048 tokens 11.2 / 14.3, 4096 24.9 / 28.4, of 1 to 4096 16.7 / 15.2
// so the steps a block may have to take grow with the part of the GPU in use, where
// a unit's keys are spread over several blocks. Lengths are not known here, so the rule
// goes by the rows of the table and has a wrong side: full rows at its borders (8192
// tokens above), ragged ones in long rows, and 72 to 74 units, whose clusters of four
// do not all find a place at once (74 units, D=64, 1024 tokens 9.3 / 8.2, 8192 42 / 31).
__host__ constexpr int paged_cluster(long long units, long long most, int sms, int max_cluster) {
  for (int c = max_cluster; c >= 1; c /= 2) {
    const long long blocks = units * c;
    if (c > 1 && c / 2 >= most) continue;   // no more blocks than steps
    if (blocks > (c == 16 ? sms : 2 * sms)) continue;
    const int steps = c > 1 && 2 * blocks > 3 * sms ? 16 : 2 * blocks > sms ? 8 : 4;
    return most <= static_cast<long long>(c) * steps ? c : 0;
  }
  return 0;
}

// Strides of a cache in units of 16 bytes (page, head, token): 32 bits each, so a
// stride may be 64 GB, and one instruction for each product, which has 64.
struct Units {
  uint32_t b, h, n;
};
struct PagedAttnArgs {
  const uint16_t* q;
  const uint4 *k_cache, *v_cache;
  uint16_t* o;
  float* lse;
  Strides sq, so;             // b request, h head
  Units skc, svc;             // of the caches
  const int *table, *lens;
  long long table_stride;
  int B, Hq, Hkv, P, W, page;
  int row_tiles;              // tiles of ROWS heads in a group
  float scale;     // log2(e) / sqrt(D)
  // What paged_join_kernel has to add up: {unit, first block, last block}, unit < 0
  // for nothing. One per unit where there are no more units than blocks, else one
  // per block, of the unit that begins and does not end in it.
  int4* split;
  float2* part_ml; // per block two partial results: [2 block + first][row] max and sum
  float* part_o;   // ... and [2 block + first][row][D]
  int* err;
};

template <int D>
struct PagedCfg {
  static constexpr int WARPS = 4;
  static constexpr int STAGES = 3;
  static constexpr int KEYS = 2048 / D;       // of a warp in a step: 4 KB of K, 4 KB of V
  static constexpr int STEP = WARPS * KEYS;
  static constexpr int GROUPS = KEYS / 16;    // runs of 16 keys: each lies in one page
  static constexpr int ALL = GROUPS == 2 ? 0x1010 : 0x10;  // keys of the runs, 8 bits each, when all are real
  static constexpr int TILE = KEYS * D * 2;   // bytes of a warp's K (or V) of a step
  static constexpr int RING = WARPS * STAGES * 2 * TILE;
  static constexpr int MERGE = WARPS * 8 * D * 4;  // the warps' fp32 results of 8 rows
  static constexpr int SMEM = RING + MERGE;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// `bytes` of the 16 are read, the rest is filled with zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// c (16 x 8 fp32) += a (16 x 16) b (16 x 8), 16-bit operands
template <bool BF>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF>
__device__ __forceinline__ float2 unpack16(uint32_t x) {
  if (BF) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float x, float y) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
  float2 x;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(addr) : "memory");
  return x;
}

// A running softmax of four columns: folds in a part with maximum and sum ml
// and unnormalised columns x.
struct PartSum {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float2 ml, float4 x) {
    const float mn = fmaxf(m, ml.x), ref = mn == -INFINITY ? 0.f : mn;
    const float w = ex2(m - ref), y = ex2(ml.x - ref);
    m = mn;
    l = l * w + ml.y * y;
    o.x = o.x * w + x.x * y;
    o.y = o.y * w + x.y * y;
    o.z = o.z * w + x.z * y;
    o.w = o.w * w + x.w * y;
  }
};

// Weights are 2^(s - m + bias): m is the running maximum when it last grew by
// more than 2^8 (scaling o and l only then), and in fp16 the bias keeps weights
// down to 2^-21 of the largest out of the subnormals (they end at 2^15).
template <bool BF>
__device__ __forceinline__ constexpr float weight_bias() { return BF ? 0.f : 7.f; }

// Writes columns col .. col + 3 of a head's result. Weights that sum to 0 (no key with
// a page, or every score -inf) give what a request without a token gets, o = 0 beside
// lse = -inf, and not 0 / 0.
template <bool BF>
__device__ __forceinline__ void store_part_sum(const PagedAttnArgs& a, const PartSum& x, int b, int head, int col) {
  const float inv = x.l == 0.f ? 0.f : 1.f / x.l;
  *reinterpret_cast<uint2*>(a.o + a.so.at(b, head, 0) + col) =
      make_uint2(pack16<BF>(x.o.x * inv, x.o.y * inv), pack16<BF>(x.o.z * inv, x.o.w * inv));
  if (col == 0)
    a.lse[static_cast<long long>(b) * a.Hq + head] = 0.6931471805599453f * (x.m - weight_bias<BF>() + log2f(x.l));
}

// x + y, the sums of the weights' first and second terms; x alone where it is not
// finite: an infinite value times a second term of 0 or below says nothing.
__device__ __forceinline__ float add_finite(float x, float y) { return fabsf(x) < INFINITY ? x + y : x; }

// Two 16-bit values, infinities (and NaN) replaced by finite ones, for the same reason.
template <bool BF>
__device__ __forceinline__ uint32_t finite16(uint32_t x) {
  if (BF) {
    const __nv_bfloat162 top = __nv_bfloat162(__ushort_as_bfloat16(0x7f7f), __ushort_as_bfloat16(0x7f7f));
    const __nv_bfloat162 y = __hmin2(__hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x), __hneg2(top)), top);
    return *reinterpret_cast<const uint32_t*>(&y);
  }
  const __half2 top = __half2(__ushort_as_half(0x7bff), __ushort_as_half(0x7bff));
  const __half2 y = __hmin2(__hmax2(*reinterpret_cast<const __half2*>(&x), __hneg2(top)), top);
  return *reinterpret_cast<const uint32_t*>(&y);
}

// Adds up the warps' results of a unit, 8 rows at a time through shared memory
// (`buf`, 8 D floats a warp; 32-byte pieces xor-ed with the row, so neither side
// conflicts), and calls emit(row, column, sum) for every four columns.
template <int D, int E, int MT, typename Emit>
__device__ __forceinline__ void merge_warps(unsigned char* buf, float2 (&s_ml)[4][8], float (&o)[MT][D / 8][4],
                                            float (&m)[MT][E], float (&l)[MT][E], const Emit& emit) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row_w = lane >> 2;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float sum = l[mt][e];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      __syncthreads();   // buf and s_ml are free
      unsigned char* mine = buf + (warp * 8 + row_w) * (D * 4) + (lane & 3) * 8;
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<float2*>(mine + ((i ^ row_w) << 5)) =
            E == 1 ? make_float2(add_finite(o[mt][i][0], o[mt][i][2]), add_finite(o[mt][i][1], o[mt][i][3]))
                   : make_float2(o[mt][i][2 * e], o[mt][i][2 * e + 1]);
      if ((lane & 3) == 0) s_ml[warp][row_w] = make_float2(m[mt][e], sum);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8 * (D / 4) / 128; ++i) {
        const int at = i * 128 + static_cast<int>(threadIdx.x), row = at / (D / 4), col = at % (D / 4) * 4;
        PartSum part;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          part.add(s_ml[w][row], *reinterpret_cast<const float4*>(buf + (w * 8 + row) * (D * 4) +
                                                                 (((col >> 3) ^ row) << 5) + (col & 4) * 4));
        emit(mt * 16 + e * 8 + row, col, part);
      }
    }
}

__device__ __forceinline__ const uint4* unit_at(const uint4* base, const Units& s, uint32_t b, uint32_t h,
                                                uint32_t n) {
  return base + (static_cast<uint64_t>(b) * s.b + static_cast<uint64_t>(h) * s.h + static_cast<uint64_t>(n) * s.n);
}

// A place on the line of steps.
struct PagedAt {
  int b, head, rt;  // request, kv head, row tile
  int t, nt;        // step of the unit, steps of the unit
  int len;
};

__device__ __forceinline__ int request_len(const PagedAttnArgs& a, int b) {
  return min(max(a.lens[b], 0), a.W * a.page);
}

// The result of `heads` heads of a request without a token, by the whole block.
template <int D, int THREADS>
__device__ __forceinline__ void empty_row(const PagedAttnArgs& a, int b, int head0, int heads) {
  for (int i = threadIdx.x; i < heads * (D / 2); i += THREADS)
    *reinterpret_cast<uint32_t*>(a.o + a.so.at(b, head0 + i / (D / 2), 0) + i % (D / 2) * 2) = 0;
  for (int h = threadIdx.x; h < heads; h += THREADS)
    a.lse[static_cast<long long>(b) * a.Hq + head0 + h] = -INFINITY;
}

// A block's stretch of the line, found by every block for itself.
struct Line {
  long long total, end;  // steps of the line; where the stretch ends
  int blocks;            // blocks that have a stretch
};
struct LineShared {
  long long sums[16], first;  // a sum per warp; first: the stretch's first step in its request
  int b;                      // that request
};

// Adds up the lengths, divides the line, finds this block's stretch and deals
// with the requests without a token. Returns the stretch's steps.
template <int STEP, int D, int THREADS>
__device__ __forceinline__ long long line_begin(const PagedAttnArgs& a, int units, bool by_unit, Line& line,
                                                LineShared& shared) {
  static_assert(THREADS / 32 <= static_cast<int>(sizeof(shared.sums) / sizeof(shared.sums[0])), "a sum per warp");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const auto steps = [&](int b) { return (request_len(a, b) + STEP - 1) / STEP; };
  const int per = (a.B + THREADS - 1) / THREADS;
  const int b0 = min(static_cast<int>(threadIdx.x) * per, a.B), b1 = min(b0 + per, a.B);
  long long mine = 0, total = 0;
  for (int b = b0; b < b1; ++b) mine += static_cast<long long>(steps(b)) * units;
  long long sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += y;
  }
  if (lane == 31) shared.sums[warp] = sum;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) sum += shared.sums[w];
    total += shared.sums[w];
  }
  const int blocks = static_cast<int>(min(static_cast<long long>(gridDim.x), total)), c = blockIdx.x;
  const long long g0 = c < blocks ? c * total / blocks : total;
  const long long g1 = c < blocks ? (c + 1) * total / blocks : total;
  long long first = sum - mine;
  if (first <= g0 && g0 < sum) {
    int b = b0;
    for (;; ++b) {
      const long long n = static_cast<long long>(steps(b)) * units;
      if (g0 < first + n) break;
      first += n;
    }
    shared.b = b;
    shared.first = g0 - first;
  }
  line.total = total;
  line.end = g1;
  line.blocks = blocks;
  if (!by_unit && threadIdx.x == 0) a.split[blockIdx.x] = make_int4(-1, 0, 0, 0);
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    if (request_len(a, b) != 0) continue;
    empty_row<D, THREADS>(a, b, 0, a.Hq);
    if (by_unit)
      for (int u = threadIdx.x; u < units; u += THREADS) a.split[b * units + u] = make_int4(-1, 0, 0, 0);
  }
  __syncthreads();
  return g1 - g0;
}

// Where the stretch begins.
template <int STEP>
__device__ __forceinline__ PagedAt line_at(const PagedAttnArgs& a, const LineShared& shared) {
  PagedAt at;
  at.b = shared.b;
  at.len = request_len(a, at.b);
  at.nt = (at.len + STEP - 1) / STEP;
  const int unit = static_cast<int>(shared.first / at.nt);
  at.t = static_cast<int>(shared.first - static_cast<long long>(unit) * at.nt);
  at.head = unit / a.row_tiles;
  at.rt = unit - at.head * a.row_tiles;
  return at;
}

// The unit behind x's on the line.
template <int STEP>
__device__ __forceinline__ void next_unit(const PagedAttnArgs& a, PagedAt& x) {
  x.t = 0;
  if (++x.rt < a.row_tiles) return;
  x.rt = 0;
  if (++x.head < a.Hkv) return;
  x.head = 0;
  do x.len = request_len(a, ++x.b); while (x.len == 0);
  x.nt = (x.len + STEP - 1) / STEP;
}

// For paged_join_kernel: the unit that begins in this block, `done` its last step
// here, and the block that holds the unit's last step where it is cut.
__device__ __forceinline__ void line_record(const PagedAttnArgs& a, const Line& line, const PagedAt& done, bool whole,
                                            bool by_unit) {
  if (whole && !by_unit) return;
  const int unit = (done.b * a.Hkv + done.head) * a.row_tiles + done.rt;
  const long long last = line.end - 1 + (done.nt - 1 - done.t);
  a.split[by_unit ? unit : static_cast<int>(blockIdx.x)] =
      make_int4(whole ? -1 : unit, blockIdx.x,
                whole ? 0 : static_cast<int>(((last + 1) * line.blocks - 1) / line.total), 0);
}

// ROWS query heads of a group per unit: 8 (half of an m16 fragment, whose other
// half takes the weights' second terms), 16 (one fragment) or 32 (two); a group
// above 32 is cut into row tiles, each of which reads the cache again.
template <int D, bool BF, int ROWS, bool CLUSTER>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedAttnArgs a) {
  using C = PagedCfg<D>;
  constexpr int MT = ROWS > 16 ? 2 : 1, E = ROWS == 8 ? 1 : 2;  // fragments, rows a thread holds of each
  constexpr float kBias = weight_bias<BF>();
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ LineShared s_line;
  __shared__ int s_valid[C::WARPS][C::STAGES];
  __shared__ float2 s_ml[C::WARPS][8];
  __shared__ float2 s_unit_ml[ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.Hq / a.Hkv, units = a.Hkv * a.row_tiles;
  const bool by_unit = static_cast<long long>(a.B) * units <= gridDim.x;
  wait_for_prior_launch();
  // ---- this block's steps ----
  PagedAt at;
  Line line{};
  long long n_steps;
  int rank = 0, ranks = 1;   // ranks: also how many steps on the block's next one is
  if constexpr (CLUSTER) {
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const int unit = blockIdx.x / ranks;
    at.b = unit / units;
    at.head = (unit - at.b * units) / a.row_tiles;
    at.rt = unit % a.row_tiles;
    at.len = request_len(a, at.b);
    at.nt = (at.len + C::STEP - 1) / C::STEP;
    at.t = rank;     // steps in turn: where a block begins does not depend on the length
    n_steps = at.nt > rank ? (at.nt - rank + ranks - 1) / ranks : 0;
  } else {
    n_steps = line_begin<C::STEP, D, 128>(a, units, by_unit, line, s_line);
    if (n_steps == 0) return;
    at = line_at<C::STEP>(a, s_line);
  }

  // ---- loads ----
  constexpr int CH = D / 8, RPI = 32 / CH;      // 16-byte pieces of a row, rows a warp covers at once
  const int lc = lane % CH, lr = lane / CH;
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * 2 * C::TILE;
  // piece c of row r lies at r * 2 D + ((c ^ (r & 7)) << 4): RPI rows further on the
  // xor changes by a constant
  const uint32_t ring_lane = ring + lr * (D * 2) + ((lc ^ lr) << 4);
  const int key_w = warp * C::KEYS, page_w = key_w / a.page, off_w = key_w - page_w * a.page;
  const int step_pages = ranks * C::STEP / a.page, step_rest = ranks * C::STEP - step_pages * a.page;
  // The next step to load and the one behind it, their pages already looked up.
  struct Next {
    PagedAt at;
    int page, off;      // of the warp's first key
    int ids[C::GROUPS];
  } ld, ld2;
  const auto fetch_ids = [&](Next& x) {
    // entries behind the request's last page are not used, but in the table
    const int* row = a.table + x.at.b * a.table_stride;
#pragma unroll
    for (int g = 0; g < C::GROUPS; ++g) {
      const int page = x.page + (x.off + g * 16 >= a.page);   // a page holds 16 or more
      x.ids[g] = page < a.W ? row[page] : 0;
    }
  };
  const auto advance = [&](Next& x) {
    x.at.t += ranks;
    if (CLUSTER || x.at.t < x.at.nt) {
      x.page += step_pages;
      x.off += step_rest;
      if (x.off >= a.page) {
        x.off -= a.page;
        ++x.page;
      }
    } else {
      next_unit<C::STEP>(a, x.at);
      x.page = page_w;
      x.off = off_w;
    }
  };
  const auto issue = [&](int stage, const Next& x) {
    const uint32_t dst = ring_lane + stage * 2 * C::TILE;
    const int left = x.at.len - (x.at.t * C::STEP + key_w);
    int valid = 0;
#pragma unroll
    for (int g = 0; g < C::GROUPS; ++g) {
      int n = min(max(left - g * 16, 0), 16), id = x.ids[g];
      if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.P)) {
        if (n && lane == 0) atomicCAS(a.err, 0, static_cast<int>(kErrPage));
        n = id = 0;
      }
      valid |= n << (8 * g);
      int off = x.off + g * 16;
      if (off >= a.page) off -= a.page;
      const uint4* k = unit_at(a.k_cache + lc, a.skc, id, x.at.head, off + lr);
      const uint4* v = unit_at(a.v_cache + lc, a.svc, id, x.at.head, off + lr);
      const uint32_t d = dst + g * 16 * (D * 2);
      if (n == 16) {
#pragma unroll
        for (int i = 0; i < 16 / RPI; ++i) {
          const uint32_t to = (d ^ (((i * RPI) & 7) << 4)) + i * RPI * (D * 2);
          cp_async16(to, unit_at(k, a.skc, 0, 0, i * RPI));
          cp_async16(to + C::TILE, unit_at(v, a.svc, 0, 0, i * RPI));
        }
      } else if (left > 0) {   // rows behind the last token are filled with zeros, not read
#pragma unroll
        for (int i = 0; i < 16 / RPI; ++i) {
          const uint32_t to = (d ^ (((i * RPI) & 7) << 4)) + i * RPI * (D * 2);
          const int bytes = i * RPI + lr < n ? 16 : 0;
          cp_async16(to, unit_at(k, a.skc, 0, 0, i * RPI), bytes);
          cp_async16(to + C::TILE, unit_at(v, a.svc, 0, 0, i * RPI), bytes);
        }
      }
    }
    if (lane == 0) s_valid[warp][stage] = valid;
  };
  long long issued = 0;
  ld.at = at;
  {
    const int key = at.t * C::STEP + key_w;
    ld.page = key / a.page;
    ld.off = key - ld.page * a.page;
  }
  fetch_ids(ld);
  ld2 = ld;
  if (CLUSTER || n_steps > 1) {
    advance(ld2);
    fetch_ids(ld2);
  }
  const auto issue_next = [&](int stage) {
    if (issued < n_steps) {
      issue(stage, ld);
      ld = ld2;
      if (++issued + 1 < n_steps) {
        advance(ld2);
        fetch_ids(ld2);
      }
    }
    cp_async_commit();
  };

  // ---- per unit state ----
  uint32_t qf[MT][D / 16][4];
  float o[MT][D / 8][4], m[MT][E], l[MT][E];
  const auto load_q = [&](const PagedAt& x) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = x.rt * ROWS + mt * 16 + e * 8 + lane / 4;
        const bool real = e < E && r < group;
        const uint16_t* q = a.q + a.sq.at(x.b, x.head * group + min(r, group - 1), 0) + (lane & 3) * 2;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          qf[mt][ks][e] = real ? *reinterpret_cast<const uint32_t*>(q + ks * 16) : 0u;
          qf[mt][ks][e + 2] = real ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + 8) : 0u;
        }
      }
  };
  const auto clear = [&]() {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        m[mt][e] = -INFINITY;
        l[mt][e] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][i][e] = 0.f;
    }
  };
  // ldmatrix addresses of a lane inside a run of 16 keys, for columns 0 .. 15
  const uint32_t k_lane = ((lane >> 4) * 8 + (lane & 7)) * (D * 2) + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
  const uint32_t v_lane = (((lane >> 3) & 1) * 8 + (lane & 7)) * (D * 2) + (((lane >> 4) ^ (lane & 7)) << 4);

  int first_t = at.t;
  load_q(at);
  clear();
  if constexpr (CLUSTER) {
    if (at.len == 0) {   // the whole cluster
      if (rank == 0) empty_row<D, 128>(a, at.b, at.head * group + at.rt * ROWS, min(ROWS, group - at.rt * ROWS));
      return;
    }
  }
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) issue_next(s);
  int stage = C::STAGES - 1;
  for (long long it = 0; it < n_steps; ++it) {
    const int free_stage = stage;
    stage = stage + 1 == C::STAGES ? 0 : stage + 1;
    cp_async_wait<C::STAGES - 2>();
    __syncwarp();   // the step's rows are in, and every lane has left the stage before it
    issue_next(free_stage);
    __syncwarp();   // whole warps from here on
    const int valid = s_valid[warp][stage];
    if (valid != 0) {
      const uint32_t kb = ring + stage * 2 * C::TILE + k_lane, vb = ring + stage * 2 * C::TILE + C::TILE + v_lane;
      float s[MT][2 * C::GROUPS][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 2 * C::GROUPS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][i][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int g = 0; g < C::GROUPS; ++g) {
          uint32_t f[4];
          ldsm4(f, (kb ^ (ks << 5)) + g * 16 * (D * 2));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16<BF>(s[mt][2 * g], qf[mt][ks], f[0], f[1]);
            mma16<BF>(s[mt][2 * g + 1], qf[mt][ks], f[2], f[3]);
          }
        }
      if (valid != C::ALL) {
#pragma unroll
        for (int i = 0; i < 2 * C::GROUPS; ++i) {
          const int n = (valid >> (8 * (i >> 1))) & 255, key = (i & 1) * 8 + (lane & 3) * 2;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2 * E; ++e)
              if (key + (e & 1) >= n) s[mt][i][e] = -INFINITY;
        }
      }
      uint32_t p[MT][C::GROUPS][4], p2[MT][C::GROUPS][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float top[E];
        bool grown = false;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          top[e] = fmaxf(s[mt][0][2 * e], s[mt][0][2 * e + 1]);
#pragma unroll
          for (int i = 1; i < 2 * C::GROUPS; ++i)
            top[e] = fmaxf(top[e], fmaxf(s[mt][i][2 * e], s[mt][i][2 * e + 1]));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2)) * a.scale;
          grown |= top[e] > m[mt][e] + 8.f;
        }
        if (__any_sync(0xffffffffu, grown)) {
          float w[E];
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float mn = fmaxf(m[mt][e], top[e]);
            w[e] = mn == -INFINITY ? 1.f : ex2(m[mt][e] - mn);
            m[mt][e] = mn;
            l[mt][e] *= w[e];
          }
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][i][e] *= w[E == 1 ? 0 : e >> 1];
        }
        // Weights enter the product with v as two 16-bit terms, the rounded weight
        // and what the rounding left, so that neither o nor (summed in fp32) lse
        // loses to it. The second terms of 8 rows are the fragment's other 8.
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float ref = m[mt][e] == -INFINITY ? 0.f : kBias - m[mt][e];
#pragma unroll
          for (int i = 0; i < 2 * C::GROUPS; ++i) {
            const float x = ex2(fmaf(s[mt][i][2 * e], a.scale, ref));
            const float y = ex2(fmaf(s[mt][i][2 * e + 1], a.scale, ref));
            l[mt][e] += x + y;
            const uint32_t hi = pack16<BF>(x, y);
            const float2 r = unpack16<BF>(hi);
            const uint32_t lo = pack16<BF>(x - r.x, y - r.y);
            if (E == 1) {
              p[mt][i >> 1][2 * (i & 1)] = hi;
              p[mt][i >> 1][2 * (i & 1) + 1] = lo;
            } else {
              p[mt][i >> 1][2 * (i & 1) + e] = hi;
              p2[mt][i >> 1][2 * (i & 1) + e] = lo;
            }
          }
        }
      }
#pragma unroll
      for (int g = 0; g < C::GROUPS; ++g)
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          uint32_t f[4];
          ldsm4_t(f, (vb ^ (dt << 5)) + g * 16 * (D * 2));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16<BF>(o[mt][2 * dt], p[mt][g], f[0], f[1]);
            mma16<BF>(o[mt][2 * dt + 1], p[mt][g], f[2], f[3]);
          }
          if constexpr (E == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = finite16<BF>(f[i]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma16<BF>(o[mt][2 * dt], p2[mt][g], f[0], f[1]);
              mma16<BF>(o[mt][2 * dt + 1], p2[mt][g], f[2], f[3]);
            }
          }
        }
    }
    if (it + 1 < n_steps && (CLUSTER || at.t + 1 < at.nt)) {
      at.t += ranks;
      continue;
    }
    if constexpr (CLUSTER) break;

    // ---- the unit's end, or the stretch's ----
    const PagedAt done = at;
    if (it + 1 < n_steps) {   // the next unit's queries are on their way meanwhile
      next_unit<C::STEP>(a, at);
      load_q(at);
    }
    const bool whole = first_t == 0 && done.t + 1 == done.nt;
    merge_warps<D, E, MT>(smem + C::RING, s_ml, o, m, l, [&](int row, int col, const PartSum& x) {
      const int r = done.rt * ROWS + row;
      if (r >= group) return;
      if (whole) {
        store_part_sum<BF>(a, x, done.b, done.head * group + r, col);
      } else {
        const long long slot = (2ll * blockIdx.x + (first_t == 0)) * min(group, ROWS) + row;
        *reinterpret_cast<float4*>(a.part_o + slot * D + col) = x.o;
        if (col == 0) a.part_ml[slot] = make_float2(x.m, x.l);
      }
    });
    if (first_t == 0 && threadIdx.x == 0) line_record(a, line, done, whole, by_unit);
    first_t = 0;
    clear();
  }

  if constexpr (CLUSTER) {
    // this block's part into its shared memory (the ring: every load has landed
    // and been read), then every block adds up a share of the columns
    float* part = reinterpret_cast<float*>(smem);
    merge_warps<D, E, MT>(smem + C::RING, s_ml, o, m, l, [&](int row, int col, const PartSum& x) {
      *reinterpret_cast<float4*>(part + row * D + col) = x.o;
      if (col == 0) s_unit_ml[row] = make_float2(x.m, x.l);
    });
    cluster_sync();
    const int rows = min(ROWS, group - at.rt * ROWS), head0 = at.head * group + at.rt * ROWS;
    for (int i = rank * 128 + threadIdx.x; i < rows * (D / 4); i += ranks * 128) {
      const int row = i / (D / 4), col = i % (D / 4) * 4;
      const uint32_t po = smem_u32(part + row * D + col), pm = smem_u32(&s_unit_ml[row]);
      PartSum sum;
      for (int r0 = 0; r0 < ranks; r0 += 4) {   // ranks is a multiple of 4 or less than 4
        float4 x[4];
        float2 ml[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int from = min(r0 + r, ranks - 1);
          x[r] = cluster_load4(cluster_addr(po, from));
          ml[r] = cluster_load2(cluster_addr(pm, from));
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r0 + r < ranks) sum.add(ml[r], x[r]);
      }
      store_part_sum<BF>(a, sum, at.b, head0 + row, col);
    }
    cluster_sync();   // no block leaves while another reads its part
  }
}

// Adds the parts of the units that a border of paged_attn_kernel cut: block x
// takes record x, and blocks y the unit's columns in turn, `most` at a time. The
// parts are those of consecutive blocks, so in key order. A thread owns four
// columns of a row and some of the parts, four of them in flight with a running
// maximum; the threads of a column meet in shared memory.
constexpr int kJoinThreads = 256;

// Whether a record names a unit of the call and blocks of its launch. A block of
// paged_wide_kernel that gave up a wait leaves without its records, and a workspace
// does not start at zero: what is there instead must address nothing.
__host__ __device__ constexpr bool record_in_range(int unit, int first, int last, long long units, long long blocks) {
  return unit >= 0 && unit < units && first >= 0 && first <= last && last < blocks;
}

template <int D, bool BF>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedAttnArgs a, int row_tile, int most,
                                                                   int blocks) {
  __shared__ float4 s_o[kJoinThreads];
  __shared__ float2 s_ml[kJoinThreads];
  wait_for_prior_launch();
  const int4 record = a.split[blockIdx.x];
  if (!record_in_range(record.x, record.y, record.z, static_cast<long long>(a.B) * a.Hkv * a.row_tiles, blocks)) return;
  const int group = a.Hq / a.Hkv, rows = min(group, row_tile);
  const int rt = record.x % a.row_tiles, b = record.x / (a.row_tiles * a.Hkv);
  const int head0 = (record.x / a.row_tiles - b * a.Hkv) * group + rt * row_tile;
  const int first = record.y, n = record.z - record.y + 1;
  const int cols = min(rows, group - rt * row_tile) * (D / 4);
  // as many threads a column as give each up to four parts
  const int width = min(cols, most), parts = min(kJoinThreads / width, (n + 3) / 4);
  const int part = static_cast<int>(threadIdx.x) / width;
  for (int c0 = blockIdx.y * width; c0 < cols; c0 += gridDim.y * width) {
    const int c = c0 + static_cast<int>(threadIdx.x) % width, r = c / (D / 4), col = c % (D / 4) * 4;
    const bool mine = part < parts && c < cols;
    PartSum sum;
    if (mine) {
      // part i is the second partial result of the first block, the first one of the others
      for (int i0 = part; i0 < n; i0 += 4 * parts) {
        float2 ml[4];
        float4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = min(i0 + j * parts, n - 1);
          const long long slot = (2ll * (first + i) + (i == 0)) * rows + r;
          ml[j] = a.part_ml[slot];
          x[j] = *reinterpret_cast<const float4*>(a.part_o + slot * D + col);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i0 + j * parts < n) sum.add(ml[j], x[j]);
      }
      s_o[threadIdx.x] = sum.o;
      s_ml[threadIdx.x] = make_float2(sum.m, sum.l);
    }
    __syncthreads();
    if (mine && part == 0) {
      for (int p = 1; p < parts; ++p) sum.add(s_ml[p * width + threadIdx.x], s_o[p * width + threadIdx.x]);
      store_part_sum<BF>(a, sum, b, head0 + r, col);
    }
    __syncthreads();
  }
}

}  // namespace fab
