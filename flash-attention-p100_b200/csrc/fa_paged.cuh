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
constexpr int kTableThreads = 1024;

// What the second half of extend and release needs of a request.
struct alignas(16) TableRow {
  int tok;    // first token of the request in the call's packed tokens (extend)
  int page;   // first page of the request in the call's pages
  int len;    // length before the call
  int count;  // tokens granted (extend) or pages given back (release)
};
struct alignas(16) TableHead {
  int pages;  // pages the call takes or gives back
  int free;   // free pages before the call
  int pad[2];
};

__device__ __forceinline__ int clamp_count(int n, int P) { return min(max(n, 0), P); }

__device__ __forceinline__ int clip_int(long long x) {
  return x > 0x7fffffffll ? 0x7fffffff : static_cast<int>(x);
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
  if (warp == 0) {
    long long s = lane < static_cast<int>(blockDim.x >> 5) ? sums[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += y;
    }
    sums[lane] = s;
  }
  __syncthreads();
  *total = sums[31];
  return x + (warp ? sums[warp - 1] : 0);
}

// Last row of rows[0, B) whose member `tok` or `page` is <= x (row 0's is 0).
template <int TableRow::*M>
__device__ __forceinline__ int find_row(const TableRow* rows, int B, int x) {
  int lo = 0, hi = B;  // rows[lo] <= x, rows[hi] > x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (rows[mid].*M <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Which requests of an extend call are served and where their tokens and pages
// start: two running sums over the requests, in order, by one block.
//   e = sum of new tokens (served or not): the packed position of the tokens
//   c = sum of new pages of the requests that fit their row and the call
// A request is served if it needs no page or c <= free.
__device__ __forceinline__ void extend_rows(const int* new_lens, const int* lens, const int* free_count,
                                            int* granted, int* lens_out, int* free_out,
                                            TableHead* head, TableRow* rows, int B, int W, int P,
                                            int page, int T) {
  __shared__ long long sums[32];
  const int free = clamp_count(*free_count, P);
  const long long cap = static_cast<long long>(W) * page;
  long long tok0 = 0, page0 = 0;
  int taken = 0;
  for (int r0 = 0; r0 < B; r0 += kTableThreads) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    const int n = r < B ? max(new_lens[r], 0) : 0;
    const int len = r < B ? lens[r] : 0;
    long long all;
    const long long e = tok0 + block_sum(n, sums, &all);
    tok0 += all;
    const bool fits = n > 0 && len >= 0 && static_cast<long long>(len) + n <= cap && e <= T;
    const int p0 = fits ? (len + page - 1) / page : 0;
    const int want = fits ? static_cast<int>((static_cast<long long>(len) + n + page - 1) / page) - p0 : 0;
    const long long c = page0 + block_sum(want, sums, &all);
    page0 += all;
    const bool ok = fits && (want == 0 || c <= free);
    if (ok && want) taken = static_cast<int>(c);
    if (r < B) {
      rows[r] = TableRow{clip_int(e - n), clip_int(c - want), len, ok ? n : 0};
      granted[r] = ok ? n : 0;
      lens_out[r] = len + (ok ? n : 0);
    }
  }
  // pages taken: c of the last served request that takes any
  __shared__ int most;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  taken = __reduce_max_sync(0xffffffffu, taken);
  if ((threadIdx.x & 31) == 0) atomicMax(&most, taken);
  __syncthreads();
  if (threadIdx.x == 0) {
    *head = TableHead{most, free, {0, 0}};
    *free_out = free - most;
  }
}

// The slots of the call's tokens and the new entries of the block table, by
// threads `first`, `first + step`, ... of the launch. New entries lie behind
// the entries that this reads (a request's pages so far), so the order of the
// threads does not matter. A thread takes kSlotRun tokens in a row: one search.
constexpr int kSlotRun = 4;

__device__ __forceinline__ void extend_fill(const TableHead* head, const TableRow* rows, int* table,
                                            long long table_stride, const int* free_pages,
                                            int* slots, int B, int P, int page, int T,
                                            long long first, long long step) {
  const int free = head->free, pages = head->pages;
  for (long long t0 = first * kSlotRun; t0 < T; t0 += step * kSlotRun) {
    int r = find_row<&TableRow::tok>(rows, B, static_cast<int>(t0));
    TableRow row = rows[r];
#pragma unroll
    for (int i = 0; i < kSlotRun; ++i) {
      const int t = static_cast<int>(t0) + i;
      if (t0 + i >= T) break;
      while (r + 1 < B && rows[r + 1].tok <= t) row = rows[++r];
      int slot = -1;
      if (t - row.tok < row.count) {
        const int pos = row.len + t - row.tok, j = pos / page;
        const int fresh = j - (row.len + page - 1) / page;  // >= 0: a page of this call
        const int id = fresh >= 0 ? free_pages[free - 1 - row.page - fresh] : table[r * table_stride + j];
        if (static_cast<unsigned>(id) < static_cast<unsigned>(P)) slot = id * page + (pos - j * page);
      }
      slots[t] = slot;
    }
  }
  for (long long k = first; k < pages; k += step) {
    const int r = find_row<&TableRow::page>(rows, B, static_cast<int>(k));
    const TableRow row = rows[r];
    const int j = (row.len + page - 1) / page + static_cast<int>(k) - row.page;
    table[r * table_stride + j] = free_pages[free - 1 - k];
  }
}

// Which requests of a release call give pages back and where those start.
__device__ __forceinline__ void release_rows(const unsigned char* finished, const int* lens,
                                             const int* free_count, int* lens_out, int* free_out,
                                             TableHead* head, TableRow* rows, int B, int W, int P,
                                             int page) {
  __shared__ long long sums[32];
  const int free = clamp_count(*free_count, P);
  long long page0 = 0;
  for (int r0 = 0; r0 < B; r0 += kTableThreads) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    const bool done = r < B && finished[r] != 0;
    const int len = r < B ? lens[r] : 0;
    const int n = done ? (min(max(len, 0), W * page) + page - 1) / page : 0;
    long long all;
    const long long c = page0 + block_sum(n, sums, &all);
    page0 += all;
    if (r < B) {
      rows[r] = TableRow{0, clip_int(c - n), len, n};
      lens_out[r] = done ? 0 : len;
    }
  }
  if (threadIdx.x == 0) {
    // more pages than the stack has room for cannot come from one pool: the
    // rest are dropped
    const int back = static_cast<int>(min(page0, static_cast<long long>(P - free)));
    *head = TableHead{back, free, {0, 0}};
    *free_out = free + back;
  }
}

__device__ __forceinline__ void release_fill(const TableHead* head, const TableRow* rows,
                                             const int* table, long long table_stride,
                                             int* free_pages, int B, long long first, long long step) {
  const int free = head->free, pages = head->pages;
  for (long long k = first; k < pages; k += step) {
    const int r = find_row<&TableRow::page>(rows, B, static_cast<int>(k));
    free_pages[free + k] = table[r * table_stride + (k - rows[r].page)];
  }
}

struct ExtendArgs {
  const int *new_lens, *lens, *free_pages, *free_count;
  int *table, *slots, *granted, *lens_out, *free_out;
  long long table_stride;
  TableHead* head;
  TableRow* rows;
  int B, W, P, page, T;
};

__global__ void __launch_bounds__(kTableThreads) extend_kernel(const ExtendArgs a) {
  extend_rows(a.new_lens, a.lens, a.free_count, a.granted, a.lens_out, a.free_out, a.head, a.rows, a.B,
              a.W, a.P, a.page, a.T);
  __syncthreads();
  extend_fill(a.head, a.rows, a.table, a.table_stride, a.free_pages, a.slots, a.B, a.P, a.page, a.T,
              threadIdx.x, blockDim.x);
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

__global__ void __launch_bounds__(kTableThreads) release_kernel(const ReleaseArgs a) {
  release_rows(a.finished, a.lens, a.free_count, a.lens_out, a.free_out, a.head, a.rows, a.B, a.W, a.P,
               a.page);
  __syncthreads();
  release_fill(a.head, a.rows, a.table, a.table_stride, a.free_pages, a.B, threadIdx.x, blockDim.x);
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

// One 16-byte piece of k and of v per thread.
template <int D>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long row = i / (D / 8);
  if (row >= static_cast<long long>(a.T) * a.Hkv) return;
  const int c = static_cast<int>(i % (D / 8)) * 8;
  const int t = static_cast<int>(row / a.Hkv), h = static_cast<int>(row % a.Hkv);
  const int slot = a.slots[t];
  if (slot < 0 || slot >= a.P * a.page) return;
  const int id = slot / a.page, off = slot % a.page;
  *reinterpret_cast<uint4*>(a.k_cache + a.skc.at(id, h, off) + c) =
      *reinterpret_cast<const uint4*>(a.k + a.sk.at(0, h, t) + c);
  *reinterpret_cast<uint4*>(a.v_cache + a.svc.at(id, h, off) + c) =
      *reinterpret_cast<const uint4*>(a.v + a.sv.at(0, h, t) + c);
}

// ---------------------------------------------------------------------------
// attention of one new token per request
// ---------------------------------------------------------------------------
struct PagedAttnArgs {
  const uint16_t *q, *k_cache, *v_cache;
  uint16_t* o;
  float* lse;
  Strides sq, so, skc, svc;  // q, o: b request, h head; caches: b page, h head, n token
  const int *table, *lens;
  long long table_stride;
  int Hq, Hkv, P, W, page;
  float scale;  // log2(e) / sqrt(D)
  int* err;
};

template <bool BF>
__device__ __forceinline__ float2 unpack16(uint32_t x) {
  if (BF) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
template <bool BF>
__device__ __forceinline__ uint16_t round16(float x) {
  if (BF) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}

// One block per (request, query head); each warp takes every fourth key, each
// lane D/32 of its columns.
template <int D, bool BF>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedAttnArgs a) {
  constexpr int C = D / 32;
  const int b = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, kh = h / (a.Hq / a.Hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = min(max(a.lens[b], 0), a.W * a.page);
  float q[C], o[C] = {}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < C; i += 2) {
    const float2 x = unpack16<BF>(*reinterpret_cast<const uint32_t*>(a.q + a.sq.at(b, h, 0) + lane * C + i));
    q[i] = x.x;
    q[i + 1] = x.y;
  }
  for (int j = warp; j < len; j += 4) {
    const int id = a.table[b * a.table_stride + j / a.page];
    if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.P)) {
      if (lane == 0) atomicCAS(a.err, 0, static_cast<int>(kErrPage));
      continue;
    }
    const uint16_t* k = a.k_cache + a.skc.at(id, kh, j % a.page) + lane * C;
    const uint16_t* v = a.v_cache + a.svc.at(id, kh, j % a.page) + lane * C;
    float s = 0.f;
    for (int i = 0; i < C; i += 2) {
      const float2 x = unpack16<BF>(*reinterpret_cast<const uint32_t*>(k + i));
      s += q[i] * x.x + q[i + 1] * x.y;
    }
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.scale;
    const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;
    const float w = exp2f(m - ref), p = exp2f(s - ref);
    m = mn;
    l = l * w + p;
    for (int i = 0; i < C; i += 2) {
      const float2 x = unpack16<BF>(*reinterpret_cast<const uint32_t*>(v + i));
      o[i] = o[i] * w + p * x.x;
      o[i + 1] = o[i + 1] * w + p * x.y;
    }
  }
  __shared__ float so[4][D], sm[4], sl[4];
  for (int i = 0; i < C; ++i) so[warp][lane * C + i] = o[i];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, acc = 0.f;
  for (int w = 0; w < 4; ++w) {
    const float e = exp2f(sm[w] - ref);
    sum += sl[w] * e;
    if (threadIdx.x < D) acc += so[w][threadIdx.x] * e;
  }
  if (threadIdx.x < D)
    a.o[a.so.at(b, h, 0) + threadIdx.x] = round16<BF>(len ? acc / sum : 0.f);
  if (threadIdx.x == 0)
    a.lse[static_cast<long long>(b) * a.Hq + h] =
        len ? 0.6931471805599453f * (top + log2f(sum)) : -INFINITY;
}

}  // namespace fab
