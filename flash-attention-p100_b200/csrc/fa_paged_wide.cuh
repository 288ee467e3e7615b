// fa_paged_wide.cuh -- the paged cache's attention for wide groups of query heads
// (multi-query models; kPagedWarpHeads says which), on tcgen05.
//
// Such a group gives each cached byte enough work that mma.sync, at the few warps
// that accumulators in registers allow, is slower than HBM: paged_attn_kernel takes
// 85 us at 32 heads for a 0.27 GB cache, and reads the cache once for each 32 of
// them. Here a block walks its stretch of the same line in steps of 64 or 128 keys:
// S = Q K^T and O += P V as 128-row MMAs with O in tensor memory.
//
// Head h is row h / 4 of quadrant h % 4 of the tile: tensor memory gives a warp the
// lanes of one quadrant, and a quadrant's warps one scheduler, so few heads still
// keep all four schedulers' softmax warps busy. A warp has 16 of its quadrant's
// lanes: a thread has one head and half a step's keys, the thread 16 further on the
// other half (TMEM shape 16x32bx2). W is the number of softmax warps:
//
//   W = 4, up to 64 heads: steps of 64 keys, two blocks an SM, each of half its shared
//     and tensor memory, so that one's softmax runs beside the other's loads and
//     products (32 heads: 59.0 -> 56.0 us against one block and 128 keys). A unit's
//     heads take 16 lanes of each quadrant; the next unit's queries go into the other
//     16, whose products nobody reads meanwhile.
//   W = 8, 65 to 128 heads of a row tile: steps of 128 keys, one block, two Q tiles.
//
//   warps 0 .. W-1  queries, softmax, the unit's end
//   warp  W         MMA issue;  warp W + 1  TMA loads, a run of keys of one page each
// TMEM: two buffers of KEYS columns, S of a step and then its P over it, and O. S of
// step j + 2 is issued behind the products of step j, which the tensor core finishes
// first, so the softmax of a step waits for its S alone.
// Weights are two 16-bit terms and lse is summed in fp32, as in paged_attn_kernel;
// the terms' products stay apart so that an infinite value takes the first alone. At
// W = 4 P's second terms are the quadrant's other 16 rows and one product serves both
// (64-wide heads: 48.0 -> 43.3 us against a product of their own). At W = 8 they
// are columns [64,128) of P, and their products columns [384, 384 + D).
//
// Measured, the sequences of kPagedWarpHeads, for 32 / 64 / 128 heads: D = 128 55 / 60 /
// 79 us (4.9 / 4.5 / 3.5 TB/s), D = 64 38 / 40 / 55 us. About 7 us are the line's start
// and its join; at 32 heads HBM moves the rest at 5.6 TB/s, with a third of the issue
// slots and of the tensor pipe busy. At W = 8 the chain of one step after another
// (S, softmax, P) bounds it: tensor memory has no room for a second block's, or at
// D = 64 where it has, 10 warps of 96 registers are no faster (58 us).
#pragma once
#include "fa_fwd.cuh"
#include "fa_paged.cuh"

namespace fab {

template <int D, int W>
struct WideCfg {
  static constexpr bool PAIR = W == 4;           // two blocks an SM
  static constexpr int KEYS = PAIR ? 64 : 128;   // of a step
  static constexpr int CH = D / 64;              // 64-column chunks of a row
  static constexpr int CHUNK = KEYS * 128;       // bytes of a chunk of K or V
  static constexpr int Q = 128 * D * 2;          // bytes of 128 rows of queries
  static constexpr int TILE = KEYS * D * 2;      // of a step's K and of its V
  static constexpr int SLOTS = D == 128 ? 5 : 12;  // ring: K_0, V_0, K_1, V_1, ...
  static constexpr int OFF_RING = PAIR ? Q : 2 * Q;   // a unit's queries and the next one's
  static constexpr int SMEM = OFF_RING + SLOTS * TILE;
  static_assert(SMEM + 2048 <= (PAIR ? 233472 / 2 : 233472), "shared memory over the limit");
  static constexpr int FLAGS = 32;               // steps whose bad runs are kept
  static constexpr uint32_t COL_O = 2 * KEYS, COL_O2 = COL_O + 128, COLS = PAIR ? 256 : 512;
};

// Barriers; those of two are a step's (q: a unit's) by its parity, as its issue runs
// ahead of its use. S of step j + 1 comes behind the products of step j - 1 and stands
// for them, so those have barriers of their own only for the last step but one (pv)
// and where a unit or the stretch ends (end).
template <int SLOTS>
struct WideShared {
  uint64_t q[2], full[SLOTS], empty[SLOTS], s[2], p[2], pv, end, done;
  uint32_t tmem;
  int abort;
};

// The MMA warp stays whole: every lane runs its loop with the same values, and only
// the elected lane's instructions take effect, so that descriptors are computed in
// uniform registers. From inside a branch of one lane each MMA took 70 to 95 cycles to
// issue, whatever its size (64-wide heads, 128 of them: 60.2 -> 56.7 us).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t lead;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(lead));
  return lead;
}
__device__ __forceinline__ void mma_ss_lead(uint32_t lead, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts_lead(uint32_t lead, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}

// S (128 x KEYS) = Q (128 x D, K-major) K_step^T
template <int D, bool BF, int KEYS>
__device__ __forceinline__ void issue_qk_step(uint32_t lead, uint32_t d_tmem, uint32_t q_s, uint32_t k_s) {
  constexpr uint32_t idesc = idesc_f16(128, KEYS, false, false, BF);
  const uint64_t dq = sdesc_sw128(q_s, 16, 1024), dk = sdesc_sw128(k_s, 16, 1024);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    mma_ss_lead(lead, d_tmem, sdesc_add(dq, (kk >> 2) * 16384 + (kk & 3) * 32),
                sdesc_add(dk, (kk >> 2) * KEYS * 128 + (kk & 3) * 32), idesc, kk > 0 ? 1u : 0u);
}
// O (128 x D) (+)= P (128 x KEYS, pairs in tensor memory) V_step (MN-major)
template <int D, bool BF, int KEYS>
__device__ __forceinline__ void issue_pv_step(uint32_t lead, uint32_t d_tmem, uint32_t p_tmem, uint32_t v_s,
                                              bool accumulate) {
  constexpr uint32_t idesc = idesc_f16(128, D, false, true, BF);
  const uint64_t dv = sdesc_sw128(v_s, KEYS * 128, 1024);
#pragma unroll
  for (int kk = 0; kk < KEYS / 16; ++kk)
    mma_ts_lead(lead, d_tmem, p_tmem + kk * 8, sdesc_add(dv, kk * 2048), idesc, (accumulate || kk > 0) ? 1u : 0u);
}

// A tile's place in the ring: 2 j is K of step j, 2 j + 1 its V.
template <int SLOTS>
struct RingAt {
  int slot;
  uint32_t phase = 0;
  __device__ __forceinline__ void skip(int tiles) {   // at most SLOTS
    slot += tiles;
    if (slot >= SLOTS) {
      slot -= SLOTS;
      phase ^= 1;
    }
  }
};

// W softmax warps: 4 for groups of up to 64 heads, 8 above.
// `run_log2`: a run of 2^run_log2 keys lies in one page and is one box of tm_k, tm_v.
template <int D, bool BF, int W>
__global__ void __launch_bounds__(32 * (W + 2), WideCfg<D, W>::PAIR ? 2 : 1)
    paged_wide_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const PagedAttnArgs a, int run_log2) {
  using C = WideCfg<D, W>;
  constexpr int SOFTMAX = 32 * W, MMA_WARP = W, TMA_WARP = W + 1;
  constexpr int KEYS = C::KEYS;
  constexpr float kBias = weight_bias<BF>();
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ LineShared s_line;
  if (!smem_aligned_or_report(smem, a.err)) return;
  __shared__ WideShared<C::SLOTS> s_bar;
  __shared__ int s_bad[C::FLAGS];
  const uint32_t s_q = smem_u32(smem), s_ring = s_q + C::OFF_RING;
  const uint32_t b_q = smem_u32(s_bar.q), b_full = smem_u32(s_bar.full), b_empty = smem_u32(s_bar.empty);
  const uint32_t b_s = smem_u32(s_bar.s), b_p = smem_u32(s_bar.p), b_pv = smem_u32(&s_bar.pv),
                 b_end = smem_u32(&s_bar.end), b_done = smem_u32(&s_bar.done);
  volatile int* abort_flag = &s_bar.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.Hq / a.Hkv, units = a.Hkv * a.row_tiles;
  const bool by_unit = static_cast<long long>(a.B) * units <= gridDim.x;
  const Ctl ctl{abort_flag, a.err};

  wait_for_prior_launch();
  Line line;
  const long long n = line_begin<KEYS, D, 32 * (W + 2)>(a, units, by_unit, line, s_line);
  if (n == 0) return;
  if (threadIdx.x == 0) {
    mbar_init(b_q, SOFTMAX);
    mbar_init(b_q + 8, SOFTMAX);
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(b_full + 8 * s, 1);
      mbar_init(b_empty + 8 * s, 1);
    }
    mbar_init(b_s, 2);   // the products, and the issuer's word that K and its bad runs are there
    mbar_init(b_s + 8, 2);
    mbar_init(b_p, W);
    mbar_init(b_p + 8, W);
    mbar_init(b_pv, 1);
    mbar_init(b_end, 1);
    mbar_init(b_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == MMA_WARP) tmem_alloc(smem_u32(&s_bar.tmem), C::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_bar.tmem;
  PagedAt at = line_at<KEYS>(a, s_line);
  const auto advance = [&](PagedAt& x) {
    if (++x.t == x.nt) next_unit<KEYS>(a, x);
  };
  using Ring = RingAt<C::SLOTS>;

  if (warp == TMA_WARP) {
    // ------------------------------------------------------------ loads
    const int runs = KEYS >> run_log2;   // 1 to 8, one a lane
    int id = 0, off = 0;
    const auto look_up = [&](const PagedAt& x) {
      const int key = x.t * KEYS + (lane << run_log2);
      const int page = key / a.page;
      off = key - page * a.page;
      // behind the last token: a page outside the cache, which loads as zeros
      id = lane < runs && key < x.len ? a.table[x.b * a.table_stride + page] : a.P;
    };
    look_up(at);
    Ring tile{0};
    long long issued = 0;
    bool ok = true;
    for (long long j = 0; j < n && ok; ++j) {
      const bool real = lane < runs && at.t * KEYS + (lane << run_log2) < at.len;
      const bool bad = real && static_cast<unsigned>(id) >= static_cast<unsigned>(a.P);
      const int page = bad ? a.P : id, row = off, head = at.head;
      const unsigned bad_runs = __ballot_sync(0xffffffffu, bad);
      if (bad_runs && lane == 0) atomicCAS(a.err, 0, static_cast<int>(kErrPage));
      if (j + 1 < n) {   // the next step's pages are on their way meanwhile
        advance(at);
        look_up(at);
      }
#pragma unroll
      for (int kind = 0; kind < 2 && ok; ++kind) {
        const int slot = tile.slot;
        const uint32_t full = b_full + 8 * slot;
        ok = lane != 0 || mbar_wait(b_empty + 8 * slot, tile.phase ^ 1, ctl, kErrTimeoutLoad);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          if (kind == 0) s_bad[j % C::FLAGS] = static_cast<int>(bad_runs);
          mbar_arrive_expect_tx(full, C::TILE);
        }
        __syncwarp();
        if (lane < runs) {
          const uint32_t dst = s_ring + slot * C::TILE + (lane << run_log2) * 128;
#pragma unroll
          for (int c = 0; c < C::CH; ++c)
            tma_load_4d(dst + c * C::CHUNK, kind ? static_cast<const void*>(&tm_v) : static_cast<const void*>(&tm_k),
                        full, c * 64, row, head, page);
        }
        tile.skip(1);
        ++issued;
      }
    }
    if (!ok && lane == 0) {
      // loads in flight land before the block leaves: the last SLOTS of them
      const int last = static_cast<int>(issued < C::SLOTS ? issued : C::SLOTS);
      Ring i = tile;
      i.slot -= last;
      if (i.slot < 0) {
        i.slot += C::SLOTS;
        i.phase ^= 1;
      }
      for (int k = 0; k < last; ++k, i.skip(1)) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(b_full + 8 * i.slot, i.phase) && globaltimer_ns() - t0 < 100000000ull) {
        }
      }
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------------------ MMA issue
    __syncwarp();
    const uint32_t lead = elect_one(), tmem0 = __shfl_sync(0xffffffffu, tmem, 0);
    const long long steps = __shfl_sync(0xffffffffu, n, 0);
    const auto wait = [&](uint32_t bar, uint32_t parity) {
      const bool ok = mbar_wait(bar, parity, ctl, kErrTimeoutMma);
      return static_cast<bool>(__all_sync(0xffffffffu, ok));
    };
    const auto commit = [&](uint32_t bar) {
      if (lead) mma_commit(bar);
    };
    Ring k{0}, v{1};
    // S of the next step; `ahead` is its place, `unit` its unit of the stretch,
    // whose Q is in buffer unit & 1
    PagedAt ahead = at;
    int unit = 0;
    bool new_unit = true;
    const auto next_s = [&](int buf) -> bool {
      if (new_unit && !wait(b_q + 8 * (unit & 1), (unit >> 1) & 1)) return false;
      if (!wait(b_full + 8 * k.slot, k.phase)) return false;
      tc_fence_after();
      issue_qk_step<D, BF, KEYS>(lead, tmem0 + KEYS * buf, C::PAIR ? s_q : s_q + (unit & 1) * C::Q,
                                 s_ring + k.slot * C::TILE);
      commit(b_s + 8 * buf);
      if (lead) mbar_arrive(b_s + 8 * buf);
      commit(b_empty + 8 * k.slot);
      k.skip(2);
      new_unit = __any_sync(0xffffffffu, ahead.t + 1 == ahead.nt);
      if (new_unit) ++unit;
      return true;
    };
    bool ok = next_s(0);
    if (ok && steps > 1) {
      advance(ahead);
      ok = next_s(1);
    }
    bool first = true;       // the unit's first step here: O starts over
    for (long long j = 0; j < steps && ok; ++j) {
      ok = wait(b_full + 8 * v.slot, v.phase) && wait(b_p + 8 * (j & 1), (j >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      const uint32_t p = tmem0 + KEYS * (j & 1);
      issue_pv_step<D, BF, KEYS>(lead, tmem0 + C::COL_O, p, s_ring + v.slot * C::TILE, !first);
      if (!C::PAIR)
        issue_pv_step<D, BF, KEYS>(lead, tmem0 + C::COL_O2, p + KEYS / 2, s_ring + v.slot * C::TILE, !first);
      first = __any_sync(0xffffffffu, at.t + 1 == at.nt);
      if (j + 2 == steps) commit(b_pv);
      if (first || j + 1 == steps) commit(b_end);
      commit(b_empty + 8 * v.slot);
      v.skip(2);
      if (j + 1 < steps) advance(at);
      if (j + 2 < steps) {
        advance(ahead);
        ok = next_s(j & 1);
      }
    }
    // every MMA issued above completes before tensor memory is released
    commit(b_done);
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(b_done, 0) && globaltimer_ns() - t0 < FAB_WAIT_LIMIT_NS) {
    }
  } else {
    // ------------------------------------------------------------ softmax
    constexpr int PER = KEYS / 2;   // keys a thread
    const int half = lane >> 4;
    const int head_row = 4 * (16 * (warp >> 2) + (lane & 15)) + (warp & 3);   // this thread's head in the tile
    const uint32_t quad = tmem + (static_cast<uint32_t>(32 * (warp & 3) + 16 * (warp >> 2)) << 16);
    const auto wait = [&](uint32_t bar, uint32_t parity) {
      const bool ok = mbar_wait(bar, parity, ctl, kErrTimeoutSoftmax);
      return static_cast<bool>(__all_sync(0xffffffffu, ok));
    };
    // a unit's queries, half a row a thread; rows without a head are zero
    const auto load_q = [&](const PagedAt& x, int buf) {
      constexpr int HEADS = 16 * W, PIECES = D / 16;
      const int i = threadIdx.x % HEADS, c0 = static_cast<int>(threadIdx.x) / HEADS * PIECES;
      const int quadrant = i / (HEADS / 4), at_row = i % (HEADS / 4);
      const int r = x.rt * 128 + 4 * at_row + quadrant;
      const bool real = r < group;
      const uint16_t* q = a.q + a.sq.at(x.b, x.head * group + (real ? r : 0), 0) + c0 * 8;
      uint4 piece[PIECES];
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
        piece[c] = real ? *reinterpret_cast<const uint4*>(q + c * 8) : make_uint4(0, 0, 0, 0);
      const int row = 32 * quadrant + (C::PAIR ? 16 * buf : 0) + at_row;
      const uint32_t tile = C::PAIR ? s_q : s_q + buf * C::Q;
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
        st_shared_v4(tile + sw128_offset(row, c0 + c, 128), piece[c].x, piece[c].y, piece[c].z, piece[c].w);
      fence_async_smem();
      mbar_arrive(b_q + 8 * buf);
    };
    load_q(at, 0);
    float m = -INFINITY, l = 0.f;
    int unit = 0, first_t = at.t;
    bool ok = true, first = true;   // first: of the unit here, whose Q is in buffer unit & 1
    Ring v{1};
    for (long long j = 0; j < n && ok; ++j, v.skip(2)) {
      const long long left_here = n - j;
      if (first && at.nt - at.t < left_here) {   // the next unit's queries
        PagedAt x = at;
        next_unit<KEYS>(a, x);
        load_q(x, (unit + 1) & 1);
      }
      // a pair's units take the two halves of each quadrant's lanes in turn
      const uint32_t t_hi = C::PAIR ? quad + ((unit & 1) << 20) : quad, t_lo = C::PAIR ? t_hi ^ (1u << 20) : quad;
      const uint32_t t_s = t_hi + KEYS * (j & 1), t_p2 = C::PAIR ? t_lo + KEYS * (j & 1) : t_s + KEYS / 2;
      const uint32_t t_o = t_hi + C::COL_O, t_o2 = t_lo + (C::PAIR ? C::COL_O : C::COL_O2);
      ok = wait(b_s + 8 * (j & 1), (j >> 1) & 1);
      if (!ok) break;
      const unsigned bad = static_cast<unsigned>(s_bad[j % C::FLAGS]);
      tc_fence_after();
      uint32_t sr[PER];   // keys PER half ..
      if constexpr (PER == 64) tmem_ld16x2_x64(t_s, sr);
      else tmem_ld16x2_x32(t_s, sr);
      tmem_ld_wait(sr);
      float* s = reinterpret_cast<float*>(sr);
      const int left = at.len - at.t * KEYS;   // keys of this step, if below KEYS
      if (left < KEYS || bad) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int key = PER * half + i;
          if (key >= left || (bad >> (key >> run_log2) & 1)) s[i] = -INFINITY;
        }
      }
      float top = fmaxf(s[0], s[1]);
#pragma unroll
      for (int i = 2; i < PER; i += 2) top = max3f(top, s[i], s[i + 1]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) * a.scale;
      float w = 1.f;
      bool rescale = false;
      if (first) {
        m = top;
      } else {
        const bool grown = top > m + 8.f;
        rescale = __any_sync(0xffffffffu, grown);
        if (grown) {
          w = ex2(m - top);   // 0 from -inf; the products so far are then 0
          m = top;
          l *= w;
        }
      }
      const float ref = m == -INFINITY ? 0.f : kBias - m;
      uint32_t hi[PER / 2], lo[PER / 2];   // keys 2 i, 2 i + 1 of this thread's
      const uint64_t scale2 = f32x2(a.scale, a.scale), ref2 = f32x2(ref, ref), minus = f32x2(-1.f, -1.f);
      uint64_t sum[2] = {f32x2(0.f, 0.f), f32x2(0.f, 0.f)};
#pragma unroll
      for (int i = 0; i < PER / 2; ++i) {
        const float2 e = f32x2_split(fma_x2(f32x2(s[2 * i], s[2 * i + 1]), scale2, ref2));
        const float x = ex2(e.x), y = ex2(e.y);
        const uint64_t xy = f32x2(x, y);
        sum[i & 1] = add_x2(sum[i & 1], xy);
        hi[i] = pack2<BF>(x, y);
        const float2 r = unpack2<BF>(hi[i]), rest = f32x2_split(fma_x2(f32x2(r.x, r.y), minus, xy));
        lo[i] = pack2<BF>(rest.x, rest.y);
      }
      const float2 both = f32x2_split(add_x2(sum[0], sum[1]));
      l += both.x + both.y;
      __syncwarp();
      if (rescale) {   // O is free once the products of the step before are done
        ok = j + 1 < n ? wait(b_s + 8 * ((j + 1) & 1), ((j + 1) >> 1) & 1) : wait(b_pv, 0);
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int i = 0; i < 2 * (D / 64); ++i) {   // this thread's half of every 64 columns
          const uint32_t col = i < D / 64 ? t_o + 64 * i : t_o2 + 64 * (i - D / 64);
          uint32_t o[32];
          tmem_ld16x2_x32(col, o);
          tmem_ld_wait(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * w);
          tmem_st16x2_x32(col, o);
        }
      }
      if constexpr (PER == 64) {
        tmem_st16x2_x32(t_s, hi);
        tmem_st16x2_x32(t_p2, lo);
      } else {
        tmem_st16x2_x16(t_s, hi);
        tmem_st16x2_x16(t_p2, lo);
      }
      if (left < KEYS) {
        // values behind the last token in its run: 0 weights must not meet NaN
        ok = wait(b_full + 8 * v.slot, v.phase);
        if (!ok) break;
        const int end = (((left - 1) >> run_log2) + 1) << run_log2;
        const uint32_t rows = s_ring + v.slot * C::TILE;
        for (int i = threadIdx.x; i < (end - left) * 8 * C::CH; i += SOFTMAX) {
          const int r = left + i / (8 * C::CH), c = i % (8 * C::CH);
          st_shared_v4(rows + (c >> 3) * C::CHUNK + r * 128 + ((c & 7) << 4), 0, 0, 0, 0);
        }
        fence_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(b_p + 8 * (j & 1));
      const bool ends = at.t + 1 == at.nt;
      if (!ends && j + 1 < n) {
        ++at.t;
        first = false;
        continue;
      }

      // ---- the unit's end, or the stretch's ----
      ok = wait(b_end, unit & 1);
      if (!ok) break;
      tc_fence_after();
      const bool whole = first_t == 0 && ends;
      const int r = at.rt * 128 + head_row;
      PartSum part;
      part.m = m;
      part.l = l + __shfl_xor_sync(0xffffffffu, l, 16);
      const long long slot = (2ll * blockIdx.x + (first_t == 0)) * min(group, 128) + head_row;
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
        uint32_t o[32], o2[32];
        tmem_ld16x2_x32(t_o + 64 * c, o);
        tmem_ld16x2_x32(t_o2 + 64 * c, o2);
        tmem_ld_wait(o);
        tmem_ld_wait(o2);
        if (r < group) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const auto x = [&](int e) { return add_finite(__uint_as_float(o[i + e]), __uint_as_float(o2[i + e])); };
            const int col = 64 * c + 32 * half + i;
            part.o = make_float4(x(0), x(1), x(2), x(3));
            if (whole) {
              store_part_sum<BF>(a, part, at.b, at.head * group + r, col);
            } else {
              *reinterpret_cast<float4*>(a.part_o + slot * D + col) = part.o;
              if (col == 0) a.part_ml[slot] = make_float2(part.m, part.l);
            }
          }
        }
        __syncwarp();
      }
      if (first_t == 0 && threadIdx.x == 0) line_record(a, line, at, whole, by_unit);
      if (j + 1 < n) next_unit<KEYS>(a, at);
      ++unit;
      first_t = 0;
      first = true;
      l = 0.f;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) {
    __syncwarp();
    tmem_dealloc(tmem, C::COLS);
  }
}

}  // namespace fab
