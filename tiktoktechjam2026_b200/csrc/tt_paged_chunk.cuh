// Attention of longer chunks over a paged K/V cache on the tensor cores
// (sm_100a); parameters, schedule and the joining of cut items are in
// tt_paged_attn.cuh.
//
// One CTA per SM is one worker.  An item is two tiles ("halves") of up to 128
// query rows each (one at head_dim 256); a row is (token, head of the KV
// head's group), so grouped heads share every K and V tile.  Both halves read
// the same ring of K and V tiles, which one producer warp fills: each page, or
// the part of it inside the tile, is one TMA box per 64 features, and a page
// that does not exist is fetched out of bounds, i.e. as zeros.  Each half has
// 4 softmax warps (a whole row per thread) and its own MMA-issuing warp:
//   S = Q K^T         TMEM, BN FP32 columns, NSB buffers per half
//   P = 2^(S - m)     FP16/BF16 pairs written over the S it came from
//   O += P V          P from TMEM, V as it lies in the page (MN-major operand)
// The softmax is the bound below head_dim 128 (one exponential per score), so
// part of the exponentials runs as a polynomial on the FMA pipe, the reference
// maximum m moves only when a tile exceeds it by 2^8 (then O and l are
// rescaled), and S runs up to NSB - 1 tiles ahead.  At head_dim 128 the tensor
// core bounds it: key tiles of 128 keep the Q operand's shared-memory reads at
// the rate of the MMA (64-wide ones read 1.5 times what the pipe can fetch).
// A half skips the tiles that none of its rows sees.
// The rows of V past a sequence's end in its last page may hold anything
// (0 * NaN would reach the sum): a spare warp zeroes them in shared memory.
#pragma once

#include <type_traits>

#include "tt_attention.cuh"  // max3
#include "tt_paged_attn.cuh"

namespace tt {

template <int HD>
struct PagedChunkLayout {
  static constexpr int NT = HD == 256 ? 1 : 2;      // halves
  static constexpr int ROWS = 128 * NT;             // rows of a workspace slot
  static constexpr int BN = HD == 128 ? 128 : 64;   // keys per tile
  static constexpr int NSB = HD == 128 ? 1 : 3;     // S buffers per half
  static constexpr int NSK = HD == 128 ? 3 : HD == 256 ? 2 : 6;  // K and V tiles in the ring
  static constexpr int NSV = HD == 128 ? 2 : HD == 256 ? 2 : 6;
  static constexpr int NQ = HD >= 128 ? 1 : 2;      // Q tile buffers per half
  static constexpr int NOB = HD <= 32 ? 2 : 1;      // O buffers per half
  static constexpr int ATOM = HD >= 64 ? 64 : HD;   // features per swizzle atom
  static constexpr int NATOM = HD / ATOM;
  static constexpr int ROW = ATOM * 2;              // bytes of an atom's row
  static constexpr int Q_ATOM = 128 * ROW, KV_ATOM = BN * ROW;
  static constexpr int Q_BYTES = NATOM * Q_ATOM, KV_BYTES = NATOM * KV_ATOM;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = NT * NQ * Q_BYTES;
  static constexpr int OFF_V = OFF_K + NSK * KV_BYTES;
  static constexpr int OFF_BAR = OFF_V + NSV * KV_BYTES;
  // Barriers: K full/empty, V full/empty/fixed, then per half Q full/empty,
  // S full, P full, PV done, O full/free, done.
  static constexpr int B_KF = 0, B_KE = NSK, B_VF = 2 * NSK, B_VE = B_VF + NSV, B_VX = B_VE + NSV, B_HALF = B_VX + NSV;
  static constexpr int H_QF = 0, H_QE = 2, H_SF = 4, H_PF = H_SF + NSB, H_PE = H_PF + NSB, H_OF = H_PE + NSB,
                       H_OR = H_OF + 2, H_DONE = H_OR + 2, N_HALF = H_DONE + 1;
  static constexpr int OFF_MISC = OFF_BAR + (B_HALF + NT * N_HALF) * 8;
  static constexpr int SMEM = OFF_MISC + 16 + 1024;
  static constexpr int TMEM_COLS = 512, TMEM_O = NSB * BN, TMEM_HALF = 512 / NT;
  static constexpr int W_PROD = 4 * NT, W_FIX = W_PROD + 1, W_MMA = W_PROD + 2;  // MMA warps: W_MMA + half
  static constexpr int NWARPS = NT == 2 ? 12 : 8;
  static constexpr int THREADS = 32 * NWARPS;
  // Register split (setmaxnreg): the launch provides THREADS x REGS_LAUNCH and
  // the launcher refuses to start a kernel built with another count (a split
  // above the launch total would make setmaxnreg.inc wait forever).  The MMA
  // warps carry two walks of the piece, the softmax warps a row of BN scores.
  static constexpr bool SPLIT = NT == 2;
  static constexpr int REGS_LAUNCH = 168;
  static constexpr int REGS_SOFTMAX = BN == 128 ? 208 : 184, REGS_OTHER = BN == 128 ? 88 : 136;
  static_assert(!SPLIT || 128 * NT * REGS_SOFTMAX + 32 * (NWARPS - 4 * NT) * REGS_OTHER <= THREADS * REGS_LAUNCH,
                "register split");
  static_assert(TMEM_O + NOB * HD <= TMEM_HALF, "TMEM budget");
  static_assert(SMEM <= 232448, "shared memory budget");
  static_assert(Q_BYTES % 1024 == 0 && KV_BYTES % 1024 == 0 && OFF_BAR % 1024 == 0, "alignment");
};

// MN-major operand (V as stored: a row per key): atoms of ATOM features lie
// `lbo` bytes apart, groups of 8 keys `sbo` bytes.
__device__ __forceinline__ uint64_t umma_sdesc_mn(uint32_t saddr, uint32_t lbo, uint32_t sbo, uint32_t swz) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(swz & 0x7u) << 61;
  return d;
}

// Instruction descriptor of kind::f16 with an FP32 accumulator: BF16 operands
// set the A and B formats (bits 7 and 10), an MN-major B sets bit 16.
__host__ __device__ constexpr uint32_t umma_idesc_16(int M, int N, bool bf16, bool b_mn) {
  return umma_idesc_f16_f32(M, N) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}

// 2^x of a pair on the FMA pipe for any x: exp2_pair_fma_y (tt_ptx.cuh) with a
// wider clamp, y = saturate((x + 126) / 256), because BF16 and the FP32 row
// sum keep what FP16 rounds to zero.  The rounding of y costs 2^-17 in x.
constexpr float kExpYScale = 1.0f / 256.0f;
constexpr float kExpYBias = 126.0f / 256.0f;
__device__ __forceinline__ uint64_t exp2_pair_wide(uint64_t yy) {
  constexpr float kShift = 12582912.f - 126.f;  // 1.5*2^23 - 126, exact in FP32
  const uint64_t s256 = f2_pack(256.f, 256.f);
  const uint64_t t = ffma2(yy, s256, f2_pack(kShift, kShift));                // 1.5*2^23 + j
  const uint64_t u = ffma2(t, f2_pack(-1.f, -1.f), f2_pack(kShift, kShift));  // -126 - j, exact
  const uint64_t f = ffma2(yy, s256, u);                                      // x - j
  uint64_t q = ffma2(f2_pack(5.517162383e-02f, 5.517162383e-02f), f, f2_pack(2.426111251e-01f, 2.426111251e-01f));
  q = ffma2(q, f, f2_pack(6.932609677e-01f, 6.932609677e-01f));
  q = ffma2(q, f, f2_pack(9.999280572e-01f, 9.999280572e-01f));
  const uint32_t r0 = static_cast<uint32_t>(q) + (static_cast<uint32_t>(t) << 23);
  const uint32_t r1 = static_cast<uint32_t>(q >> 32) + (static_cast<uint32_t>(t >> 32) << 23);
  return (static_cast<uint64_t>(r1) << 32) | r0;
}

__device__ __forceinline__ uint32_t bits_below(int x) {  // the lowest x bits (none below 0, all from 32)
  return x >= 32 ? ~0u : (x <= 0 ? 0u : (1u << x) - 1u);
}

// The tiles of an item that some row of one half sees, as ranges of the item's
// tile index: [0, a) and [c, e).
struct ChunkRange {
  int a, c, e;
  __device__ __forceinline__ bool has(int i) const { return i < a || (i >= c && i < e); }
  // Last such tile of [i0, i1), or -1.
  __device__ __forceinline__ int last(int i0, int i1) const {
    const int y = min(e, i1) - 1;
    if (y >= max(c, i0)) return y;
    const int x = min(a, i1) - 1;
    return x >= i0 ? x : -1;
  }
};

// Walks a worker's piece segment by segment (a segment is the part of one item
// that lies in the piece) for one half.
template <int HD>
struct ChunkWalk {
  using L = PagedChunkLayout<HD>;
  static constexpr int BN = L::BN;
  PagedCursor<BN> cur;
  int left;        // units of the piece from this segment on
  int i0, i1;      // the segment's tiles
  int rows;        // rows of this half
  int p0, p1;      // positions of its first and last row
  ChunkRange range;
  int last;        // its last tile in the segment, -1: none
  __device__ __forceinline__ void load(const PagedParams& p, int half, int half_tokens) {
    const int hr = half_tokens * p.group;
    i0 = cur.i;
    i1 = min(cur.it.n, i0 + left);
    rows = min(max(cur.it.rows - half * hr, 0), hr);
    range = {0, 0, 0};
    last = -1;
    if (rows == 0) return;
    p0 = cur.it.p0 + half * half_tokens;
    p1 = cur.it.p0 + half * half_tokens + (rows - 1) / p.group;
    const int end = p1 < 0 ? 0 : p1 / BN + 1;  // one past the last tile a row sees
    if (p.window == 0) {
      range.e = end;
    } else {
      const int from = max(p0 - p.window + 1, 0) / BN;  // first tile in the window
      const int sink = (min(p.sinks, BN * end) + BN - 1) / BN;
      if (cur.it.n_sink == cur.it.n) {  // no gap: the index is the tile
        range.a = min(sink, end);
        range.c = max(from, range.a);
        range.e = end;
      } else {
        range.a = min(cur.it.n_sink, end);
        range.c = max(from - cur.it.w_tile, 0) + cur.it.n_sink;
        range.e = end - cur.it.w_tile + cur.it.n_sink;
      }
    }
    last = range.last(i0, i1);
  }
  // The next segment; false at the end of the piece.
  __device__ __forceinline__ bool next(const PagedParams& p, int half, int half_tokens, int rpt) {
    left -= i1 - i0;
    if (left <= 0) return false;
    cur.next_item(p, rpt);
    load(p, half, half_tokens);
    return true;
  }
};

// Exponentials per 8 pairs on the FMA pipe.
template <int HD>
constexpr int kChunkExpFma = HD <= 32 ? 3 : 2;

template <typename T, int HD>
__global__ void __launch_bounds__(PagedChunkLayout<HD>::THREADS, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const PagedParams p, int half_tokens,
                       long long min_units) {
  using L = PagedChunkLayout<HD>;
  using PT = Pair16<T>;
  constexpr int BN = L::BN, NT = L::NT, NSB = L::NSB, NSK = L::NSK, NSV = L::NSV, NQ = L::NQ, NOB = L::NOB;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PagedStart start;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half_rows = half_tokens * p.group, rpt = NT * half_rows;
  long long total, per;
  paged_schedule<BN, 1, L::THREADS>(p, rpt, min_units, blockIdx.x, &start, &total, &per);
  paged_zero_outside(p, L::THREADS);
  if (start.b < 0) return;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  if (threadIdx.x == 0) {
    for (int i = 0; i < NSK; ++i) {
      mbar_init(&bars[L::B_KF + i], 1);
      mbar_init(&bars[L::B_KE + i], NT);
    }
    for (int i = 0; i < NSV; ++i) {
      mbar_init(&bars[L::B_VF + i], 1);
      mbar_init(&bars[L::B_VE + i], NT + 1);  // the MMA warps and the warp that zeroes stale rows
      mbar_init(&bars[L::B_VX + i], 1);
    }
    for (int h = 0; h < NT; ++h) {
      uint64_t* b = bars + L::B_HALF + h * L::N_HALF;
      for (int i = 0; i < 2; ++i) {
        mbar_init(&b[L::H_QF + i], 1);
        mbar_init(&b[L::H_QE + i], 1);
        mbar_init(&b[L::H_OF + i], 1);
        mbar_init(&b[L::H_OR + i], 4);
      }
      for (int i = 0; i < NSB; ++i) {
        mbar_init(&b[L::H_SF + i], 1);
        mbar_init(&b[L::H_PF + i], 4);
        mbar_init(&b[L::H_PE + i], 1);
      }
      mbar_init(&b[L::H_DONE], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == L::W_MMA) {
    tmem_alloc(tmem_slot, L::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const Watchdog wd{p.err, abort_flag, p.timeout_ns};
  const int n_units = static_cast<int>(min(per, total - blockIdx.x * per));
  const int page_rows = 1 << p.page_shift;
  ChunkWalk<HD> walk;

  if (warp == L::W_PROD) {
    // -------------------------------------------------------------- producer
    if constexpr (L::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_OTHER));
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const int box = min(page_rows, BN), n_box = BN / box;  // boxes of a tile: lane i fetches the i-th
    int u = 0, nq[NT] = {};
    bool ok = true;
    walk.cur.seek(p, start.b, start.off, rpt);
    walk.left = n_units;
    walk.load(p, 0, half_tokens);
    do {
#pragma unroll
      for (int h = 0; h < NT; ++h) {
        walk.load(p, h, half_tokens);
        if (walk.last < 0) continue;
        uint64_t* b = bars + L::B_HALF + h * L::N_HALF;
        const int qb = nq[h] % NQ;
        if (lane == 0) ok = wait_phase(&b[L::H_QE + qb], ((nq[h] / NQ) & 1) ^ 1, wd, 0x531);
        if (!(ok = __shfl_sync(~0u, ok, 0))) break;
        if (lane == 0) {
          const int tok = walk.cur.s.q0 + walk.cur.it.r0 / p.group + h * half_tokens;
          mbar_arrive_expect_tx(&b[L::H_QF + qb], L::NATOM * half_rows * L::ROW);
#pragma unroll
          for (int a = 0; a < L::NATOM; ++a)
            tma_load_3d(smem + L::OFF_Q + (h * NQ + qb) * L::Q_BYTES + a * L::Q_ATOM, &tmQ, &b[L::H_QF + qb],
                        a * L::ATOM, walk.cur.kvh * p.group, tok);
        }
        ++nq[h];
      }
      if (!ok) break;
      const int* row = p.tables + walk.cur.s.slot * p.table_stride;
      const int n_keys = walk.cur.s.L;
      // The page of this lane's box of tile i (n_pages, past the end, where there is none).
      auto page_of = [&](int i) -> int {
        const int key = walk.cur.it.tile(i) * BN + lane * box;
        int pg = -1;
        if (lane < n_box && key < n_keys) pg = row[key >> p.page_shift];
        return pg < 0 || pg >= p.n_pages ? p.n_pages : pg;
      };
      int page = page_of(walk.i0);
      for (int i = walk.i0; i < walk.i1; ++i, ++u) {
        const int next = i + 1 < walk.i1 ? page_of(i + 1) : 0;  // a tile ahead: its latency is off the path
        const int at = walk.cur.kvh * page_rows + ((walk.cur.it.tile(i) * BN + lane * box) & (page_rows - 1));
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int st = u % (kv ? NSV : NSK), ph = u / (kv ? NSV : NSK);
          uint64_t* full = &bars[(kv ? L::B_VF : L::B_KF) + st];
          if (lane == 0) {
            ok = wait_phase(&bars[(kv ? L::B_VE : L::B_KE) + st], (ph & 1) ^ 1, wd, 0x532 + kv);
            if (ok) mbar_arrive_expect_tx(full, L::KV_BYTES);
          }
          if (!(ok = __shfl_sync(~0u, ok, 0))) break;
          if (lane < n_box) {
            uint8_t* dst = smem + (kv ? L::OFF_V : L::OFF_K) + st * L::KV_BYTES + lane * box * L::ROW;
#pragma unroll
            for (int a = 0; a < L::NATOM; ++a)
              tma_load_3d(dst + a * L::KV_ATOM, kv ? &tmV : &tmK, full, a * L::ATOM, at, page);
          }
          __syncwarp();
        }
        if (!ok) break;
        page = next;
      }
    } while (ok && walk.next(p, 0, half_tokens, rpt));
    // Let every copy this warp started land before the CTA may exit.
    if (lane == 0) {
      for (int h = 0; h < NT; ++h)
        for (int i = max(nq[h] - NQ, 0); i < nq[h]; ++i)
          wait_drain(&bars[L::B_HALF + h * L::N_HALF + L::H_QF + i % NQ], (i / NQ) & 1, kDrainLimitNs);
      for (int i = max(u - NSK, 0); i < u; ++i) wait_drain(&bars[L::B_KF + i % NSK], (i / NSK) & 1, kDrainLimitNs);
      for (int i = max(u - NSV, 0); i < u; ++i) wait_drain(&bars[L::B_VF + i % NSV], (i / NSV) & 1, kDrainLimitNs);
    }
  } else if (warp == L::W_FIX) {
    // -------------------------------------------------------------- zeroes the stale rows of V
    if constexpr (L::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_OTHER));
    int u = 0;
    bool ok = true;
    walk.cur.seek(p, start.b, start.off, rpt);
    walk.left = n_units;
    walk.load(p, 0, half_tokens);
    do {
      const int n_keys = walk.cur.s.L;
      for (int i = walk.i0; i < walk.i1; ++i, ++u) {
        const int st = u % NSV, k0 = walk.cur.it.tile(i) * BN;
        if (!(ok = warp_wait_phase(&bars[L::B_VF + st], (u / NSV) & 1, wd, 0x534))) break;
        const int r0 = n_keys - k0;
        const int r1 = ((r0 + page_rows - 1) & ~(page_rows - 1));  // k0 or the tile is a whole number of pages
        if (r0 > 0 && r0 < BN && r1 > r0) {
          const uint32_t base = smem_u32(smem + L::OFF_V + st * L::KV_BYTES);
          for (int a = 0; a < L::NATOM; ++a)
            for (int x = r0 * L::ROW + lane * 16; x < min(r1, BN) * L::ROW; x += 512)
              st_shared_v4(base + a * L::KV_ATOM + x, 0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[L::B_VX + st]);
        }
        if (lane == 0) mbar_arrive(&bars[L::B_VE + st]);
      }
    } while (ok && walk.next(p, 0, half_tokens, rpt));
  } else if (warp >= L::W_MMA && warp < L::W_MMA + NT) {
    // -------------------------------------------------------------- MMA issuer of a half
    if constexpr (L::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_OTHER));
    if (lane == 0) {
      const int h = warp - L::W_MMA;
      uint64_t* b = bars + L::B_HALF + h * L::N_HALF;
      const uint32_t sbase = smem_u32(smem);
      const uint32_t tS = tmem_base + h * L::TMEM_HALF;
      constexpr uint32_t kSw = swizzle_kind_for_bytes(L::ROW), kSbo = 8 * L::ROW;
      constexpr uint32_t idesc_s = umma_idesc_16(128, BN, PT::kBf16, false);
      constexpr uint32_t idesc_o = umma_idesc_16(128, HD, PT::kBf16, true);
      bool ok = true;
      // Score cursor: segment walk, tile i, ring position us, this half's tile t_s and segment count q_s.
      walk.cur.seek(p, start.b, start.off, rpt);
      walk.left = n_units;
      walk.load(p, h, half_tokens);
      ChunkWalk<HD> pv = walk;
      int i_s = walk.i0, us = 0, t_s = 0, q_s = 0;
      bool more_s = true, q_ready = false;
      // Scores of the next unit; a tile that this half does not see is handed
      // back.  It runs NSB units ahead of P.V, counted in units and not in this
      // half's tiles: the producer may then always fill what is waited for.
      auto step_s = [&]() -> bool {
        while (more_s && i_s == walk.i1) {
          q_ready = false;
          more_s = walk.next(p, h, half_tokens, rpt);
          i_s = walk.i0;
        }
        if (!more_s) return true;
        const int st = us % NSK;
        const bool mine = walk.range.has(i_s);
        if (mine && !q_ready) {
          if (!wait_phase(&b[L::H_QF + q_s % NQ], (q_s / NQ) & 1, wd, 0x535)) return false;
          q_ready = true;
        }
        if (!wait_phase(&bars[L::B_KF + st], (us / NSK) & 1, wd, 0x536)) return false;
        ++us;
        if (mine) {
          tc_fence_after();
          const uint32_t sq = sbase + L::OFF_Q + (h * NQ + q_s % NQ) * L::Q_BYTES;
          const uint32_t sk = sbase + L::OFF_K + st * L::KV_BYTES;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const int at = 16 * kk / L::ATOM, off = 16 * kk % L::ATOM * 2;
            umma_f16(tS + t_s % NSB * BN, umma_sdesc(sq + at * L::Q_ATOM + off, kSbo, kSw),
                     umma_sdesc(sk + at * L::KV_ATOM + off, kSbo, kSw), idesc_s, kk > 0 ? 1u : 0u);
          }
          umma_commit(&b[L::H_SF + t_s % NSB]);
          umma_commit(&bars[L::B_KE + st]);
          if (i_s == walk.last) umma_commit(&b[L::H_QE + q_s++ % NQ]);
          ++t_s;
        } else {
          mbar_arrive(&bars[L::B_KE + st]);
        }
        ++i_s;
        return true;
      };
      for (int k = 0; ok && k < NSB; ++k) ok = step_s();
      int uv = 0, t = 0, n_o = 0;
      uint32_t fixed = 0;  // parity of the next zeroing of each V slot
      do {
        bool first = true;
        for (int i = pv.i0; ok && i < pv.i1; ++i, ++uv) {
          const int st = uv % NSV;
          const bool mine = pv.range.has(i);
          const int r0 = pv.cur.s.L - pv.cur.it.tile(i) * BN;
          const bool fix = r0 > 0 && r0 < BN && (r0 & (page_rows - 1)) != 0;
          if (!mine) {
            if (!(ok = wait_phase(&bars[L::B_VF + st], (uv / NSV) & 1, wd, 0x537))) break;
            if (fix) fixed ^= 1u << st;
            mbar_arrive(&bars[L::B_VE + st]);
            ok = step_s();
            continue;
          }
          if (!(ok = wait_phase(&b[L::H_PF + t % NSB], (t / NSB) & 1, wd, 0x538))) break;
          if (first && !(ok = wait_phase(&b[L::H_OR + n_o % NOB], ((n_o / NOB) & 1) ^ 1, wd, 0x539))) break;
          if (!(ok = wait_phase(&bars[L::B_VF + st], (uv / NSV) & 1, wd, 0x53a))) break;
          if (fix) {
            if (!(ok = wait_phase(&bars[L::B_VX + st], (fixed >> st) & 1, wd, 0x53b))) break;
            fixed ^= 1u << st;
          }
          tc_fence_after();
          const uint32_t tO = tS + L::TMEM_O + n_o % NOB * HD;
          const uint32_t sv = sbase + L::OFF_V + st * L::KV_BYTES;
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            umma_f16_ts(tO, tS + t % NSB * BN + kk * 8, umma_sdesc_mn(sv + kk * 16 * L::ROW, L::KV_ATOM, kSbo, kSw),
                        idesc_o, first && kk == 0 ? 0u : 1u);
          first = false;
          umma_commit(&bars[L::B_VE + st]);
          umma_commit(&b[L::H_PE + t % NSB]);
          if (i == pv.last) umma_commit(&b[L::H_OF + n_o++ % NOB]);
          ++t;
          ok = step_s();
        }
      } while (ok && pv.next(p, h, half_tokens, rpt));
      // All MMAs this thread issued must finish before TMEM is released.
      umma_commit(&b[L::H_DONE]);
      wait_drain(&b[L::H_DONE], 0, kDrainLimitNs);
    }
  } else if (warp >= 4 * NT) {
    if constexpr (L::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_OTHER));
  } else {
    // -------------------------------------------------------------- softmax of a half
    if constexpr (L::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::REGS_SOFTMAX));
    const int h = warp >> 2, q = warp & 3, row = q * 32 + lane;
    uint64_t* b = bars + L::B_HALF + h * L::N_HALF;
    const uint32_t tS = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + h * L::TMEM_HALF;
    const float sl2 = p.scale_log2;
    const uint64_t sl2x2 = f2_pack(sl2, sl2);
    bool ok = true;
    int t = 0, n_o = 0;
    // A finished segment's O is read after the next segment's first tile, by
    // when its last P.V has long completed.
    bool pend = false, pend_on = false;
    int pend_o = 0;
    float pend_l = 0.f, pend_m = 0.f;
    T* pend_out = nullptr;      // whole item: the row of out
    float* pend_part = nullptr;  // cut item: its slot
    int pend_row = 0;
    auto finish = [&]() -> bool {
      pend = false;
      if (!warp_wait_phase(&b[L::H_OF + pend_o % NOB], (pend_o / NOB) & 1, wd, 0x541)) return false;
      tc_fence_after();
      const uint32_t tO = tS + L::TMEM_O + pend_o % NOB * HD;
      const float inv = pend_l > 0.f ? 1.f / pend_l : 0.f;
      if (pend_on && pend_part) {
        pend_part[L::ROWS * HD + pend_row] = pend_m;
        pend_part[L::ROWS * HD + L::ROWS + pend_row] = pend_l;
      }
      constexpr int W = HD < 32 ? HD : 32;
#pragma unroll 1
      for (int c = 0; c < HD; c += W) {
        uint32_t o[W];
        if constexpr (W == 32) {
          tmem_ld_x32_sync(tO + c, o);
        } else {
          tmem_ld_x16_sync(tO + c, o);
        }
        if (!pend_on) continue;
        if (pend_part) {
          float4* dst = reinterpret_cast<float4*>(pend_part + pend_row * HD + c);
#pragma unroll
          for (int i = 0; i < W / 4; ++i)
            dst[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                                 __uint_as_float(o[4 * i + 3]));
        } else {
#pragma unroll
          for (int i = 0; i < W / 8; ++i) {
            uint4 v;
            v.x = PT::pack(__uint_as_float(o[8 * i + 0]) * inv, __uint_as_float(o[8 * i + 1]) * inv);
            v.y = PT::pack(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv);
            v.z = PT::pack(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv);
            v.w = PT::pack(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv);
            if (c + 8 * i < p.out_hd) *reinterpret_cast<uint4*>(pend_out + c + 8 * i) = v;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b[L::H_OR + pend_o % NOB]);
      return true;
    };

    walk.cur.seek(p, start.b, start.off, rpt);
    walk.left = n_units;
    walk.load(p, h, half_tokens);
    do {
      const bool on = row < walk.rows;
      const int item_row = h * half_rows + row;
      const int pos = walk.p0 + row / p.group;
      const bool cut = walk.i0 > 0 || walk.i1 < walk.cur.it.n;
      T* out = nullptr;
      float* part = nullptr;
      if (on) {
        const int r = walk.cur.it.r0 + item_row;
        const long long tok = walk.cur.s.q0 + r / p.group;
        out = static_cast<T*>(p.out) + (tok * p.heads + walk.cur.kvh * p.group + r % p.group) * p.out_hd;
      }
      if (cut) part = p.part + (2ll * blockIdx.x + (walk.i0 > 0 ? 0 : 1)) * paged_slot_floats<L::ROWS, HD>();
      if (walk.last < 0) {  // nothing here for this half
        if (on && cut) {
          part[L::ROWS * HD + item_row] = -INFINITY;
          part[L::ROWS * HD + L::ROWS + item_row] = 0.f;
          for (int d = 0; d < HD; d += 4) *reinterpret_cast<float4*>(part + item_row * HD + d) = make_float4(0, 0, 0, 0);
        } else if (on) {
          for (int d = 0; d < p.out_hd; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(0, 0, 0, 0);
        }
        continue;
      }
      const uint32_t tO = tS + L::TMEM_O + n_o % NOB * HD;
      float m_run = -INFINITY, l_run = 0.f;
      bool first = true;
      for (int i = walk.i0; ok && i <= walk.last; ++i) {
        if (!walk.range.has(i)) {
          if (i >= walk.range.a && i < walk.range.c) i = max(walk.range.c, walk.i0) - 1;  // over the gap
          continue;
        }
        const int bb = t % NSB, k0 = walk.cur.it.tile(i) * BN;
        // Warp-uniform: some row of the half does not see the whole tile.
        const bool masked = !(k0 + BN - 1 <= walk.p0 &&
                              (p.window == 0 || k0 > walk.p1 - p.window || k0 + BN <= p.sinks));
        if (!(ok = warp_wait_phase(&b[L::H_SF + bb], (t / NSB) & 1, wd, 0x542))) break;
        tc_fence_after();
        uint32_t sc[BN / 32][32];
#pragma unroll
        for (int g = 0; g < BN / 32; ++g) tmem_ld_x32(tS + bb * BN + 32 * g, sc[g]);
#pragma unroll
        for (int g = 0; g < BN / 32; ++g) tmem_ld_wait_tied(sc[g]);
        if (masked) {
          const int hi = pos - k0 + 1, lo = p.window > 0 ? pos - p.window + 1 - k0 : 0, sk = p.sinks - k0;
#pragma unroll
          for (int g = 0; g < BN / 32; ++g) {
            const uint32_t see = bits_below(hi - 32 * g) &
                                 (p.window > 0 ? ~bits_below(lo - 32 * g) | bits_below(sk - 32 * g) : ~0u);
            if (see != ~0u) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(see & (1u << e))) sc[g][e] = 0xff800000u;  // -inf
            }
          }
        }
        float mg[BN / 32];
#pragma unroll
        for (int g = 0; g < BN / 32; ++g) {
          float a[11];
#pragma unroll
          for (int e = 0; e < 10; ++e)
            a[e] = max3(__uint_as_float(sc[g][3 * e]), __uint_as_float(sc[g][3 * e + 1]),
                        __uint_as_float(sc[g][3 * e + 2]));
          a[10] = fmaxf(__uint_as_float(sc[g][30]), __uint_as_float(sc[g][31]));
          mg[g] = max3(max3(a[0], a[1], a[2]), max3(a[3], a[4], a[5]), max3(a[6], a[7], max3(a[8], a[9], a[10])));
        }
        float m_tile = fmaxf(mg[0], mg[1]);
        if constexpr (BN == 128) m_tile = fmaxf(m_tile, fmaxf(mg[2], mg[3]));
        m_tile *= sl2;
        bool resc = false;
        float m_new = m_run;
        if (m_tile > m_run + 8.0f) {  // P stays below 2^8
          resc = m_run != -INFINITY;
          m_new = m_tile;
        }
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        if (__any_sync(~0u, resc)) {
          // O must hold every earlier tile (with one S buffer it does: S of this tile was issued after P.V of the last).
          if constexpr (NSB > 1)
            if (!(ok = warp_wait_phase(&b[L::H_PE + (t - 1) % NSB], ((t - 1) / NSB) & 1, wd, 0x543))) break;
          tc_fence_after();
          const float corr = resc ? ex2_approx(m_run - m_new) : 1.f;
          l_run *= corr;
#pragma unroll 1
          for (int c = 0; c < HD; c += 16) {  // 16 columns at a time: the scores stay in registers
            uint32_t o[16];
            tmem_ld_x16_sync(tO + c, o);
#pragma unroll
            for (int d = 0; d < 16; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * corr);
            tmem_st_x16(tO + c, o);
          }
          tmem_st_wait();
        }
        m_run = m_new;
        const uint64_t negm = f2_pack(-m_use, -m_use);
        const float y_scale = sl2 * kExpYScale, y_bias = fmaf(-m_use, kExpYScale, kExpYBias);
        uint64_t sum[2] = {f2_pack(l_run, 0.f), 0ull};
        // POLY of every 8 pairs take the polynomial; none in a masked tile,
        // where a hidden score must give exactly 0 and the clamp would not.
        auto probabilities = [&](auto poly) {
          constexpr int POLY = decltype(poly)::value;
#pragma unroll
          for (int g = 0; g < BN / 32; ++g) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              uint64_t pp;
              const float s0 = __uint_as_float(sc[g][2 * e]), s1 = __uint_as_float(sc[g][2 * e + 1]);
              if ((e & 7) < POLY) {
                pp = exp2_pair_wide(f2_pack(fma_sat(s0, y_scale, y_bias), fma_sat(s1, y_scale, y_bias)));
              } else {
                const uint64_t xx = ffma2(f2_pack(s0, s1), sl2x2, negm);
                pp = f2_pack(ex2_approx(f2_lo(xx)), ex2_approx(f2_hi(xx)));
              }
              sum[e & 1] = fadd2(sum[e & 1], pp);
              pk[e] = PT::pack(f2_lo(pp), f2_hi(pp));
            }
            tmem_st_x16(tS + bb * BN + 16 * g, pk);
          }
        };
        if (masked)
          probabilities(std::integral_constant<int, 0>());
        else
          probabilities(std::integral_constant<int, kChunkExpFma<HD>>());
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b[L::H_PF + bb]);
        const uint64_t both = fadd2(sum[0], sum[1]);
        l_run = f2_lo(both) + f2_hi(both);
        ++t;
        if (first && pend && !(ok = finish())) break;
        first = false;
      }
      if (!ok) break;
      pend = true;
      pend_on = on;
      pend_o = n_o++;
      pend_l = l_run;
      pend_m = m_run;
      pend_out = out;
      pend_part = cut ? part : nullptr;
      pend_row = item_row;
    } while (walk.next(p, h, half_tokens, rpt));
    if (ok && pend) ok = finish();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == L::W_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::TMEM_COLS);
  }
}

}  // namespace tt
