// Attention of longer chunks over a paged K/V cache on the tensor cores
// (sm_100a); parameters, schedule and the joining of cut items are in
// tt_paged_attn.cuh.
//
// One CTA per SM is one worker.  An item is two tiles ("halves") of up to 128
// query rows each (one at head_dim 256); a row is (token, head of the KV
// head's group), so grouped heads share every K and V tile.  Both halves read
// the same ring of K and V tiles (64 keys), which one producer warp fills: each
// page, or the part of it inside the tile, is one TMA box per 64 features, and a
// page that does not exist is fetched out of bounds, i.e. as zeros.  Each half
// has 4 softmax warps (a whole row per thread) and two issuing warps:
//   S = +-Q K^T       TMEM, 64 FP32 columns, NSB buffers (the scale's sign)
//   P = 2^(S - m)     FP16/BF16 pairs written over the S it came from
//   O += P V          P from TMEM, V as it lies in the page (MN-major operand)
// In FP16 from head_dim 128 a quarter of the exponentials runs as a polynomial
// on the FMA pipe.  The reference maximum m moves only when a tile exceeds it by
// 2^8 (then O and l are rescaled), and S runs up to NSB - 1 tiles ahead.  A half skips the tiles that none of its rows sees.  V rows past a
// sequence's end in its last page may hold anything (0 * NaN would reach the
// sum): the score issuer of half 0 zeroes them in shared memory.
//
// P is rounded to the cache's type, which the tensor core takes beside a 16-bit V;
// m, l (of the unrounded P) and O are FP32.  Against 64 bits that brings 1.7-2.0e-4
// to 2.4-2.7e-4 in FP16 and 1.7e-3 to 2.4e-3 in BF16 (relative norm; the output's
// rounding alone is the first figure).
//
// What bounds it: a tile of 64 keys x 256 rows takes 1700-1850 cycles.  At
// head_dim 128 the tensor core needs 1280 of them (Q K^T with N = 64 runs at 48
// cycles per MMA, the rate of its operand reads from shared memory; P V at 64)
// and is active 55 % of the time at the 1.62 GHz that the power limit leaves
// (2048 new tokens over 30k keys, 16 heads over 4, BF16: 1.03 PFLOP/s).  Below that
// the softmax warps bound it, two per scheduler and each a chain of TMEM read,
// maximum, exponentials, TMEM write.  Measured and left out: key tiles of 128
// with P over S (one S buffer: the halves fall into step and wait for the
// tensor core together, 4946 cycles per 128 keys) or beside it (582 us where
// this takes 508); one issuing warp per half (550); more code than the
// instruction cache holds (141 KB of it: 104 us for 32 prompts, 85 now).
#pragma once

#include "tt_attention.cuh"  // max3
#include "tt_paged_attn.cuh"

namespace tt {

template <int HD>
struct PagedChunkLayout {
  static constexpr int NT = HD == 256 ? 1 : 2;      // halves
  static constexpr int ROWS = 128 * NT;             // rows of a workspace slot
  static constexpr int BN = 64;                     // keys per tile
  static constexpr int NSB = HD >= 128 ? 2 : 3;     // S buffers per half
  static constexpr int NST = HD == 256 ? 2 : HD == 128 ? 5 : 8;  // stages of a K and a V tile
  static constexpr int NQ = HD >= 128 ? 1 : 2;      // Q tile buffers per half
  static constexpr int NOB = HD <= 32 ? 2 : 1;      // O buffers per half
  static constexpr int ATOM = HD >= 64 ? 64 : HD;   // features per swizzle atom
  static constexpr int NATOM = HD / ATOM;
  static constexpr int ROW = ATOM * 2;              // bytes of an atom's row
  static constexpr int Q_ATOM = 128 * ROW, KV_ATOM = BN * ROW;
  static constexpr int Q_BYTES = NATOM * Q_ATOM, KV_BYTES = NATOM * KV_ATOM;
  // Segments published ahead: the scores may be NSB segments of one tile
  // before the one whose P.V is under way, and the producer ahead of them.
  static constexpr int NSEG = 6;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = NT * NQ * Q_BYTES;
  static constexpr int OFF_V = OFF_K + NST * KV_BYTES;
  static constexpr int OFF_BAR = OFF_V + NST * KV_BYTES;
  // Barriers: stage full / empty / stale rows zeroed, segment full / empty, then
  // per half Q full / empty, S full, P full, P.V done, O full / free, drained.
  static constexpr int B_F = 0, B_E = NST, B_X = 2 * NST, B_GF = 3 * NST, B_GE = B_GF + NSEG, B_HALF = B_GE + NSEG;
  static constexpr int H_QF = 0, H_QE = 2, H_SF = 4, H_PF = H_SF + NSB, H_PE = H_PF + NSB, H_OF = H_PE + NSB,
                       H_OR = H_OF + 2, H_DONE = H_OR + 2, N_HALF = H_DONE + 2;
  static constexpr int OFF_MISC = OFF_BAR + (B_HALF + NT * N_HALF) * 8;
  static constexpr int SMEM = OFF_MISC + 16 + 1024;
  static constexpr int TMEM_COLS = 512, TMEM_O = NSB * BN, TMEM_HALF = 512 / NT;
  // Warps: softmax (half w / 4, lane quadrant w % 4), producer, score and P.V
  // issuers of each half, idle ones up to whole warpgroups (setmaxnreg).
  static constexpr int W_PROD = 4 * NT, W_S = W_PROD + 1, W_PV = W_S + NT;
  static constexpr int NWARPS = NT == 2 ? 16 : 8;
  static constexpr int THREADS = 32 * NWARPS;
  // Register split (setmaxnreg): the launch provides THREADS x REGS_LAUNCH and
  // the launcher refuses to start a kernel built with another count (a split
  // above the launch total would make setmaxnreg.inc wait forever).
  static constexpr bool SPLIT = NT == 2;
  static constexpr int REGS_LAUNCH = 128;
  static constexpr int REGS_SOFTMAX = 184, REGS_OTHER = 72;
  static_assert(!SPLIT || 128 * NT * REGS_SOFTMAX + 32 * (NWARPS - 4 * NT) * REGS_OTHER <= THREADS * REGS_LAUNCH,
                "register split");
  static_assert(NSEG >= NSB + 2, "ring depth");
  static_assert(TMEM_O + NOB * HD <= TMEM_HALF, "TMEM budget");
  static_assert(SMEM <= 232448 - 1280, "shared memory budget (the rest is static)");
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
// set the A and B formats (bits 7 and 10), an MN-major B sets bit 16.  Bit 13
// negates A.
constexpr uint32_t kIdescNegateA = 1u << 13;
__host__ __device__ constexpr uint32_t umma_idesc_16(int M, int N, bool bf16, bool b_mn) {
  return umma_idesc_f16_f32(M, N) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}

// 2^x of a pair on the FMA pipe for any x: exp2_pair_fma_y (tt_ptx.cuh) with a
// wider clamp, y = saturate((x + 126) / 256), because the FP32 row sum keeps
// what FP16 rounds to zero.  The rounding of y costs 2^-17 in x.
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

// True in one lane of a converged warp, always the same one.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ uint32_t bits_below(int x) {  // the lowest x bits (none below 0, all from 32)
  return x >= 32 ? ~0u : (x <= 0 ? 0u : (1u << x) - 1u);
}

// A segment is the part of one item that lies in the worker's piece.  The
// producer warp walks the piece and publishes each segment, one ahead of the
// tiles it fetches, for the other warps: the walk's code exists once (the
// warps' hot loops have to share the instruction cache).
struct ChunkHalf {
  int rows;      // query rows
  int p0, p1;    // positions of the first and last row
  int a, c, e;   // the item's tiles that some row sees: [0, a) and [c, e)
  int last;      // the last of them in the segment, -1: none
};
struct ChunkSegment {
  int i0, i1;           // tiles of the item (i1 < 0: the piece has ended)
  int n_sink, w_shift;  // tile i is key tile i, or i + w_shift from n_sink on
  int whole;            // the segment is a whole item
  int kvh, tok, slot, keys;  // KV head, row of q of the first token, table row, length
  int fix_at, fix_r0, fix_r1;  // tile (-1: none) whose V rows fix_r0 .. fix_r1 - 1 lie past the sequence's end
  ChunkHalf half[2];
  __device__ __forceinline__ int key(int i, int bn) const { return (i < n_sink ? i : i + w_shift) * bn; }
};

template <int HD>
__device__ __forceinline__ void chunk_segment(const PagedParams& p, const PagedWalk<PagedChunkLayout<HD>::BN>& w,
                                           int half_tokens, ChunkSegment* out) {
  using L = PagedChunkLayout<HD>;
  constexpr int BN = L::BN;
  ChunkSegment g;
  g.i0 = w.i;
  g.i1 = w.i1;
  g.n_sink = w.it.n_sink;
  g.w_shift = w.it.w_tile - w.it.n_sink;
  g.whole = w.i == 0 && w.i1 == w.it.n;
  g.kvh = w.kvh;
  g.tok = w.s.q0 + w.qt * (L::NT * half_tokens);
  g.slot = w.s.slot;
  g.keys = w.s.L;
  // Only the item's last tile can hold the sequence's end.
  const int page = 1 << p.page_shift, r0 = w.s.L - w.it.tile(w.it.n - 1) * BN;
  g.fix_r0 = r0;
  g.fix_r1 = min((r0 + page - 1) & ~(page - 1), BN);  // the end of its page, or of the tile
  g.fix_at = r0 > 0 && r0 < BN && (r0 & (page - 1)) != 0 ? w.it.n - 1 : -1;
  for (int h = 0; h < L::NT; ++h) {
    ChunkHalf x = {};
    const int tokens = min(max(w.it.p1 - w.it.p0 + 1 - h * half_tokens, 0), half_tokens);
    x.rows = tokens * p.group;
    x.last = -1;
    if (tokens > 0) {
      x.p0 = w.it.p0 + h * half_tokens;
      x.p1 = x.p0 + tokens - 1;
      const int end = x.p1 < 0 ? 0 : x.p1 / BN + 1;  // one past the last tile a row sees
      if (p.window == 0) {
        x.e = end;
      } else {
        const int from = max(x.p0 - p.window + 1, 0) / BN;  // first tile in the window
        const int sink = (min(p.sinks, BN * end) + BN - 1) / BN;
        if (w.it.n_sink == w.it.n) {  // no gap: the index is the tile
          x.a = min(sink, end);
          x.c = max(from, x.a);
          x.e = end;
        } else {
          x.a = min(w.it.n_sink, end);
          x.c = max(from - w.it.w_tile, 0) + w.it.n_sink;
          x.e = end - w.it.w_tile + w.it.n_sink;
        }
      }
      const int y = min(x.e, w.i1) - 1, z = min(x.a, w.i1) - 1;
      x.last = y >= max(x.c, w.i) ? y : (z >= w.i ? z : -1);
    }
    g.half[h] = x;
  }
  *out = g;
}

// wait_phase in few instructions (there are some twenty waits in the kernel).
__device__ __forceinline__ bool chunk_wait(uint64_t* bar, uint32_t parity, const Watchdog& wd, uint32_t site) {
  if (mbar_test_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    const bool late = globaltimer_ns() - t0 > wd.timeout_ns;
    if (late) atomicCAS(wd.err, 0u, kDevErrTimeout | (site & 0xffffu));
    if (late || *wd.abort || grid_failed(wd)) {
      *wd.abort = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool chunk_wait_warp(uint64_t* bar, uint32_t parity, const Watchdog& wd, uint32_t site) {
  return __all_sync(0xffffffffu, chunk_wait(bar, parity, wd, site));
}

// Exponentials per 8 pairs on the FMA pipe: two in FP16 from head_dim 128, where
// they gain (us with them and without: 2048 new tokens over 15k keys, 8 heads
// over 2 of 256, 320 and 334; over 30k, 16 over 4 of 128, 479 and 485; ragged
// chunks, 32 over 8 of 128, 253 and 256).  None below: 16 over 4 of 64 469 and
// 464, of 32 429 and 438, but 32 prompts of 1024, 8 heads of 32, 93 and 90 and of
// 64 95 and 95, and the polynomial's error is the larger.  None in BF16: the
// polynomial ends at 2^-126 where MUFU gives 0, which FP16 rounds away and BF16
// keeps, so that a hidden key's value near the type's largest would count (256:
// 320 and 334, 128 and 64 alike); clearing hidden weights or taking 2^-126 off
// again costs 3 to 8 % at 128.
template <typename T, int HD>
constexpr int kChunkExpFma = !Pair16<T>::kBf16 && HD >= 128 ? 2 : 0;

template <typename T, int HD>
__global__ void __launch_bounds__(PagedChunkLayout<HD>::THREADS, 1)
    paged_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const PagedParams p, int half_tokens,
                       int min_tiles) {
  using L = PagedChunkLayout<HD>;
  using PT = Pair16<T>;
  constexpr int BN = L::BN, NT = L::NT, NSB = L::NSB, NST = L::NST, NQ = L::NQ, NOB = L::NOB;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PagedCut cuts[2];
  __shared__ PagedWalk<BN> walk, walk_end;  // the producer's piece
  __shared__ ChunkSegment segments[L::NSEG];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half_rows = half_tokens * p.group, tpi = NT * half_tokens;
  long long per;
  paged_schedule<BN, 2, L::THREADS>(p, tpi, min_tiles, blockIdx.x, cuts, &per);
  paged_zero_outside(p, L::THREADS);
  pdl_trigger();
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  // The ends of the piece, the barriers and TMEM, each by a warp of its own.
  if (warp < 2) {
    PagedWalk<BN> x;
    x.b = p.batch;
    if (cuts[warp].b >= 0) x.seek(p, cuts[warp], tpi);
    if (lane == 0) (warp == 0 ? walk : walk_end) = x;
  }
  if (threadIdx.x == 64) {
    for (int i = 0; i < NST; ++i) {
      mbar_init(&bars[L::B_F + i], 1);
      mbar_init(&bars[L::B_E + i], NT);  // per half: P.V of a tile it sees, the score issuer of another
      mbar_init(&bars[L::B_X + i], 1);
    }
    for (int i = 0; i < L::NSEG; ++i) {
      mbar_init(&bars[L::B_GF + i], 1);
      mbar_init(&bars[L::B_GE + i], 6 * NT);  // softmax warps and issuers
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
      mbar_init(&b[L::H_DONE + 1], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == L::W_S) {
    tmem_alloc(tmem_slot, L::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && cuts[0].b >= 0) {
    walk.end_at(walk_end);
    if (!walk.begin()) cuts[0].b = -1;
  }
  __syncthreads();
  const uint32_t tmem_base = *tmem_slot;
  const Watchdog wd{p.err, abort_flag, p.timeout_ns};
  const int page_rows = 1 << p.page_shift;

  // A consumer's place in the ring of segments.
  struct Place {
    int at = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void step() {
      if (++at == L::NSEG) {
        at = 0;
        ph ^= 1;
      }
    }
  };

  if (warp == L::W_PROD) {
    // -------------------------------------------------------------- producer
    if constexpr (L::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_OTHER));
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const int box = min(page_rows, BN), n_box = BN / box;  // boxes of a tile: lane i fetches the i-th
    int u = 0, st = 0, nq[NT] = {};
    uint32_t ph = 0;
    Place put, get;
    bool more = cuts[0].b >= 0;  // the walk stands on a segment that is not published yet
    bool ok = true;
    for (bool started = false;; started = true) {
      // Publishes the walk's segment (or the end) and moves the walk on.
      if (!(ok = chunk_wait_warp(&bars[L::B_GE + put.at], put.ph ^ 1, wd, 0x530))) break;
      if (lane == 0) {
        if (more) {
          chunk_segment<HD>(p, walk, half_tokens, &segments[put.at]);
          more = walk.next(p, tpi);
        } else {
          segments[put.at].i1 = -1;
        }
        mbar_arrive(&bars[L::B_GF + put.at]);
      }
      __syncwarp();
      more = __shfl_sync(~0u, more, 0);
      put.step();
      if (!started) continue;  // the segment after the one in hand is always published
      const ChunkSegment& g = segments[get.at];
      get.step();
      if (g.i1 < 0) break;
#pragma unroll
      for (int h = 0; h < NT; ++h) {
        if (g.half[h].last < 0) continue;
        uint64_t* b = bars + L::B_HALF + h * L::N_HALF;
        const int qb = nq[h] % NQ;
        if (!(ok = chunk_wait_warp(&b[L::H_QE + qb], ((nq[h] / NQ) & 1) ^ 1, wd, 0x531))) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&b[L::H_QF + qb], L::NATOM * half_rows * L::ROW);
#pragma unroll
          for (int a = 0; a < L::NATOM; ++a)
            tma_load_3d(smem + L::OFF_Q + (h * NQ + qb) * L::Q_BYTES + a * L::Q_ATOM, &tmQ, &b[L::H_QF + qb],
                        a * L::ATOM, g.kvh * p.group, g.tok + h * half_tokens);
        }
        ++nq[h];
      }
      if (!ok) break;
      const int* row = p.tables + g.slot * p.table_stride;
      const int n_keys = g.keys, row0 = g.kvh * page_rows, i1 = g.i1, n_sink = g.n_sink, w_shift = g.w_shift;
      // First key of this lane's box of tile i, and its page (n_pages, past the pool's end, where there is none).
      auto key_of = [&](int i) -> int { return (i < n_sink ? i : i + w_shift) * BN + lane * box; };
      auto page_of = [&](int key) -> int {
        int pg = -1;
        if (lane < n_box && key < n_keys) pg = row[key >> p.page_shift];
        return pg < 0 || pg >= p.n_pages ? p.n_pages : pg;
      };
      int key = key_of(g.i0), page = page_of(key);
#pragma unroll 1
      for (int i = g.i0; i < i1; ++i, ++u) {
        const int next_key = key_of(i + 1);
        const int next = i + 1 < i1 ? page_of(next_key) : 0;  // a tile ahead: its latency is off the path
        const int at = row0 + (key & (page_rows - 1));
        if (!(ok = chunk_wait_warp(&bars[L::B_E + st], ph ^ 1, wd, 0x532))) break;
        if (lane == 0) mbar_arrive_expect_tx(&bars[L::B_F + st], 2 * L::KV_BYTES);
        __syncwarp();
        if (lane < n_box) {
          uint8_t* dst = smem + L::OFF_K + st * L::KV_BYTES + lane * box * L::ROW;
#pragma unroll
          for (int a = 0; a < L::NATOM; ++a) {
            tma_load_3d(dst + a * L::KV_ATOM, &tmK, &bars[L::B_F + st], a * L::ATOM, at, page);
            tma_load_3d(dst + NST * L::KV_BYTES + a * L::KV_ATOM, &tmV, &bars[L::B_F + st], a * L::ATOM, at, page);
          }
        }
        __syncwarp();
        if (++st == NST) {
          st = 0;
          ph ^= 1;
        }
        key = next_key;
        page = next;
      }
      if (!ok) break;
    }
    // Let every copy this warp started land before the CTA may exit.
    if (lane == 0) {
      for (int h = 0; h < NT; ++h)
        for (int i = max(nq[h] - NQ, 0); i < nq[h]; ++i)
          wait_drain(&bars[L::B_HALF + h * L::N_HALF + L::H_QF + i % NQ], (i / NQ) & 1, kDrainLimitNs);
      for (int i = max(u - NST, 0); i < u; ++i) wait_drain(&bars[L::B_F + i % NST], (i / NST) & 1, kDrainLimitNs);
    }
  } else if (warp >= L::W_S && warp < L::W_S + 2 * NT) {
    // -------------------------------------------------------------- issuers of a half
    // Scores and P.V are issued by warps of their own: an issuer's loop is a
    // chain of waits (115 cycles even for a phase long complete) and short
    // bursts.  A warp walks its loop as a whole on values that
    // shuffles make warp-uniform, and one elected lane issues: in a region of a
    // single lane every operand would go through vector registers.
    // The score issuer waits for every stage in turn (it must not get a ring
    // ahead: a parity tells two fills apart, not three), and each stage it waits
    // for stays as it is until its half has handed it back: by P.V, which
    // follows the scores, where the half sees the tile, and by the score issuer
    // itself where it does not.  P.V then has nothing to wait for.
    if constexpr (L::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_OTHER));
    const bool scores = warp < L::W_PV;
    const int h = __shfl_sync(~0u, warp - (scores ? L::W_S : L::W_PV), 0);
    uint64_t* b = bars + L::B_HALF + h * L::N_HALF;
    const uint32_t sbase = smem_u32(smem);
    constexpr uint32_t kSw = swizzle_kind_for_bytes(L::ROW), kSbo = 8 * L::ROW;
    const uint32_t tS = __shfl_sync(~0u, tmem_base, 0) + h * L::TMEM_HALF;
    int st = 0, buf = 0, side = 0;  // stage; S buffer; Q buffer (scores) or O buffer (P.V)
    uint32_t ph = 0, buf_ph = 0, side_ph = 0;
    uint32_t fixed = 0;  // parity of the next zeroing of each stage
    bool ok = true;
    Place get;
    while (ok) {
      if (!(ok = chunk_wait_warp(&bars[L::B_GF + get.at], get.ph, wd, 0x53e))) break;
      const ChunkSegment& g = segments[get.at];
      const ChunkHalf& x = g.half[h];
      int i = __shfl_sync(~0u, g.i0, 0);
      const int i1 = __shfl_sync(~0u, g.i1, 0), a = __shfl_sync(~0u, x.a, 0), c = __shfl_sync(~0u, x.c, 0),
                e = __shfl_sync(~0u, x.e, 0), last = __shfl_sync(~0u, x.last, 0), fix_at = __shfl_sync(~0u, g.fix_at, 0);
      const int r0 = g.fix_r0, r1 = g.fix_r1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[L::B_GE + get.at]);
      get.step();
      if (i1 < 0) break;
      bool first = true;
      if (scores) {
        const uint32_t idesc = umma_idesc_16(128, BN, PT::kBf16, false) | (p.negate ? kIdescNegateA : 0u);
        const uint64_t dq0 = umma_sdesc(sbase + L::OFF_Q + h * NQ * L::Q_BYTES, kSbo, kSw);
        const uint64_t dk0 = umma_sdesc(sbase + L::OFF_K, kSbo, kSw);
#pragma unroll 1
        for (; i < i1; ++i) {
          const bool on = i < a || (i >= c && i < e);
          if (on && first) ok = chunk_wait_warp(&b[L::H_QF + side], side_ph, wd, 0x535);
          if (on) ok = ok && chunk_wait_warp(&b[L::H_PE + buf], buf_ph ^ 1, wd, 0x537);
          if (!(ok = ok && chunk_wait_warp(&bars[L::B_F + st], ph, wd, 0x536))) break;
          if (h == 0 && i == fix_at) {  // V rows past the sequence's end hold anything: zero them
            const uint32_t base = smem_u32(smem + L::OFF_V + st * L::KV_BYTES);
            for (int at = 0; at < L::NATOM; ++at)
              for (int y = r0 * L::ROW + lane * 16; y < r1 * L::ROW; y += 512)
                st_shared_v4(base + at * L::KV_ATOM + y, 0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[L::B_X + st]);
          }
          if (on) {
            first = false;
            tc_fence_after();
            const uint64_t dq = dq0 + (side * L::Q_BYTES >> 4), dk = dk0 + (st * L::KV_BYTES >> 4);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < HD / 16; ++kk) {
                const int at = 16 * kk / L::ATOM, off = 16 * kk % L::ATOM * 2;
                umma_f16(tS + buf * BN, dq + ((at * L::Q_ATOM + off) >> 4), dk + ((at * L::KV_ATOM + off) >> 4), idesc,
                         kk > 0 ? 1u : 0u);
              }
              umma_commit(&b[L::H_SF + buf]);
              if (i == last) umma_commit(&b[L::H_QE + side]);
            }
            __syncwarp();
            if (++buf == NSB) {
              buf = 0;
              buf_ph ^= 1;
            }
            if (i == last && ++side == NQ) {
              side = 0;
              side_ph ^= 1;
            }
          } else if (lane == 0) {
            mbar_arrive(&bars[L::B_E + st]);
          }
          if (++st == NST) {
            st = 0;
            ph ^= 1;
          }
        }
      } else {
        constexpr uint32_t idesc = umma_idesc_16(128, HD, PT::kBf16, true);
        const uint64_t dv0 = umma_sdesc_mn(sbase + L::OFF_V, L::KV_ATOM, kSbo, kSw);
#pragma unroll 1
        for (; i < i1; ++i) {
          const bool on = i < a || (i >= c && i < e);
          const bool fix = i == fix_at;
          if (on) {
            if (first) ok = chunk_wait_warp(&b[L::H_OR + side], side_ph ^ 1, wd, 0x539);
            ok = ok && chunk_wait_warp(&b[L::H_PF + buf], buf_ph, wd, 0x538);
            // (After P: the stage then holds this tile, so the zeroing before this one is over and the parity exact.)
            if (fix) ok = ok && chunk_wait_warp(&bars[L::B_X + st], (fixed >> st) & 1, wd, 0x53b);
            if (!ok) break;
            tc_fence_after();
            const uint64_t dv = dv0 + (st * L::KV_BYTES >> 4);
            const uint32_t tO = tS + L::TMEM_O + side * HD, tP = tS + buf * BN;
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < BN / 16; ++kk)
                umma_f16_ts(tO, tP + kk * 8, dv + (kk * 16 * L::ROW >> 4), idesc, kk == 0 && first ? 0u : 1u);
              umma_commit(&b[L::H_PE + buf]);
              umma_commit(&bars[L::B_E + st]);
              if (i == last) umma_commit(&b[L::H_OF + side]);
            }
            __syncwarp();
            first = false;
            if (++buf == NSB) {
              buf = 0;
              buf_ph ^= 1;
            }
            if (i == last && ++side == NOB) {
              side = 0;
              side_ph ^= 1;
            }
          }
          if (fix) fixed ^= 1u << st;
          if (++st == NST) st = 0;
        }
      }
    }
    // All MMAs the elected lane issued must finish before TMEM is released.
    uint64_t* done = &b[L::H_DONE + (scores ? 0 : 1)];
    if (elect_one()) umma_commit(done);
    __syncwarp();
    if (lane == 0) wait_drain(done, 0, kDrainLimitNs);
    __syncwarp();
  } else if (warp >= 4 * NT) {
    if constexpr (L::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_OTHER));
  } else {
    // -------------------------------------------------------------- softmax of a half
    if constexpr (L::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::REGS_SOFTMAX));
    const int h = warp >> 2, q = warp & 3, row = q * 32 + lane;
    uint64_t* b = bars + L::B_HALF + h * L::N_HALF;
    const uint32_t tS = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + h * L::TMEM_HALF;
    const int t = row / p.group;  // the row's token in the half
    const float sl2 = p.scale_log2;
    const uint64_t sl2x2 = f2_pack(sl2, sl2);
    bool ok = true;
    int s_buf = 0, o_buf = 0;
    uint32_t s_ph = 0, o_ph = 0;
    // A finished segment's O is read after the next segment's first tile, by
    // when its last P.V has long completed.
    bool pend = false, pend_on = false;
    int pend_o = 0;
    uint32_t pend_ph = 0;
    float pend_l = 0.f, pend_m = 0.f;
    T* pend_out = nullptr;      // whole item: the row of out
    float* pend_part = nullptr;  // cut item: its slot
    int pend_row = 0;
    auto finish = [&]() -> bool {
      pend = false;
      if (!chunk_wait_warp(&b[L::H_OF + pend_o], pend_ph, wd, 0x541)) return false;
      tc_fence_after();
      const uint32_t tO = tS + L::TMEM_O + pend_o * HD;
      const float inv = pend_l > 1e-30f ? 1.f / pend_l : 0.f;  // (a row that sees a key has l >= 1)
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
      if (lane == 0) mbar_arrive(&b[L::H_OR + pend_o]);
      return true;
    };

    for (Place get; ok; get.step()) {
      if (!(ok = chunk_wait_warp(&bars[L::B_GF + get.at], get.ph, wd, 0x540))) break;
      int i, last, p0, p1, pos, n_sink, w_shift, a, c;
      bool on;
      const int item_row = h * half_rows + row;
      T* out = nullptr;
      float* part = nullptr;  // set when the item is cut
      {
        const ChunkSegment& g = segments[get.at];
        if (g.i1 < 0) break;
        const ChunkHalf& x = g.half[h];
        a = x.a;
        c = x.c;
        i = g.i0 < a ? g.i0 : max(c, g.i0);
        last = x.last;
        p0 = x.p0;
        p1 = x.p1;
        pos = p0 + t;
        on = row < x.rows;
        n_sink = g.n_sink;
        w_shift = g.w_shift;
        if (on)
          out = static_cast<T*>(p.out) +
                (static_cast<long long>(g.tok + h * half_tokens + t) * p.heads + g.kvh * p.group + row - t * p.group) *
                    p.out_hd;
        if (!g.whole) part = p.part + (2ll * blockIdx.x + (g.i0 > 0 ? 0 : 1)) * paged_slot_floats<L::ROWS, HD>();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[L::B_GE + get.at]);
      if (last < 0) {  // nothing here for this half
        if (on && part) {
          part[L::ROWS * HD + item_row] = -INFINITY;
          part[L::ROWS * HD + L::ROWS + item_row] = 0.f;
          for (int d = 0; d < HD; d += 4) *reinterpret_cast<float4*>(part + item_row * HD + d) = make_float4(0, 0, 0, 0);
        } else if (on) {
          for (int d = 0; d < p.out_hd; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(0, 0, 0, 0);
        }
        continue;
      }
      // Every row of the half sees all of a tile that starts at k0 <= k_hi
      // and, under a window, past k_lo or within the first tokens.
      const int k_hi = p0 - BN + 1, k_lo = p.window > 0 ? p1 - p.window : -1, k_sk = p.sinks - BN;
      const int lo_pos = p.window > 0 ? pos - p.window + 1 : 0;
      const uint32_t tO = tS + L::TMEM_O + o_buf * HD;
      float m_run = -INFINITY, l_run = 0.f;
      bool first = true;
      for (;;) {
        const int k0 = (i < n_sink ? i : i + w_shift) * BN;
        const bool masked = k0 > k_hi || (k0 <= k_lo && k0 > k_sk);  // warp-uniform
        if (!(ok = chunk_wait_warp(&b[L::H_SF + s_buf], s_ph, wd, 0x542))) break;
        tc_fence_after();
        const uint32_t tSb = tS + s_buf * BN;
        uint32_t sc[BN / 32][32];
#pragma unroll
        for (int g = 0; g < BN / 32; ++g) tmem_ld_x32(tSb + 32 * g, sc[g]);
#pragma unroll
        for (int g = 0; g < BN / 32; ++g) tmem_ld_wait_tied(sc[g]);
        if (masked) {
          const int hi = pos - k0 + 1, lo = lo_pos - k0, sk = p.sinks - k0;
#pragma unroll
          for (int g = 0; g < BN / 32; ++g) {
            const uint32_t see =
                bits_below(hi - 32 * g) & (~bits_below(lo - 32 * g) | bits_below(sk - 32 * g));
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
        const float m_tile = fmaxf(mg[0], mg[1]) * sl2;
        bool resc = false;
        float m_new = m_run;
        if (m_tile > m_run + 8.0f) {  // P stays below 2^8
          resc = m_run != -INFINITY;
          m_new = m_tile;
        }
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        if (__any_sync(~0u, resc)) {
          // O must hold every earlier tile: wait for P.V of the last.
          const int pb = s_buf == 0 ? NSB - 1 : s_buf - 1;
          if (!(ok = chunk_wait_warp(&b[L::H_PE + pb], s_buf == 0 ? s_ph ^ 1 : s_ph, wd, 0x543))) break;
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
        // x = s scale - m in one rounding leaves the rounding of m, at most
        // m 2^-24, in every exponent of the row: a factor that cancels against l
        // until 2^x leaves FP16, from m = 2^27 on.  Scaling first, as the kernels
        // for short chunks do, or in such rows only, costs 4 to 8 % here.
        const uint64_t negm = f2_pack(-m_use, -m_use);
        const float y_scale = sl2 * kExpYScale, y_bias = fmaf(-m_use, kExpYScale, kExpYBias);
        uint64_t sum[2] = {f2_pack(l_run, 0.f), 0ull};
        // A hidden score gives 0 on MUFU and 2^-126 where the polynomial's
        // clamp ends: in the sum nothing beside the row's largest term, which is
        // at least 1 (a row that saw no key is known by its tiny sum), and as a
        // weight 0 in FP16.
#pragma unroll
        for (int g = 0; g < BN / 32; ++g) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            uint64_t pp;
            const float s0 = __uint_as_float(sc[g][2 * e]), s1 = __uint_as_float(sc[g][2 * e + 1]);
            if ((e & 7) < kChunkExpFma<T, HD>) {
              pp = exp2_pair_wide(f2_pack(fma_sat(s0, y_scale, y_bias), fma_sat(s1, y_scale, y_bias)));
            } else {
              const uint64_t xx = ffma2(f2_pack(s0, s1), sl2x2, negm);
              pp = f2_pack(ex2_approx(f2_lo(xx)), ex2_approx(f2_hi(xx)));
            }
            sum[e & 1] = fadd2(sum[e & 1], pp);
            pk[e] = PT::pack(f2_lo(pp), f2_hi(pp));
          }
          tmem_st_x16(tSb + 16 * g, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b[L::H_PF + s_buf]);
        const uint64_t both = fadd2(sum[0], sum[1]);
        l_run = f2_lo(both) + f2_hi(both);
        if (++s_buf == NSB) {
          s_buf = 0;
          s_ph ^= 1;
        }
        if (first && pend && !(ok = finish())) break;
        first = false;
        ++i;
        if (i >= a && i < c) i = c;
        if (i > last) break;
      }
      if (!ok) break;
      pend = true;
      pend_on = on;
      pend_o = o_buf;
      pend_ph = o_ph;
      pend_l = l_run;
      pend_m = m_run;
      pend_out = out;
      pend_part = part;
      pend_row = item_row;
      if (++o_buf == NOB) {
        o_buf = 0;
        o_ph ^= 1;
      }
    }
    if (ok && pend) ok = finish();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == L::W_S) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::TMEM_COLS);
  }
}

}  // namespace tt
