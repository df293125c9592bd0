// Attention of a chunk of new tokens over a paged K/V cache, with grouped KV
// heads, an optional sliding window and a few first tokens that stay visible:
// parameters, work schedule and the kernel for short chunks (sm_100a).
//
// Sequence b has the query rows cu_q[b] .. cu_q[b+1] of its T new tokens and L
// = lens[slot] keys, the new ones included.  Query j stands at t = L - T + j
// and sees key u iff 0 <= u <= t and (no window, or t - u < window, or u <
// sinks):
//   o = sum_u 2^(s_u - m) v_u / sum_u 2^(s_u - m),  s_u = (q . k_u) scale log2 e.
// A row that sees no key (t < 0) is zero, and so is a row of no sequence.
//
// Work is laid out on one line: an item (some tokens of one sequence for one KV
// head) takes as much of it as its queries span keys, plus a constant.  The
// line is cut into equal pieces, one per worker, and a cut inside an item falls
// on a key tile, so a single long sequence and a ragged batch both fill the
// GPU.  Sums over the items of a sequence are closed forms: no kernel walks
// items to find its piece.  An item that lies in one piece is finished by its
// worker; the parts of an item that was cut (O unnormalised, m, l, in FP32) go
// to the workspace and are joined by paged_join_kernel, always in worker order,
// so results do not depend on timing.
#pragma once

#include <cuda_bf16.h>

#include "tt_ptx.cuh"

namespace tt {

struct PagedParams {
  const void* q;               // [n_tokens, heads, HD], element strides below, last dimension dense
  long long q_token, q_head;
  const void* k_pages;         // [n_pages, kv_heads, page, HD], pages k_stride elements apart
  const void* v_pages;
  long long k_stride, v_stride;
  const int* tables;           // [n_slots, table_width], rows table_stride apart; < 0: no page
  long long table_stride;
  const int* lens;             // [n_slots]
  const int* cu_q;             // [batch + 1]
  const int* slots;            // [batch], or nullptr: slot b is sequence b
  void* out;                   // [n_tokens, heads * out_hd]
  float* part;                 // parts of cut items
  int n_tokens, batch, n_slots, heads, kv_heads, group;
  int n_pages, page_shift, table_width;
  int window, sinks;           // window 0: none
  int out_hd;
  int row_lo, row_hi;          // this launch serves sequences of row_lo .. row_hi query rows (T * group)
  int n_workers;
  int item_len;                // extra length of an item on the line, in keys: its queries' loads and its output
  float scale_log2;            // scale log2 e; in the chunk kernel its size, and `negate` its sign
  int negate;
  unsigned int* err;
  unsigned long long timeout_ns;
};

struct PagedSeq {
  int q0, T, L, slot;
};

// Sequence b with every field brought into range: rows outside q, a slot or a
// length that does not exist become an empty sequence or an empty cache.
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
  PagedSeq s;
  s.q0 = min(max(p.cu_q[b], 0), p.n_tokens);
  s.T = max(min(p.cu_q[b + 1], p.n_tokens) - s.q0, 0);
  s.slot = p.slots ? p.slots[b] : b;
  const bool ok = s.slot >= 0 && s.slot < p.n_slots;
  s.slot = ok ? s.slot : 0;
  const long long room = static_cast<long long>(p.table_width) << p.page_shift;
  const int len = ok ? p.lens[s.slot] : 0;
  s.L = static_cast<int>(min(static_cast<long long>(max(len, 0)), room));
  return s;
}

constexpr int kPagedMaxWorkers = 2048;

// One item: the tokens qt * tpi .. of a sequence (rows: token * group + head of
// the group) and the key tiles that some row of it can see.  With a window the
// tiles are [0, n_sink) and [w_tile, ...); tile(i) maps the i-th of n.
template <int TK>
struct PagedItem {
  int r0, rows, p0, p1;  // first row, rows, positions of the first and last token
  int n, n_sink, w_tile;
  __device__ __forceinline__ void set(const PagedParams& p, const PagedSeq& s, int qt, int tpi) {
    const int t0 = qt * tpi, t1 = min(t0 + tpi, s.T);
    r0 = t0 * p.group;
    rows = (t1 - t0) * p.group;
    p0 = s.L - s.T + t0;
    p1 = s.L - s.T + t1 - 1;
    const int total = p1 < 0 ? 1 : p1 / TK + 1;  // an item of rows that see nothing keeps one tile, wholly masked
    n_sink = total;
    w_tile = total;
    n = total;
    if (p.window > 0) {
      const int first = max(p0 - p.window + 1, 0);
      const int ns = (min(p.sinks, first) + TK - 1) / TK;
      const int wt = first / TK;
      if (ns < wt) {
        n_sink = ns;
        w_tile = wt;
        n = ns + total - wt;
      }
    }
  }
  __device__ __forceinline__ int tile(int i) const { return i < n_sink ? i : i - n_sink + w_tile; }
  // Whether every row sees every key of [k0, k0 + TK).
  __device__ __forceinline__ bool whole(const PagedParams& p, int k0) const {
    return k0 + TK - 1 <= p0 && (p.window == 0 || k0 > p1 - p.window || k0 + TK <= p.sinks);
  }
};

__device__ __forceinline__ int paged_q_tiles(const PagedParams& p, const PagedSeq& s, int tpi) {
  const int rows = s.T * p.group;
  return rows >= p.row_lo && rows <= p.row_hi ? (s.T + tpi - 1) / tpi : 0;
}

// a / b for a >= 0, b > 0; 64-bit division is a long subroutine and rarely needed.
__device__ __forceinline__ long long div_pos(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

// sum over j < n of max(a + j d, 0), d > 0, where j0 is the first j with a + j d >= 0.
__device__ __forceinline__ long long ramp_sum(long long a, int d, int j0, int n) {
  const long long m = max(n - j0, 0);
  return m * (a + static_cast<long long>(j0) * d) + d * (m * (m - 1) / 2);
}
__device__ __forceinline__ int ramp_start(long long a, int d) {
  return a >= 0 ? 0 : static_cast<int>(div_pos(-a + d - 1, d));
}

// Length on the line of the first q of sequence s's nq items for one KV head:
// item j spans the keys up to position p1(j), less, under a window, those
// between the first tokens and the window of p0(j).
template <int TK>
struct PagedLine {
  long long up, gap;  // p1(0) + 1; p0(0) + 1 - window - sinks
  int up0, gap0, nq, tpi, L, item_len;
  bool window;
  __device__ __forceinline__ PagedLine(const PagedParams& p, const PagedSeq& s, int nq_, int tpi_)
      : nq(nq_), tpi(tpi_), L(s.L), item_len(p.item_len), window(p.window > 0) {
    const long long base = s.L - s.T;
    up = base + tpi;
    up0 = ramp_start(up, tpi);
    gap = base - p.window + 1 - p.sinks;
    gap0 = window ? ramp_start(gap, tpi) : 0;
  }
  __device__ __forceinline__ long long before(int q) const {
    if (q == 0) return 0;
    const int whole = q == nq ? q - 1 : q;  // the last item may hold fewer tokens
    long long len = static_cast<long long>(q) * item_len + ramp_sum(up, tpi, up0, whole);
    if (q == nq) len += L;
    if (window) len -= ramp_sum(gap, tpi, gap0, q);
    return len;
  }
  __device__ __forceinline__ long long all() const { return before(nq); }
};

// A cut of the line: sequence and length into it (b < 0: the end of the line).
struct PagedCut {
  int b;
  long long off;
};

// Walks one worker's piece item by item: sequence, KV head, item, tiles i .. i1.
template <int TK>
struct PagedWalk {
  int b, kvh, qt, nq, i, i1;
  PagedSeq s;
  PagedItem<TK> it;
  int end_b, end_kvh, end_qt, end_i;
  long long at, len;  // seek: where in the item the cut falls, and the item's length

  // Places the walk on a cut.  The whole warp takes part: the item is found 32
  // candidates at a time (this stands before a kernel's first load).
  __device__ __forceinline__ void seek(const PagedParams& p, const PagedCut& c, int tpi) {
    const int lane = threadIdx.x & 31;
    b = c.b;
    s = paged_seq(p, b);
    nq = paged_q_tiles(p, s, tpi);
    const PagedLine<TK> line(p, s, nq, tpi);
    const long long head = line.all();
    kvh = p.kv_heads == 1 ? 0 : static_cast<int>(div_pos(c.off, head));
    const long long off = c.off - kvh * head;
    qt = 0;  // the last item that begins at or before off
    long long start = 0, next = head;
    for (int n = nq; n > 1;) {
      const int step = (n + 31) >> 5, q = qt + lane * step;
      const long long x = lane * step < n ? line.before(q) : head + 1;
      const int hit = 31 - __clz(__ballot_sync(~0u, x <= off));  // (lane 0 always: q = qt)
      start = __shfl_sync(~0u, x, hit);
      if (hit < 31) next = min(next, __shfl_sync(~0u, x, hit + 1));
      qt += hit * step;
      n = min(step, n - hit * step);
    }
    at = off - start;
    len = next - start;
    it.set(p, s, qt, tpi);
    i = tile_at(at);
  }
  // The tile on which a cut at length x of the item falls.  Every kernel and
  // worker must find the same one: one multiplication and no contraction.
  __device__ __forceinline__ int tile_at(long long x) const {
    return min(static_cast<int>(__fmul_rn(__ll2float_rn(x), __fdiv_rn(__int2float_rn(it.n), __ll2float_rn(len)))),
               it.n - 1);
  }

  __device__ __forceinline__ bool at_end() const { return b == end_b && kvh == end_kvh && qt == end_qt; }
  __device__ __forceinline__ void end_at(const PagedWalk& e) {
    end_b = e.b;
    end_kvh = e.kvh;
    end_qt = e.qt;
    end_i = e.i;
  }
  // After seek and end_at: whether the piece holds any tile.
  __device__ __forceinline__ bool begin() {
    i1 = at_end() ? end_i : it.n;
    return i < i1;
  }
  // On to the next item; false at the end of the piece.
  __device__ __forceinline__ bool next(const PagedParams& p, int tpi) {
    if (at_end()) return false;
    i = 0;
    if (++qt == nq) {
      qt = 0;
      if (++kvh == p.kv_heads) {
        kvh = 0;
        do {
          if (++b >= p.batch) return false;
          s = paged_seq(p, b);
          nq = paged_q_tiles(p, s, tpi);
        } while (nq == 0);
      }
    }
    it.set(p, s, qt, tpi);
    i1 = at_end() ? end_i : it.n;
    return i1 > 0;
  }
};

// Block-wide: the piece length `per` and the cuts where the workers
// first_worker .. first_worker + NC - 1 begin (NC < 32).  Every thread takes part.
template <int TK, int NC, int THREADS>
__device__ __forceinline__ void paged_schedule(const PagedParams& p, int tpi, int min_tiles, int first_worker,
                                               PagedCut* cuts, long long* per) {
  constexpr int NWARPS = THREADS / 32;
  __shared__ long long warp_sum[NWARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < NC) cuts[tid].b = -1;
  long long lo = 0, hi = 0, carry = 0, each = 0;  // this thread's sequence lies at lo .. hi on the line
  int b = 0;
  auto mark = [&]() {
    for (int w = 0; w < NC; ++w) {
      const long long cut = (first_worker + w) * each;
      if (cut >= lo && cut < hi) cuts[w] = {b, cut - lo};
    }
  };
  // One round per THREADS sequences; a second pass, with the length known, only
  // for batches of more than one round.  (The loops stay rolled: their code
  // stands in every kernel.)
#pragma unroll 1
  for (int pass = 0; pass < (p.batch <= THREADS ? 1 : 2); ++pass) {
    carry = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < p.batch; b0 += THREADS) {
      b = b0 + tid;
      long long u = 0;
      if (b < p.batch) {
        const PagedSeq s = paged_seq(p, b);
        const int nq = paged_q_tiles(p, s, tpi);
        if (nq > 0) u = PagedLine<TK>(p, s, nq, tpi).all() * p.kv_heads;
      }
      long long inc = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(~0u, inc, o);
        if (lane >= o) inc += v;
      }
      __syncthreads();  // the round before has read warp_sum
      if (lane == 31) warp_sum[warp] = inc;
      __syncthreads();
      long long sums = lane < NWARPS ? warp_sum[lane] : 0;
#pragma unroll
      for (int o = 1; o < NWARPS; o <<= 1) {
        const long long v = __shfl_up_sync(~0u, sums, o);
        if (lane >= o) sums += v;
      }
      const long long before = carry + (warp > 0 ? __shfl_sync(~0u, sums, warp > 0 ? warp - 1 : 0) : 0);
      carry += __shfl_sync(~0u, sums, NWARPS - 1);
      lo = before + inc - u;
      hi = before + inc;
      if (pass == 1) mark();
    }
    if (pass == 0)
      each = max(div_pos(carry + p.n_workers - 1, p.n_workers), static_cast<long long>(min_tiles) * TK);
  }
  if (p.batch <= THREADS) mark();
  *per = each;
  __syncthreads();
}

// Zeros the rows of q that belong to no sequence (before cu_q[0], from cu_q[batch] on).
__device__ __forceinline__ void paged_zero_outside(const PagedParams& p, int threads) {
  const int lo = p.batch > 0 ? min(max(p.cu_q[0], 0), p.n_tokens) : 0;
  const int hi = p.batch > 0 ? min(max(p.cu_q[p.batch], lo), p.n_tokens) : 0;
  const long long row = static_cast<long long>(p.heads) * p.out_hd / 8;  // 16-byte pieces
  const long long n = (lo + p.n_tokens - hi) * row;
  uint4* out = static_cast<uint4*>(p.out);
  for (long long i = blockIdx.x * static_cast<long long>(threads) + threadIdx.x; i < n;
       i += static_cast<long long>(gridDim.x) * threads) {
    const long long at = i < lo * row ? i : i - lo * row + hi * row;
    out[at] = make_uint4(0, 0, 0, 0);
  }
}

template <typename T>
struct Pair16;  // two 16-bit values in a register, and the MMA on them
template <>
struct Pair16<__half> {
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Pair16<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// ---------------------------------------------------------------------------
// Parts of cut items.  Worker w owns the slots 2w (its piece begins inside an
// item) and 2w + 1 (an item that begins in its piece and goes on past it).
// A slot holds ROWS x HD of O, then ROWS of m and ROWS of l.
// ---------------------------------------------------------------------------
template <int ROWS, int HD>
__host__ __device__ constexpr long long paged_slot_floats() {
  return static_cast<long long>(ROWS) * (HD + 2);
}

// Joins the parts of the item that the start of worker c cuts, if c is the
// first worker to start inside it: with M = max_i m_i,
//   O = sum_i O_i 2^(m_i - M) / sum_i l_i 2^(m_i - M).
// One block per (worker, RB rows of the item).  A thread has four features of a
// row; where rows are few, the parts are dealt over several threads and their
// sums joined in a fixed order.  The launch is programmatic, so blocks start on
// SMs that the attention kernel has left and run the schedule beside its tail;
// most find that they have nothing to join.  Those wait for the attention
// kernel too: what comes after this grid (a node of a captured graph, say)
// depends on this grid alone, so it must not end before that kernel has.

struct JoinSum {
  float m, l;
  float4 o;
  __device__ __forceinline__ void add(float mk, float lk, const float4& ok) {
    const float top = fmaxf(m, mk), base = top == -INFINITY ? 0.f : top;
    const float a = ex2_approx(m - base), b = ex2_approx(mk - base);
    m = top;
    l = l * a + lk * b;
    o.x = o.x * a + ok.x * b;
    o.y = o.y * a + ok.y * b;
    o.z = o.z * a + ok.z * b;
    o.w = o.w * a + ok.w * b;
  }
};

template <typename T, int HD, int TK, int ROWS, int RB, int THREADS>
__global__ void __launch_bounds__(THREADS) paged_join_kernel(const PagedParams p, int tpi, int min_tiles) {
  __shared__ PagedCut cut;
  __shared__ uint8_t holds[kPagedMaxWorkers];  // whether the k-th worker from c on has a part
  __shared__ JoinSum sums[THREADS];
  __shared__ PagedWalk<TK> cur;
  __shared__ int n_after;  // workers from c on that start inside the item; 0: nothing to join here
  long long per;
  const int c = blockIdx.x + 1;  // worker 0 starts at an item's beginning
  paged_schedule<TK, 1, THREADS>(p, tpi, min_tiles, c, &cut, &per);
  if (cut.b < 0) return pdl_wait();
  if (threadIdx.x < 32) {
    PagedWalk<TK> w;
    w.seek(p, cut, tpi);
    if (threadIdx.x == 0) {
      cur = w;
      const bool mine = cur.i > 0 && cur.it.rows > static_cast<int>(blockIdx.y) * RB &&
                        !(cur.at > per && cur.tile_at(cur.at - per) > 0);  // worker c - 1 starts inside too
      n_after = mine ? static_cast<int>(div_pos(cur.len - cur.at + per - 1, per)) : 0;
    }
  }
  __syncthreads();
  if (n_after == 0) return pdl_wait();
  for (int k = threadIdx.x; k < n_after; k += THREADS)
    holds[k] = cur.tile_at(cur.at + k * per) < (k + 1 < n_after ? cur.tile_at(cur.at + (k + 1) * per) : cur.it.n);
  __syncthreads();
  pdl_wait();
  const int row0 = blockIdx.y * RB, rows = min(cur.it.rows - row0, RB);
  constexpr long long SLOT = paged_slot_floats<ROWS, HD>();
  const float* first = p.part + (2ll * (c - 1) + 1) * SLOT;
  const float* rest = p.part + 2ll * c * SLOT;  // then every 2 SLOT
  constexpr int TPR = HD / 4, GROUPS = THREADS / TPR;
  const int g = threadIdx.x / TPR, d = threadIdx.x % TPR * 4;
  // Rows of the block's threads, and the share of the parts that a thread takes.
  const int deal = rows < GROUPS ? GROUPS / rows : 1;
  const int share = deal > 1 ? g / rows : 0, row_in = deal > 1 ? g - share * rows : g;
  for (int r0 = 0; r0 < rows; r0 += GROUPS) {
    const int row = row0 + r0 + row_in;
    const bool on = row < row0 + rows && share < deal;
    JoinSum sum = {-INFINITY, 0.f, make_float4(0, 0, 0, 0)};
    if (on) {
      const int m_at = ROWS * HD + row, l_at = m_at + ROWS, o_at = row * HD + d;
      if (share == 0) sum = {first[m_at], first[l_at], *reinterpret_cast<const float4*>(first + o_at)};
      int k = share;
      constexpr int U = 4;  // parts in flight where they are many
#pragma unroll 1
      for (; k + (U - 1) * deal < n_after; k += U * deal) {
        float mk[U], lk[U];
        float4 ok[U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
          const bool has = holds[k + x * deal];
          const float* s = rest + 2 * SLOT * (k + x * deal);
          mk[x] = has ? s[m_at] : -INFINITY;
          lk[x] = has ? s[l_at] : 0.f;
          ok[x] = has ? *reinterpret_cast<const float4*>(s + o_at) : make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int x = 0; x < U; ++x) sum.add(mk[x], lk[x], ok[x]);
      }
#pragma unroll 1
      for (; k < n_after; k += deal)
        if (holds[k]) {
          const float* s = rest + 2 * SLOT * k;
          sum.add(s[m_at], s[l_at], *reinterpret_cast<const float4*>(s + o_at));
        }
    }
    if (deal > 1) {
      sums[threadIdx.x] = sum;
      __syncthreads();
      if (on && share == 0)
        for (int x = 1; x < deal; ++x) {
          const JoinSum& y = sums[threadIdx.x + x * rows * TPR];
          sum.add(y.m, y.l, y.o);
        }
    }
    if (on && share == 0 && d < p.out_hd) {
      const float inv = sum.l > 0.f ? 1.f / sum.l : 0.f;
      const int t = row / p.group, tok = cur.s.q0 + cur.qt * tpi + t, h = cur.kvh * p.group + row - t * p.group;
      uint2* dst = reinterpret_cast<uint2*>(static_cast<T*>(p.out) +
                                            (static_cast<long long>(tok) * p.heads + h) * p.out_hd + d);
      *dst = make_uint2(Pair16<T>::pack(sum.o.x * inv, sum.o.y * inv), Pair16<T>::pack(sum.o.z * inv, sum.o.w * inv));
    }
  }
}

// ---------------------------------------------------------------------------
// Short chunks: at most 16 query rows per item, so the cache is read at most
// once per 16 rows and the memory system bounds the kernel (12 sequences of 20k
// to 65k tokens, 8 KV heads of 128, 2.0 GB: 305 us a call, 6.55 TB/s, the rate
// of a plain copy).  Every warp is a
// worker of its own with a private ring of NST stages (TK keys and values,
// 16-byte asynchronous copies), no block-wide synchronisation in the loop:
//   S = Q K^T (mma.sync m16n8k16, FP32), online softmax on the fragments,
//   O += P V with P rounded to the cache's type (the A operand's layout is the
//   accumulator's, so P never leaves registers).
// That rounding is the one besides the output's: mma.sync takes no wider A with
// a 16-bit V, and P in two terms would double the P V instructions.  l sums
// the unrounded P.  Against 64 bits it brings 2.0-2.3e-4 to 2.3-2.8e-4 in FP16 and
// 1.7e-3 to 2.1-2.3e-3 in BF16 (relative norm; the output's rounding alone is the
// first figure).
// At head_dim 256 O and the queries leave the rows kernel short of registers: it
// stores 136 bytes a thread outside them and loads 68.
// Values of keys past the sequence's end are zero-filled by the copy: stale
// rows of a page never reach the sum.
// ---------------------------------------------------------------------------
template <int HD>
struct PagedRowsLayout {
  static constexpr int TK = HD >= 128 ? 16 : 2048 / HD;  // keys per tile: 4 KB of K (8 KB at 256 features)
  static constexpr int WARPS = HD == 256 ? 4 : 8;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int NST = 3;
  static constexpr int RB = HD * 2;  // bytes of a row
  static constexpr int TILE = TK * RB;
  static constexpr int STAGE = 2 * TILE;
  static constexpr int SMEM = WARPS * NST * STAGE + 128;
  static constexpr int CH = RB / 16;                 // 16-byte pieces of a row
  static constexpr int RPL = RB >= 128 ? 1 : 128 / RB;  // rows per 128 bytes
  static constexpr int SWM = CH < 8 ? CH - 1 : 7;
  static_assert(SMEM <= 232448, "shared memory budget");
};

// 16-byte asynchronous copy of data that is read once (first to leave L2).
__device__ __forceinline__ uint64_t policy_evict_first() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void cp_async_16_once(uint32_t dst, const void* src, uint32_t src_bytes, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(src_bytes),
               "l"(policy)
               : "memory");
}

// Byte offset of 16-byte piece c of row r: the pieces are permuted so that the
// same piece of eight consecutive rows falls into eight different bank groups.
template <int HD>
__device__ __forceinline__ uint32_t paged_rows_at(int r, int c) {
  using L = PagedRowsLayout<HD>;
  return r * L::RB + ((c ^ ((r / L::RPL) & L::SWM)) << 4);
}

// Copies keys k0 .. k0 + TK - 1 of one KV head and their values to sk (then the values).
template <typename T, int HD>
__device__ __forceinline__ void paged_rows_fetch(const PagedParams& p, const int* row, int n_keys, int kvh, int k0,
                                                 uint32_t sk, uint64_t policy) {
  using L = PagedRowsLayout<HD>;
  const int lane = threadIdx.x & 31;
  const int page_at = (k0 >> p.page_shift) + lane;
  int page = page_at < p.table_width ? row[page_at] : -1;  // lane i: the i-th page of the tile
  if (page >= p.n_pages) page = -1;
  const uint32_t sv = sk + L::TILE;
#pragma unroll
  for (int c0 = 0; c0 < L::TK * L::CH; c0 += 32) {
    const int c = c0 + lane, r = c / L::CH, ch = c % L::CH;
    const int key = k0 + r;
    const int pg = __shfl_sync(~0u, page, (key >> p.page_shift) - (k0 >> p.page_shift));
    const bool ok = pg >= 0 && key < n_keys;
    const long long in_page =
        (static_cast<long long>(kvh) << p.page_shift) * HD + (key & ((1 << p.page_shift) - 1)) * HD + ch * 8;
    const long long at = ok ? pg : 0;
    cp_async_16_once(sk + paged_rows_at<HD>(r, ch), static_cast<const T*>(p.k_pages) + at * p.k_stride + in_page,
                     ok ? 16u : 0u, policy);
    cp_async_16_once(sv + paged_rows_at<HD>(r, ch), static_cast<const T*>(p.v_pages) + at * p.v_stride + in_page,
                     ok ? 16u : 0u, policy);
  }
}

// A warp's softmax over the tiles that it takes of an item: queries, running
// maximum and sum (this lane's keys) and O, as fragments of the MMA; a lane has
// rows lane / 4 and lane / 4 + 8.
template <typename T, int HD>
struct PagedRows {
  using L = PagedRowsLayout<HD>;
  using PT = Pair16<T>;
  static constexpr int TK = L::TK;
  uint32_t qf[HD / 16][4];
  float o[HD / 8][4];
  float m[2], l[2];
  int pos[2];

  __device__ __forceinline__ void start(const PagedParams& p, const PagedSeq& seq, const PagedItem<TK>& it, int kvh) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = min(lane / 4 + 8 * h, it.rows - 1) + it.r0;
      const int tok = r / p.group, head = kvh * p.group + r % p.group;
      pos[h] = seq.L - seq.T + tok;
      const T* src = static_cast<const T*>(p.q) + (seq.q0 + tok) * p.q_token + head * p.q_head + lane % 4 * 2;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        qf[kk][h] = *reinterpret_cast<const uint32_t*>(src + kk * 16);
        qf[kk][2 + h] = *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8);
      }
      m[h] = -INFINITY;
      l[h] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
  }

  __device__ __forceinline__ void tile(const PagedParams& p, uint32_t sk, int k0, bool whole) {
    const int lane = threadIdx.x & 31;
    const uint32_t sv = sk + L::TILE;
    float s[TK / 8][4];
#pragma unroll
    for (int n = 0; n < TK / 8; n += 2) {
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        uint32_t b[4];  // keys 8n .. 8n+7 at features 0-7, 8-15, then keys 8n+8 .. 8n+15
        ldmatrix_x4(sk + paged_rows_at<HD>(8 * n + (lane & 7) + (lane & 16 ? 8 : 0), 2 * kk + ((lane >> 3) & 1)), b);
        PT::mma(s0, qf[kk], b[0], b[1]);
        PT::mma(s1, qf[kk], b[2], b[3]);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        // (Never contracted into the subtraction of m below: m is such a product, rounded, and a huge score's rounding
        // would become an exponent.)
        s[n][x] = __fmul_rn(s0[x], p.scale_log2);
        s[n + 1][x] = __fmul_rn(s1[x], p.scale_log2);
      }
    }
    if (!whole) {
#pragma unroll
      for (int n = 0; n < TK / 8; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int key = k0 + 8 * n + lane % 4 * 2 + (x & 1), t = pos[x >> 1];
          if (key > t || (p.window > 0 && t - key >= p.window && key >= p.sinks)) s[n][x] = -INFINITY;
        }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < TK / 8; ++n) {
      top[0] = fmaxf(top[0], fmaxf(s[n][0], s[n][1]));
      top[1] = fmaxf(top[1], fmaxf(s[n][2], s[n][3]));
    }
    float base[2];
    bool moved = false;
    float corr[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 2));
      const float next = fmaxf(m[h], top[h]);
      base[h] = next == -INFINITY ? 0.f : next;  // a row that has seen no key: every 2^(s - 0) below is 0
      corr[h] = ex2_approx(m[h] - base[h]);
      moved |= next > m[h];
      m[h] = next;
      l[h] *= corr[h];
    }
    if (__any_sync(~0u, moved)) {
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        o[d][0] *= corr[0];
        o[d][1] *= corr[0];
        o[d][2] *= corr[1];
        o[d][3] *= corr[1];
      }
    }
#pragma unroll
    for (int n = 0; n < TK / 8; n += 2) {
      uint32_t pf[4];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float e0 = ex2_approx(s[n + g][0] - base[0]), e1 = ex2_approx(s[n + g][1] - base[0]);
        const float e2 = ex2_approx(s[n + g][2] - base[1]), e3 = ex2_approx(s[n + g][3] - base[1]);
        l[0] += e0 + e1;
        l[1] += e2 + e3;
        pf[2 * g] = PT::pack(e0, e1);
        pf[2 * g + 1] = PT::pack(e2, e3);
      }
#pragma unroll
      for (int d = 0; d < HD / 8; d += 2) {
        uint32_t b[4];  // keys 8n .. 8n+15 (two halves) at features 8d .. 8d+7, then the next eight
        ldmatrix_x4_trans(sv + paged_rows_at<HD>(8 * n + (lane & 15), d + (lane >> 4)), b);
        PT::mma(o[d], pf, b[0], b[1]);
        PT::mma(o[d + 1], pf, b[2], b[3]);
      }
    }
  }

  // Makes l the sums of whole rows.
  __device__ __forceinline__ void close() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(~0u, l[h], 1);
      l[h] += __shfl_xor_sync(~0u, l[h], 2);
    }
  }
  // Leaves the part (O unnormalised, m, l) at `slot`, laid out for 16 rows.
  __device__ __forceinline__ void leave(float* slot, int rows) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = lane / 4 + 8 * h;
      if (row >= rows) continue;
      if (lane % 4 == 0) {
        slot[16 * HD + row] = m[h];
        slot[16 * HD + 16 + row] = l[h];
      }
#pragma unroll
      for (int d = 0; d < HD / 8; ++d)
        *reinterpret_cast<float2*>(slot + row * HD + 8 * d + lane % 4 * 2) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
    }
  }
};

template <typename T, int HD>
__global__ void __launch_bounds__(PagedRowsLayout<HD>::THREADS, 1)
    paged_rows_kernel(const PagedParams p, int tpi, int min_tiles) {
  using L = PagedRowsLayout<HD>;
  using PT = Pair16<T>;
  constexpr int TK = L::TK, NST = L::NST;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PagedCut cuts[L::WARPS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = ((smem_u32(smem_raw) + 127) & ~127u) + warp * NST * L::STAGE;
  long long per;
  const int worker0 = blockIdx.x * L::WARPS;
  paged_schedule<TK, L::WARPS + 1, L::THREADS>(p, tpi, min_tiles, worker0, cuts, &per);
  paged_zero_outside(p, L::THREADS);
  pdl_trigger();
  const int worker = worker0 + warp;
  // Each warp finds the cut at which its piece begins, the last one also the end of the block's pieces.
  __shared__ PagedWalk<TK> found[L::WARPS + 1];
  for (int w = warp; w <= L::WARPS; w += L::WARPS) {
    PagedWalk<TK> x;
    x.b = p.batch;
    if (cuts[w].b >= 0) x.seek(p, cuts[w], tpi);
    if (lane == 0) found[w] = x;
  }
  __syncthreads();
  if (cuts[warp].b < 0) return;
  PagedWalk<TK> cur = found[warp];
  cur.end_at(found[warp + 1]);
  if (!cur.begin()) return;
  PagedWalk<TK> ahead = cur;
  bool more = true;  // `ahead` has a tile
  const uint64_t policy = policy_evict_first();

  // Copies the K and V tile under `ahead` into stage st and moves it on.
  auto fetch = [&](int st) {
    paged_rows_fetch<T, HD>(p, p.tables + ahead.s.slot * p.table_stride, ahead.s.L, ahead.kvh,
                            ahead.it.tile(ahead.i) * TK, ring + st * L::STAGE, policy);
    if (++ahead.i == ahead.i1) more = ahead.next(p, tpi);
  };

#pragma unroll
  for (int st = 0; st < NST - 1; ++st) {
    if (more) fetch(st);
    cp_async_commit();
  }

  PagedRows<T, HD> x;
  bool fresh = true;
  bool from_start = cur.i == 0;  // the current item's first tile is in this piece
  int st = 0;
  for (;;) {
    if (fresh) {
      fresh = false;
      x.start(p, cur.s, cur.it, cur.kvh);
    }
    if (more) fetch(st == 0 ? NST - 1 : st - 1);
    cp_async_commit();
    cp_async_wait<NST - 1>();
    __syncwarp();
    const uint32_t sk = ring + st * L::STAGE;
    if (++st == NST) st = 0;
    const int k0 = cur.it.tile(cur.i) * TK;
    x.tile(p, sk, k0, cur.it.whole(p, k0));
    __syncwarp();  // every lane has read the stage before a later round refills it

    if (++cur.i == cur.i1) {  // the item, or its part in this piece, is done
      x.close();
      if (cur.i1 == cur.it.n && from_start) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = lane / 4 + 8 * h;
          if (row >= cur.it.rows) continue;
          const float inv = x.l[h] > 0.f ? 1.f / x.l[h] : 0.f;
          const int r = cur.it.r0 + row, tok = cur.s.q0 + r / p.group, head = cur.kvh * p.group + r % p.group;
          T* dst = static_cast<T*>(p.out) + (static_cast<long long>(tok) * p.heads + head) * p.out_hd + lane % 4 * 2;
#pragma unroll
          for (int d = 0; d < HD / 8; ++d)
            if (8 * d < p.out_hd)
              *reinterpret_cast<uint32_t*>(dst + 8 * d) = PT::pack(x.o[d][2 * h] * inv, x.o[d][2 * h + 1] * inv);
        }
      } else {
        x.leave(p.part + (2ll * worker + (from_start ? 1 : 0)) * paged_slot_floats<16, HD>(), cur.it.rows);
      }
      fresh = true;
      from_start = true;
      if (!cur.next(p, tpi)) break;
    }
  }
  cp_async_wait<0>();
}

// Short chunks over short caches: one block per sequence and KV head, whose
// warps take the item's tiles in turn and join their parts in shared memory.
// No schedule and no second kernel, so the call is as short as its chain of
// loads (lengths, page numbers, keys); a long cache would leave the GPU to a
// few blocks.  64 sequences of up to 2048 tokens, 8 heads of 64 (131 MB): 30.9 us
// a call against 34.9 cut over the GPU; 64 windows of 1024 tokens, 8 KV heads of
// 128 (271 MB): 50 against 57, 5.4 TB/s.
constexpr int kItemWarps = 4;
template <int HD>
constexpr int kItemSmem = kItemWarps * PagedRowsLayout<HD>::NST * PagedRowsLayout<HD>::STAGE + 128;

template <typename T, int HD>
__global__ void __launch_bounds__(32 * kItemWarps) paged_item_kernel(const PagedParams p, int tpi) {
  using L = PagedRowsLayout<HD>;
  constexpr int TK = L::TK, NST = L::NST, THREADS = 32 * kItemWarps;
  constexpr int SLOT = static_cast<int>(paged_slot_floats<16, HD>());
  static_assert(kItemWarps * SLOT * 4 + 128 <= kItemSmem<HD>, "the parts take the ring's place");
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  const uint32_t ring = smem_u32(smem) + warp * NST * L::STAGE;
  float* parts = reinterpret_cast<float*>(smem);
  const int kvh = blockIdx.x, b = blockIdx.y;
  const PagedSeq s = paged_seq(p, b);
  if (kvh == 0 && b == 0) {  // rows of no sequence
    const int lo = min(max(p.cu_q[0], 0), p.n_tokens), hi = min(max(p.cu_q[p.batch], lo), p.n_tokens);
    const long long row = static_cast<long long>(p.heads) * p.out_hd / 8, n = (lo + p.n_tokens - hi) * row;
    for (long long i = threadIdx.x; i < n; i += THREADS)
      static_cast<uint4*>(p.out)[i < lo * row ? i : i - lo * row + hi * row] = make_uint4(0, 0, 0, 0);
  }
  const int* row = p.tables + s.slot * p.table_stride;
  const uint64_t policy = policy_evict_first();
  PagedItem<TK> it;
  for (int qt = 0; qt * tpi < s.T; ++qt) {
    it.set(p, s, qt, tpi);
    int ahead = warp;
#pragma unroll
    for (int st = 0; st < NST - 1; ++st, ahead += kItemWarps) {
      if (ahead < it.n) paged_rows_fetch<T, HD>(p, row, s.L, kvh, it.tile(ahead) * TK, ring + st * L::STAGE, policy);
      cp_async_commit();
    }
    PagedRows<T, HD> x;
    x.start(p, s, it, kvh);
    int st = 0;
#pragma unroll 1
    for (int i = warp; i < it.n; i += kItemWarps, ahead += kItemWarps) {
      if (ahead < it.n)
        paged_rows_fetch<T, HD>(p, row, s.L, kvh, it.tile(ahead) * TK, ring + (st == 0 ? NST - 1 : st - 1) * L::STAGE,
                                policy);
      cp_async_commit();
      cp_async_wait<NST - 1>();
      __syncwarp();
      const int k0 = it.tile(i) * TK;
      x.tile(p, ring + st * L::STAGE, k0, it.whole(p, k0));
      if (++st == NST) st = 0;
      __syncwarp();  // every lane has read the stage before a later round refills it
    }
    x.close();
    cp_async_wait<0>();
    __syncthreads();  // every ring is done with
    x.leave(parts + warp * SLOT, it.rows);
    __syncthreads();
    constexpr int TPR = HD / 4;
    for (int y = threadIdx.x; y < it.rows * TPR; y += THREADS) {
      const int r = y / TPR, d = y % TPR * 4;
      JoinSum sum = {parts[16 * HD + r], parts[16 * HD + 16 + r], *reinterpret_cast<const float4*>(parts + r * HD + d)};
#pragma unroll
      for (int w = 1; w < kItemWarps; ++w) {
        const float* q = parts + w * SLOT;
        sum.add(q[16 * HD + r], q[16 * HD + 16 + r], *reinterpret_cast<const float4*>(q + r * HD + d));
      }
      if (d >= p.out_hd) continue;
      const float inv = sum.l > 0.f ? 1.f / sum.l : 0.f;
      const int t = r / p.group, tok = s.q0 + qt * tpi + t, head = kvh * p.group + r - t * p.group;
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (static_cast<long long>(tok) * p.heads + head) * p.out_hd + d) =
          make_uint2(Pair16<T>::pack(sum.o.x * inv, sum.o.y * inv), Pair16<T>::pack(sum.o.z * inv, sum.o.w * inv));
    }
    __syncthreads();  // before the next item's copies
  }
}

}  // namespace tt
