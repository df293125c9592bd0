// Host side of the paged K/V cache entry points (tt_cache_*, tt_paged_attention).
// Included once, at the end of tt_b200.cu, whose launch helpers it uses.
#pragma once

#include <cmath>
#include <exception>

#include "tt_cache.cuh"
#include "tt_paged_attn.cuh"
#include "tt_paged_chunk.cuh"

namespace {

// No C++ exception leaves a C entry point.
template <typename F>
int guarded(F f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return fail(TT_ERR_LAUNCH, "%s", e.what());
  } catch (...) {
    return fail(TT_ERR_LAUNCH, "unknown C++ exception");
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Checks the fields of a cache that every call uses, plus what `values` (K and
// V) and `counts` (refs) ask for, and fills the kernels' parameters.  The stride
// of a dimension of one entry addresses nothing: any will do, here and below.
int cache_params(const tt_kv_cache* c, bool values, bool counts, CacheParams* out) {
  if (!c || !c->tables || !c->lens || (counts && !c->refs) || (values && (!c->k || !c->v)))
    return fail(TT_ERR_ARG, "null cache field");
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128 && c->page != 256)
    return fail(TT_ERR_UNSUPPORTED, "page %d not in {16, 32, 64, 128, 256}", c->page);
  if (c->n_slots <= 0 || c->table_width <= 0 || c->n_pages <= 0 ||
      (c->n_slots > 1 && c->table_stride < c->table_width))
    return fail(TT_ERR_SHAPE, "invalid slots, table width, table stride or pages (%d, %d, %lld, %d)", c->n_slots,
                c->table_width, static_cast<long long>(c->table_stride), c->n_pages);
  if (static_cast<long long>(c->table_width) * c->page >= 1LL << 30)
    return fail(TT_ERR_SHAPE, "table rows of %d pages of %d tokens reach 2^30 tokens", c->table_width, c->page);
  memset(out, 0, sizeof(*out));
  out->tables = c->tables;
  out->table_stride = c->table_stride;
  out->lens = c->lens;
  out->refs = c->refs;
  out->n_pages = c->n_pages;
  out->n_slots = c->n_slots;
  out->table_width = c->table_width;
  while ((1 << out->page_shift) < c->page) ++out->page_shift;
  if (!values) return TT_OK;
  if (c->head_dim != 16 && c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(TT_ERR_UNSUPPORTED, "stored head_dim %d not in {16, 32, 64, 128, 256}", c->head_dim);
  if (c->layers <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535)
    return fail(TT_ERR_SHAPE, "invalid layers or kv_heads (%d, %d)", c->layers, c->kv_heads);
  const long long page_elems = static_cast<long long>(c->kv_heads) * c->page * c->head_dim;
  if (page_elems > 0x3fffffffLL) return fail(TT_ERR_SHAPE, "a page of %lld values is too large", page_elems);
  const long long k_page = c->n_pages > 1 ? c->k_page_stride : page_elems;
  const long long v_page = c->n_pages > 1 ? c->v_page_stride : page_elems;
  const long long k_layer = c->layers > 1 ? c->k_layer_stride : 0, v_layer = c->layers > 1 ? c->v_layer_stride : 0;
  if (!aligned16(c->k) || !aligned16(c->v) || (k_page | v_page | k_layer | v_layer) % 8 != 0)
    return fail(TT_ERR_ALIGN, "pools must be 16-byte aligned and their strides multiples of 8 elements");
  if (k_page < page_elems || v_page < page_elems)
    return fail(TT_ERR_SHAPE, "page strides are smaller than a page (%lld values)", page_elems);
  out->k = static_cast<uint8_t*>(c->k);
  out->v = static_cast<uint8_t*>(c->v);
  out->k_layer = k_layer * 2;
  out->v_layer = v_layer * 2;
  out->k_stride = k_page * 2;
  out->v_stride = v_page * 2;
  out->layers = c->layers;
  out->kv_heads = c->kv_heads;
  out->row_bytes = c->head_dim * 2;
  return TT_OK;
}

// ---------------------------------------------------------------- attention
// Sequences of at most this many query rows (tokens * group) take the kernels
// for short chunks, whose items hold that many rows.  In us, those against the
// chunk kernel: 16 rows, 16 sequences of 8000 keys, 8 KV heads of 128, 109 and
// 118 (64 of 2000, heads of 64: 62 and 101); 32 rows 195 and 128 (109 and 103).
constexpr int kRowsMax = 16;
// Key tiles that a worker takes at least: shorter pieces would cost more in
// joining than they save.
constexpr int kRowsMinTiles = 2, kChunkMinTiles = 4;
// What an item costs beside its key tiles (its queries, its output, the
// pipeline's run in and out), in tiles.  Ragged chunks over 8K caches, 424 items:
// 334 us with 2 for the chunk kernel, 300 with 4, 290 with 6, 294 with 12;
// calls whose items are alike do not depend on it.
constexpr int kRowsItemTiles = 3, kChunkItemTiles = 6;

template <int HD>
size_t paged_part_bytes(int sm_count) {
  const size_t rows = 2ull * sm_count * PagedRowsLayout<HD>::WARPS * paged_slot_floats<kRowsMax, HD>();
  const size_t chunk = 2ull * sm_count * paged_slot_floats<PagedChunkLayout<HD>::ROWS, HD>();
  return (rows > chunk ? rows : chunk) * sizeof(float);
}

int paged_workspace(int hd, int sm_count, size_t* bytes) {
  switch (hd) {
    case 8:
    case 16: *bytes = paged_part_bytes<16>(sm_count); return TT_OK;
    case 32: *bytes = paged_part_bytes<32>(sm_count); return TT_OK;
    case 64: *bytes = paged_part_bytes<64>(sm_count); return TT_OK;
    case 128: *bytes = paged_part_bytes<128>(sm_count); return TT_OK;
    case 256: *bytes = paged_part_bytes<256>(sm_count); return TT_OK;
    default: return fail(TT_ERR_UNSUPPORTED, "head_dim %d not in {8, 16, 32, 64, 128, 256}", hd);
  }
}

template <typename T, int HD, int TK, int ROWS, int RB, int THREADS>
int launch_paged_join(const PagedParams& p, int tpi, int min_tiles, cudaStream_t stream) {
  if (p.n_workers > kPagedMaxWorkers) return fail(TT_ERR_UNSUPPORTED, "%d workers", p.n_workers);
  PdlScope programmatic;
  launch_kernel(paged_join_kernel<T, HD, TK, ROWS, RB, THREADS>, dim3(p.n_workers - 1, ROWS / RB), THREADS, 0, stream, p,
                tpi, min_tiles);
  return after_launch("paged attention join");
}

// Sequences of row_lo .. row_hi query rows.
template <typename T, int HD>
int launch_paged_rows(PagedParams p, int row_lo, int row_hi, int sm_count, cudaStream_t stream) {
  using L = PagedRowsLayout<HD>;
  auto kern = paged_rows_kernel<T, HD>;
  if (int rc = prepare_kernel(kern, L::SMEM)) return rc;
  p.row_lo = row_lo;
  p.row_hi = row_hi;
  p.n_workers = sm_count * L::WARPS;
  p.item_len = kRowsItemTiles * L::TK;
  launch_kernel(kern, sm_count, L::THREADS, L::SMEM, stream, p, kRowsMax / p.group, kRowsMinTiles);
  if (int rc = after_launch("paged attention (rows)")) return rc;
  return launch_paged_join<T, HD, L::TK, kRowsMax, kRowsMax, 256>(p, kRowsMax / p.group, kRowsMinTiles, stream);
}

// Whether a call takes the kernel without cuts (one block per sequence and KV
// head): no sequence has more rows than fit an item, and none can have more
// cache in sight than a block streams in some 15 us.  In us, this against cut
// pieces, 8 KV heads of 128: one sequence of 500 keys 13 and 20, of 8000 98 and
// 52; 64 of 1000 54 and 62, 64 of 100 to 8000 217 and 193 (the last blocks run
// alone).  Lengths are on the device, so without a window it is the table's
// width that counts: the same short sequences in wider tables (at head_dim 64,
// of more than 2560 tokens) take the cut pieces.
constexpr long long kItemBytes = 640 * 1024;
bool paged_item_route(int stored_hd, long long max_rows, int window, int sinks, long long room) {
  const long long reach = static_cast<long long>(window) + sinks + kRowsMax;  // keys that a window leaves an item
  const long long keys = window > 0 && reach < room ? reach : room;
  return max_rows <= kRowsMax && keys * stored_hd * 4 <= kItemBytes;
}

template <typename T, int HD>
int launch_paged_item(const PagedParams& p, cudaStream_t stream) {
  auto kern = paged_item_kernel<T, HD>;
  if (int rc = prepare_kernel(kern, kItemSmem<HD>)) return rc;
  launch_kernel(kern, dim3(p.kv_heads, p.batch), 32 * kItemWarps, kItemSmem<HD>, stream, p, kRowsMax / p.group);
  return after_launch("paged attention (items)");
}

template <typename T, int HD>
int launch_paged_chunk(PagedParams p, int row_lo, int sm_count, cudaStream_t stream) {
  using L = PagedChunkLayout<HD>;
  auto kern = paged_chunk_kernel<T, HD>;
  KernelInfo ki;
  if (int rc = kernel_info(reinterpret_cast<const void*>(kern), L::SMEM, &ki)) return rc;
  if (L::SPLIT ? ki.regs != L::REGS_LAUNCH : ki.regs > 255)
    return fail(TT_ERR_UNSUPPORTED, "paged attention kernel built with %d registers per thread, expected %d", ki.regs,
                L::REGS_LAUNCH);
  p.row_lo = row_lo;
  p.row_hi = 0x7fffffff;
  p.n_workers = sm_count;
  p.item_len = kChunkItemTiles * L::BN;
  // This kernel masks and compares raw scores, which a positive factor does not
  // reorder: a negative scale's sign goes into Q K^T, and a scale of zero is
  // one so small that 2^(s - m) is 1 in FP32 for every score below 2^76.
  p.negate = p.scale_log2 < 0.f;
  p.scale_log2 = fmaxf(fabsf(p.scale_log2), 0x1p-100f);
  const int half_tokens = 128 / p.group, page = 1 << p.page_shift;
  CUtensorMap tq, tk, tv;
  {
    const uint64_t dims[3] = {HD, static_cast<uint64_t>(p.heads), static_cast<uint64_t>(p.n_tokens)};
    const uint64_t strides[2] = {static_cast<uint64_t>(p.q_head) * 2, static_cast<uint64_t>(p.q_token) * 2};
    const uint32_t box[3] = {L::ATOM, static_cast<uint32_t>(p.group), static_cast<uint32_t>(half_tokens)};
    if (int rc = encode_f16(&tq, p.q, 3, dims, strides, box)) return rc;
  }
  for (int kv = 0; kv < 2; ++kv) {
    const uint64_t dims[3] = {HD, static_cast<uint64_t>(p.kv_heads) * page, static_cast<uint64_t>(p.n_pages)};
    const uint64_t strides[2] = {HD * 2, static_cast<uint64_t>(kv ? p.v_stride : p.k_stride) * 2};
    const uint32_t box[3] = {L::ATOM, static_cast<uint32_t>(page < L::BN ? page : L::BN), 1};
    if (int rc = encode_f16(kv ? &tv : &tk, kv ? p.v_pages : p.k_pages, 3, dims, strides, box)) return rc;
  }
  launch_kernel(kern, sm_count, L::THREADS, L::SMEM, stream, tq, tk, tv, p, half_tokens, kChunkMinTiles);
  if (int rc = after_launch("paged attention (chunk)")) return rc;
  return launch_paged_join<T, HD, L::BN, L::ROWS, 32, 128>(p, L::NT * half_tokens, kChunkMinTiles, stream);
}

// Each sequence goes by its own number of query rows; max_rows only saves
// launches whose kernel could have no work.
template <typename T, int HD>
int launch_paged(const PagedParams& p, bool items, int max_rows, int sm_count, cudaStream_t stream) {
  if (items) return launch_paged_item<T, HD>(p, stream);
  const long long pairs = static_cast<long long>(p.batch) * p.kv_heads;
  // With a handful of (sequence, KV head) pairs a piece for every warp would
  // divide an item into a hundred parts, whose join grows with head_dim; the
  // chunk kernel has a piece per SM.  Single tokens over 8000 keys, in us on the
  // GPU, chunk kernel and this, with 8, 16 and 32 pairs:
  //   4 heads to a KV head of 256: 33 44, 41 48, 60 72; of 128: 24 37, 27 32, 37 36;
  //   of 64: 19 21, 23 22, 32 24; of 32: 17 13, 22 16, 31 19;
  //   one head to it, 256: 27 31, 37 41, 58 67; 128: 21 23, 26 25, 37 33;
  //   64: 18 17, 23 19, 32 23; 32: 17 13, 22 16, 31 19.
  constexpr int kFewPairs = HD == 256 ? 32 : HD == 128 ? 16 : 0;
  if (max_rows <= kRowsMax && pairs > kFewPairs)
    return launch_paged_rows<T, HD>(p, 0, 0x7fffffff, sm_count, stream);
  // With few (sequence, KV head) pairs the chunk kernel takes short sequences
  // along, at most two per SM: 8 sequences of 3000 keys, 8 KV heads of 128, 4 of them
  // with 300 new tokens, 114 us against 132 with a second pair of launches, 32 such 177
  // against 175, 64 such 263 against 241.
  if (p.group > kRowsMax || pairs <= 2ll * sm_count)
    return launch_paged_chunk<T, HD>(p, 0, sm_count, stream);
  if (int rc = launch_paged_chunk<T, HD>(p, kRowsMax + 1, sm_count, stream)) return rc;
  return launch_paged_rows<T, HD>(p, 0, kRowsMax, sm_count, stream);
}

template <typename T>
int launch_paged_t(const PagedParams& p, int hd, bool items, int max_rows, int sm_count, cudaStream_t stream) {
  switch (hd) {
    case 16: return launch_paged<T, 16>(p, items, max_rows, sm_count, stream);
    case 32: return launch_paged<T, 32>(p, items, max_rows, sm_count, stream);
    case 64: return launch_paged<T, 64>(p, items, max_rows, sm_count, stream);
    case 128: return launch_paged<T, 128>(p, items, max_rows, sm_count, stream);
    default: return launch_paged<T, 256>(p, items, max_rows, sm_count, stream);
  }
}

}  // namespace

extern "C" {

int tt_cache_reserve(const tt_kv_cache* cache, const int* cu_q, const int* slots, int batch, int* status,
                     void* stream) {
  return guarded([&]() -> int {
    DeviceState* ds;
    if (int rc = current_device_state(&ds)) return rc;
    CacheParams c;
    if (int rc = cache_params(cache, false, true, &c)) return rc;
    if (!status || !cu_q) return fail(TT_ERR_ARG, "null argument");
    if (batch < 0 || batch > kCacheMaxBatch)
      return fail(TT_ERR_SHAPE, "batch %d outside 0 .. %d", batch, kCacheMaxBatch);
    if (int rc = prepare_kernel(cache_reserve_kernel, kCacheMaxBatch * 4)) return rc;
    launch_kernel(cache_reserve_kernel, 1, kCacheThreads, static_cast<size_t>(batch) * 4,
                  static_cast<cudaStream_t>(stream), c, cu_q, slots, batch, status);
    return after_launch("cache reserve");
  });
}

int tt_cache_append(const tt_kv_cache* cache, const void* k, const int64_t* k_strides, const void* v,
                    const int64_t* v_strides, int n_tokens, const int* cu_q, const int* slots, int batch,
                    const int* status, void* stream) {
  return guarded([&]() -> int {
    DeviceState* ds;
    if (int rc = current_device_state(&ds)) return rc;
    CacheParams c;
    if (int rc = cache_params(cache, true, false, &c)) return rc;
    if ((n_tokens > 0 && (!k || !v)) || !k_strides || !v_strides || !cu_q) return fail(TT_ERR_ARG, "null argument");
    if (n_tokens < 0 || batch < 0) return fail(TT_ERR_SHAPE, "invalid n_tokens or batch (%d, %d)", n_tokens, batch);
    if (n_tokens == 0 || batch == 0) return TT_OK;
    AppendSrc src[2];
    const void* ptr[2] = {k, v};
    const int64_t* st[2] = {k_strides, v_strides};
    for (int i = 0; i < 2; ++i) {
      const char* name = i ? "v" : "k";
      src[i] = {static_cast<const uint16_t*>(ptr[i]), st[i][0], c.kv_heads > 1 ? st[i][1] : 0, st[i][2]};
      if (n_tokens == 1) src[i].token = st[i][2] == 1 ? 0 : 1;
      if (st[i][2] == 1) {
        if (!aligned16(ptr[i]) || src[i].token % 8 != 0 || src[i].head % 8 != 0)
          return fail(TT_ERR_ALIGN, "%s rows must be 16-byte aligned", name);
      } else if (src[i].token != 1) {
        return fail(TT_ERR_ARG, "%s must be dense in its features or in its tokens", name);
      }
    }
    const int smem = c.row_bytes / 2 * (kAppendTokens + 2) * 2;
    if (int rc = prepare_kernel(cache_append_kernel, smem)) return rc;
    launch_kernel(cache_append_kernel, dim3((n_tokens + kAppendTokens - 1) / kAppendTokens, c.kv_heads),
                  kAppendThreads, smem, static_cast<cudaStream_t>(stream), c, src[0], src[1], cu_q, slots, batch,
                  n_tokens, status);
    return after_launch("cache append");
  });
}

int tt_cache_release(const tt_kv_cache* cache, const int* slots, int n, int window, int sinks, void* stream) {
  return guarded([&]() -> int {
    DeviceState* ds;
    if (int rc = current_device_state(&ds)) return rc;
    CacheParams c;
    if (int rc = cache_params(cache, false, true, &c)) return rc;
    if (window < 0 || sinks < 0) return fail(TT_ERR_ARG, "window and sinks must not be negative (%d, %d)", window, sinks);
    if (n < 0 || (!slots && n > c.n_slots)) return fail(TT_ERR_SHAPE, "invalid slot count %d", n);
    if (n == 0) return TT_OK;
    launch_kernel(cache_release_kernel, n, 256, 0, static_cast<cudaStream_t>(stream), c, slots, n, window, sinks);
    return after_launch("cache release");
  });
}

int tt_cache_fork(const tt_kv_cache* cache, const int* parents, const int* children, int n, int* scratch, int* status,
                  void* stream) {
  return guarded([&]() -> int {
    DeviceState* ds;
    if (int rc = current_device_state(&ds)) return rc;
    CacheParams c;
    if (int rc = cache_params(cache, true, true, &c)) return rc;
    if ((n > 0 && (!parents || !children)) || !scratch || !status) return fail(TT_ERR_ARG, "null argument");
    constexpr int kMaxBits = kCacheMaxSlots / 32 * 4;
    if (n < 0 || n > kCacheMaxBatch || c.n_slots > kCacheMaxSlots || c.layers > 32767)
      return fail(TT_ERR_SHAPE, "fork takes at most %d pairs, %d slots and 32767 layers (got %d, %d, %d)",
                  kCacheMaxBatch, kCacheMaxSlots, n, c.n_slots, c.layers);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (int rc = prepare_kernel(cache_fork_plan_kernel, kCacheMaxBatch * 4 + kMaxBits)) return rc;
    launch_kernel(cache_fork_plan_kernel, 1, kCacheThreads, static_cast<size_t>(n) * 4 + (c.n_slots + 31) / 32 * 4, s, c,
                  parents, children, n, scratch, status);
    if (int rc = after_launch("cache fork plan")) return rc;
    if (n == 0) return TT_OK;
    launch_kernel(cache_fork_kernel, dim3(n, 2 * c.layers), 256, 0, s, c, parents, children,
                  static_cast<const int*>(scratch));
    return after_launch("cache fork");
  });
}

int tt_cache_compact(const tt_kv_cache* cache, int* scratch, int* live, void* stream) {
  return guarded([&]() -> int {
    DeviceState* ds;
    if (int rc = current_device_state(&ds)) return rc;
    CacheParams c;
    if (int rc = cache_params(cache, true, true, &c)) return rc;
    if (!scratch || !live) return fail(TT_ERR_ARG, "null argument");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    launch_kernel(cache_compact_plan_kernel, 1, kCacheThreads, 0, s, c, scratch, live);
    if (int rc = after_launch("cache compact plan")) return rc;
    launch_kernel(cache_compact_kernel, 4 * ds->sm_count, 512, 0, s, c, static_cast<const int*>(scratch));
    return after_launch("cache compact");
  });
}

int tt_cache_copy_pages(const tt_kv_cache* cache, const int* src, const int* dst, int n, void* stream) {
  return guarded([&]() -> int {
    DeviceState* ds;
    if (int rc = current_device_state(&ds)) return rc;
    CacheParams c;
    if (int rc = cache_params(cache, true, false, &c)) return rc;
    if (n > 0 && (!src || !dst)) return fail(TT_ERR_ARG, "null argument");
    if (n < 0) return fail(TT_ERR_SHAPE, "invalid page count %d", n);
    if (n == 0) return TT_OK;
    launch_kernel(cache_copy_pages_kernel, 4 * ds->sm_count, 512, 0, static_cast<cudaStream_t>(stream), c, src, dst, n);
    return after_launch("cache copy pages");
  });
}

int tt_paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim, int max_q_len, int window, int sinks,
                                       int table_width, int page, size_t* bytes) {
  return guarded([&]() -> int {
    DeviceState* ds;
    if (int rc = current_device_state(&ds)) return rc;
    if (!bytes) return fail(TT_ERR_ARG, "null argument");
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
      return fail(TT_ERR_SHAPE, "heads %d must be a multiple of kv_heads %d", heads, kv_heads);
    if (int rc = paged_workspace(head_dim, ds->sm_count, bytes)) return rc;
    if (max_q_len > 0 && paged_item_route(stored_head_dim(head_dim), static_cast<long long>(max_q_len) * (heads / kv_heads),
                                          window, sinks, static_cast<long long>(table_width) * page))
      *bytes = 0;
    return TT_OK;
  });
}

int tt_paged_attention(const tt_kv_cache* cache, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                       const int* cu_q, const int* slots, int batch, void* out, int n_tokens, int heads, int head_dim,
                       int is_bf16, float scale, int window, int sinks, int max_q_len, void* workspace,
                       size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    DeviceState* ds;
    if (int rc = current_device_state(&ds)) return rc;
    CacheParams c;
    if (int rc = cache_params(cache, true, false, &c)) return rc;
    if ((n_tokens > 0 && (!q || !out)) || !cu_q) return fail(TT_ERR_ARG, "null argument");
    if (n_tokens < 0 || batch < 0 || heads <= 0 || heads % c.kv_heads != 0 || heads / c.kv_heads > 128)
      return fail(TT_ERR_SHAPE, "invalid sizes (n_tokens %d, batch %d, heads %d, kv_heads %d)", n_tokens, batch, heads,
                  c.kv_heads);
    if (window < 0 || sinks < 0) return fail(TT_ERR_ARG, "window and sinks must not be negative (%d, %d)", window, sinks);
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!std::isfinite(scale_log2)) return fail(TT_ERR_ARG, "scale %g is not finite or too large", scale);
    size_t need = 0;
    if (int rc = paged_workspace(head_dim, ds->sm_count, &need)) return rc;
    if (stored_head_dim(head_dim) != cache->head_dim)
      return fail(TT_ERR_SHAPE, "head_dim %d is stored %d wide, the cache has %d", head_dim, stored_head_dim(head_dim),
                  cache->head_dim);
    const int group = heads / c.kv_heads;
    if (static_cast<long long>(n_tokens) * group >= 1LL << 30) return fail(TT_ERR_SHAPE, "too many query rows");
    const int max_rows = (max_q_len > 0 && max_q_len < n_tokens ? max_q_len : n_tokens) * group;
    if (batch == 0 && n_tokens > 0)  // no sequence has these rows
      return check_cuda(cudaMemsetAsync(out, 0, static_cast<size_t>(n_tokens) * heads * head_dim * 2,
                                        static_cast<cudaStream_t>(stream)),
                        "cudaMemsetAsync");
    const bool items = batch <= 65535 &&
                       paged_item_route(cache->head_dim, max_rows, window, sinks,
                                        static_cast<long long>(c.table_width) << c.page_shift);
    if (!items && (!workspace || workspace_bytes < need))
      return fail(TT_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
    if (n_tokens == 1) q_token_stride = static_cast<int64_t>(heads) * cache->head_dim;
    if (heads == 1) q_head_stride = cache->head_dim;
    if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || q_token_stride % 8 != 0 || q_head_stride % 8 != 0)
      return fail(TT_ERR_ALIGN, "q, out and workspace must be 16-byte aligned, q's strides multiples of 8");
    if (n_tokens == 0) return TT_OK;
    PagedParams p;
    memset(&p, 0, sizeof(p));
    p.q = q;
    p.q_token = q_token_stride;
    p.q_head = q_head_stride;
    p.k_pages = cache->k;
    p.v_pages = cache->v;
    p.k_stride = c.k_stride / 2;
    p.v_stride = c.v_stride / 2;
    p.tables = c.tables;
    p.table_stride = c.table_stride;
    p.lens = c.lens;
    p.cu_q = cu_q;
    p.slots = slots;
    p.out = out;
    p.part = static_cast<float*>(workspace);
    p.n_tokens = n_tokens;
    p.batch = batch;
    p.n_slots = c.n_slots;
    p.heads = heads;
    p.kv_heads = c.kv_heads;
    p.group = group;
    p.n_pages = c.n_pages;
    p.page_shift = c.page_shift;
    p.table_width = c.table_width;
    const int room = c.table_width << c.page_shift;  // no position reaches it
    p.window = window < room ? window : 0;
    p.sinks = sinks < room ? sinks : room;
    p.out_hd = head_dim;
    p.scale_log2 = scale_log2;
    p.err = ds->err;
    p.timeout_ns = g_timeout_ns.load();
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return is_bf16 ? launch_paged_t<__nv_bfloat16>(p, cache->head_dim, items, max_rows, ds->sm_count, s)
                   : launch_paged_t<__half>(p, cache->head_dim, items, max_rows, ds->sm_count, s);
  });
}

}  // extern "C"
