"""Thin PyTorch-tensor wrappers over the single-op entry points of libtt_b200.

Each wrapper validates dtypes/shapes, allocates its outputs with PyTorch on
the input's device, and launches on the current PyTorch stream of that
device.  Temporaries (FP32 copies of biases, the uint8 view of a mask) may be
released as soon as the call returns: PyTorch's caching allocator only hands
their memory to later work on the same stream, which runs after the kernel.  They exist for the per-kernel parity tests and for callers that
compose the ops themselves; the model path calls ``tt_model_forward`` once.
"""

from __future__ import annotations

from ctypes import byref, c_int64, c_size_t
from typing import Dict, Optional, Tuple

import torch

from ._lib import KVCache, check, lib


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _cuda(t: torch.Tensor, name: str) -> None:
    _need(t.is_cuda and t.is_contiguous(), f"{name} must be a contiguous CUDA tensor")


def stored_head_dim(head_dim: int) -> int:
    """Features per head of the q/k/v^T buffers: head_dim 8 is stored 16 wide."""
    return max(head_dim, 16)


def seq_pad_of(seq: int) -> int:
    """Row length of the V^T buffer: seq rounded up to a multiple of 8."""
    return (seq + 7) // 8 * 8


def layernorm_rows(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5,
                   out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """LayerNorm over the last dim of FP32 ``x``; FP16 or FP32 result."""
    _cuda(x, "x")
    _need(x.dtype == torch.float32, "x must be FP32")
    _need(out_dtype in (torch.float16, torch.float32), "out_dtype must be FP16 or FP32")
    d = x.shape[-1]
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().tt_layernorm_rows(x.data_ptr(), weight.float().contiguous().data_ptr(),
                                      bias.float().contiguous().data_ptr(), out.data_ptr(),
                                      x.numel() // d, d, float(eps), int(out_dtype == torch.float16),
                                      _stream(x)))
    return out


def qkv_projection(normalized: torch.Tensor, w_qkv: torch.Tensor, b_qkv: torch.Tensor, heads: int
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """normalized [B, S, D] FP16 -> q, k [B, H, S, hs] FP16 and v^T [B, H, hs, S_pad] FP16.

    hs = max(D // heads, 16): head_dim 8 is stored 16 wide (q/k features 8..15 zero).
    """
    _cuda(normalized, "normalized")
    _need(normalized.dtype == torch.float16 and w_qkv.dtype == torch.float16, "FP16 operands required")
    B, S, D = normalized.shape
    hs = stored_head_dim(D // heads)
    sp = seq_pad_of(S)
    q = torch.empty(B, heads, S, hs, dtype=torch.float16, device=normalized.device)
    k = torch.empty_like(q)
    vt = torch.zeros(B, heads, hs, sp, dtype=torch.float16, device=normalized.device)
    b32 = b_qkv.float().contiguous()
    with torch.cuda.device(normalized.device):
        check(lib().tt_qkv_projection(normalized.data_ptr(), w_qkv.contiguous().data_ptr(), b32.data_ptr(),
                                      q.data_ptr(), k.data_ptr(), vt.data_ptr(), B, S, D, heads, sp,
                                      _stream(normalized)))
    return q, k, vt


def attention(q: torch.Tensor, k: torch.Tensor, vt: torch.Tensor, scale: float, causal: bool = True,
              key_mask: Optional[torch.Tensor] = None, head_dim: Optional[int] = None) -> torch.Tensor:
    """q, k [B, H, S, hs], vt [B, H, hs, S_pad] FP16 -> context [B, S, H*hd] FP16.

    hd = head_dim (default hs); head_dim 8 takes qkv_projection's 16-wide layout.
    """
    for t, n in ((q, "q"), (k, "k"), (vt, "vt")):
        _cuda(t, n)
        _need(t.dtype == torch.float16, f"{n} must be FP16")
    B, H, S, hs = q.shape
    hd = hs if head_dim is None else int(head_dim)
    _need(stored_head_dim(hd) == hs, f"head_dim {hd} is stored {stored_head_dim(hd)} wide, got {hs}")
    sp = vt.shape[-1]
    ctx = torch.empty(B, S, H * hd, dtype=torch.float16, device=q.device)
    mask_ptr = 0
    kv_ptr = 0
    kv_end = None
    with torch.cuda.device(q.device):
        if key_mask is not None:
            m8 = key_mask.to(torch.bool).contiguous().view(torch.uint8)
            kv_end = torch.empty(B, dtype=torch.int32, device=q.device)
            check(lib().tt_mask_kv_end(m8.data_ptr(), B, S, kv_end.data_ptr(), _stream(q)))
            mask_ptr, kv_ptr = m8.data_ptr(), kv_end.data_ptr()
        check(lib().tt_causal_attention(q.data_ptr(), k.data_ptr(), vt.data_ptr(), mask_ptr, kv_ptr,
                                        ctx.data_ptr(), B, S, H, hd, sp, float(scale), int(causal),
                                        _stream(q)))
    return ctx


def linear_residual_layernorm(a: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, residual: torch.Tensor,
                              ln_weight: torch.Tensor, ln_bias: torch.Tensor, eps: float = 1e-5,
                              normalized_dtype: torch.dtype = torch.float16,
                              row_mask: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(residual + a @ w^T + bias, LayerNorm of it).  a FP16 [.., K], residual FP32 [.., D]."""
    _cuda(a, "a")
    _cuda(residual, "residual")
    _need(a.dtype == torch.float16 and w.dtype == torch.float16, "FP16 operands required")
    _need(residual.dtype == torch.float32, "residual must be FP32")
    K = a.shape[-1]
    D = residual.shape[-1]
    n = residual.numel() // D
    resid_out = torch.empty_like(residual)
    norm = torch.empty(residual.shape, dtype=normalized_dtype, device=a.device)
    mask_ptr = 0
    if row_mask is not None:
        m8 = row_mask.to(torch.bool).contiguous().view(torch.uint8)
        mask_ptr = m8.data_ptr()
    with torch.cuda.device(a.device):
        check(lib().tt_linear_residual_layernorm(
            a.data_ptr(), w.contiguous().data_ptr(), bias.float().contiguous().data_ptr(), residual.data_ptr(),
            ln_weight.float().contiguous().data_ptr(), ln_bias.float().contiguous().data_ptr(),
            resid_out.data_ptr(), norm.data_ptr(), n, K, D, float(eps),
            int(normalized_dtype == torch.float16), mask_ptr, _stream(a)))
    return resid_out, norm


def linear_gelu(a: torch.Tensor, w: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """GELU_erf(a @ w^T + bias) with FP16 operands, FP32 math, FP16 out."""
    _cuda(a, "a")
    _need(a.dtype == torch.float16 and w.dtype == torch.float16, "FP16 operands required")
    K = a.shape[-1]
    n_out = w.shape[0]
    n = a.numel() // K
    out = torch.empty(*a.shape[:-1], n_out, dtype=torch.float16, device=a.device)
    with torch.cuda.device(a.device):
        check(lib().tt_linear_gelu(a.data_ptr(), w.contiguous().data_ptr(), bias.float().contiguous().data_ptr(),
                                   out.data_ptr(), n, K, n_out, _stream(a)))
    return out


def ffn_residual_layernorm(a: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor, w2: torch.Tensor,
                           b2: torch.Tensor, residual: torch.Tensor, ln_weight: torch.Tensor,
                           ln_bias: torch.Tensor, eps: float = 1e-5,
                           normalized_dtype: torch.dtype = torch.float16,
                           row_mask: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(residual + GELU(a @ w1^T + b1) @ w2^T + b2, LayerNorm of it) in one fused kernel."""
    _cuda(a, "a")
    _cuda(residual, "residual")
    _need(a.dtype == torch.float16 and w1.dtype == torch.float16 and w2.dtype == torch.float16,
          "FP16 operands required")
    _need(residual.dtype == torch.float32, "residual must be FP32")
    D = residual.shape[-1]
    n = residual.numel() // D
    resid_out = torch.empty_like(residual)
    norm = torch.empty(residual.shape, dtype=normalized_dtype, device=a.device)
    mask_ptr = 0
    if row_mask is not None:
        m8 = row_mask.to(torch.bool).contiguous().view(torch.uint8)
        mask_ptr = m8.data_ptr()
    with torch.cuda.device(a.device):
        check(lib().tt_ffn_residual_layernorm(
            a.data_ptr(), w1.contiguous().data_ptr(), b1.float().contiguous().data_ptr(),
            w2.contiguous().data_ptr(), b2.float().contiguous().data_ptr(), residual.data_ptr(),
            ln_weight.float().contiguous().data_ptr(), ln_bias.float().contiguous().data_ptr(),
            resid_out.data_ptr(), norm.data_ptr(), n, D, w1.shape[0], float(eps),
            int(normalized_dtype == torch.float16), mask_ptr, _stream(a)))
    return resid_out, norm


# ---------------------------------------------------------------------------
# Paged K/V cache
#
# A cache is a few plain tensors: pages k, v [pages, kv_heads, page, hs] of one
# layer (or [layers, pages, ...] where a call moves every layer), int32 tables
# [slots, width] (-1: no page), lens [slots] and refs [pages].  A call's batch
# entry b is slot slots[b] (slot b without ``slots``), and its new tokens are
# rows cu_q[b] .. cu_q[b + 1] - 1 of the token tensors.  ``PagedKVCache`` keeps
# these tensors together.
# ---------------------------------------------------------------------------
PAGED_DTYPES = (torch.float16, torch.bfloat16)
PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (8, 16, 32, 64, 128, 256)


def _index(t: Optional[torch.Tensor], name: str, device: int, dims: int = 1) -> int:
    """Address of an int32 index tensor (0 for None)."""
    if t is None:
        return 0
    if t.dtype is not torch.int32 or t.get_device() != device or t.dim() != dims or (
            t.stride(1) != 1 < t.shape[1] if dims == 2 else not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 tensor of {dims} dimension(s) on cuda:{device}")
    return t.data_ptr()


def _cache(k: Optional[torch.Tensor], v: Optional[torch.Tensor], tables: torch.Tensor, lens: torch.Tensor,
           refs: Optional[torch.Tensor], page: int = 0) -> KVCache:
    """struct tt_kv_cache of checked tensors.  (Messages are built on failure only: a decode step makes this call for
    every layer.)"""
    if not tables.is_cuda:
        raise ValueError("tables must be a CUDA tensor")
    dev = tables.get_device()
    tables_at, lens_at, refs_at = _index(tables, "tables", dev, 2), _index(lens, "lens", dev), _index(refs, "refs", dev)
    slots, width = tables.shape
    if lens.shape[0] != slots:
        raise ValueError(f"lens has {lens.shape[0]} entries, tables {slots} rows")
    if k is None:
        return KVCache(None, None, 0, 0, 0, 0, tables_at, tables.stride(0), lens_at, refs_at, 0, refs.shape[0], 0, page, 0,
                       slots, width)
    shape = k.shape
    dims = len(shape)
    if dims not in (4, 5) or v.shape != shape:
        raise ValueError("k and v must be [pages, kv_heads, page, head_dim] pages of one layer, or [layers, pages, ...], "
                         "of one shape")
    if k.dtype not in PAGED_DTYPES or v.dtype is not k.dtype:
        raise ValueError("k and v pages must be FP16 or BF16")
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError(f"k and v pages must be on cuda:{dev}")
    layers, k_layer, v_layer = 1, 0, 0
    ks, vs = k.stride(), v.stride()
    if dims == 5:
        layers, k_layer, v_layer = shape[0], ks[0], vs[0]
        shape, ks, vs = shape[1:], ks[1:], vs[1:]
    pages, kv_heads, page, head_dim = shape
    dense = (page * head_dim, head_dim, 1)
    if (ks[1:] != dense or vs[1:] != dense) and not (kv_heads == 1 and ks[2:] == vs[2:] == dense[1:]):
        raise ValueError("each page of k and v must be contiguous")
    if refs is not None and refs.shape[0] != pages:
        raise ValueError(f"refs must have one entry for each of the {pages} pages")
    return KVCache(k.data_ptr(), v.data_ptr(), k_layer, v_layer, ks[0], vs[0], tables_at, tables.stride(0), lens_at, refs_at,
                   layers, pages, kv_heads, page, head_dim, slots, width)


# The handle of the device's current stream: the call PyTorch itself launches with where it exists.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _run(device: int, fn, cache: KVCache, *args) -> None:
    """Calls a libtt_b200 entry point on the device's current stream."""
    stream = _raw_stream(device)
    if torch.cuda.current_device() == device:
        rc = fn(byref(cache), *args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(byref(cache), *args, stream)
    if rc:
        check(rc)


def _reach(tokens: int) -> int:
    """A window or a number of first tokens for the 32-bit entry points: no position reaches 2^30."""
    return max(-1, min(int(tokens), 1 << 30))


def _batch(cu_q: torch.Tensor, slots: Optional[torch.Tensor], tables: torch.Tensor) -> Tuple[int, int, int]:
    """(address of cu_q, address of slots, sequences of the call)."""
    n, dev = cu_q.shape[0] - 1, tables.get_device()
    if n < 0:
        raise ValueError("cu_q needs at least one entry")
    if slots is None:
        if n > tables.shape[0]:
            raise ValueError(f"{n} sequences, but {tables.shape[0]} table rows")
    elif slots.shape[0] != n:
        raise ValueError(f"cu_q describes {n} sequences, slots {slots.shape[0]}")
    return _index(cu_q, "cu_q", dev), _index(slots, "slots", dev), n


def cache_reserve(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, cu_q: torch.Tensor, page: int,
                  slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Allocates the pages that the new tokens of (distinct) slots need and adds the tokens to ``lens``.

    All or nothing.  Returns an int32 status [1] on the device: 0 done, > 0 that many pages are
    missing, -1 a sequence would outgrow its table row, -2 a bad slot or cu_q.
    """
    c = _cache(None, None, tables, lens, refs, page)
    cu, sl, n = _batch(cu_q, slots, tables)
    status = torch.empty(1, dtype=torch.int32, device=tables.device)
    _run(tables.get_device(), lib().tt_cache_reserve, c, cu, sl, n, status.data_ptr())
    return status


_Strides = c_int64 * 3


def cache_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                 lens: torch.Tensor, cu_q: torch.Tensor, slots: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None) -> None:
    """Writes the new tokens' k, v [tokens, kv_heads, hs] into one layer's pages; ``lens`` counts them already.

    k and v may be strided views that are dense in their features, or dense in their tokens
    (``qkv_projection``'s vt as ``vt[0, :, :, :n].permute(2, 0, 1)``).  With the ``status`` of the
    ``cache_reserve`` that made the room, nothing is written where that was refused.
    """
    c = _cache(k_pages, v_pages, tables, lens, None)
    dev, want = tables.get_device(), (k.shape[0], c.kv_heads, c.head_dim)
    if k_pages.dim() != 4:
        raise ValueError("append writes one layer's pages")
    if k.shape != want or v.shape != want:
        raise ValueError(f"k and v must be [tokens, {want[1]}, {want[2]}]")
    if k.dtype is not k_pages.dtype or v.dtype is not k_pages.dtype or k.get_device() != dev or v.get_device() != dev:
        raise ValueError("k and v must have the pages' dtype and device")
    cu, sl, n = _batch(cu_q, slots, tables)
    _run(tables.get_device(), lib().tt_cache_append, c, k.data_ptr(), _Strides(*k.stride()), v.data_ptr(), _Strides(*v.stride()),
         want[0], cu, sl, n, _index(status, "status", dev))


def cache_release(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, page: int,
                  slots: Optional[torch.Tensor] = None, window: int = 0, sinks: int = 0) -> None:
    """Frees the slots (all without ``slots``), or with a window the pages that no later query of them can see."""
    c = _cache(None, None, tables, lens, refs, page)
    n = tables.shape[0] if slots is None else slots.shape[0]
    dev = tables.get_device()
    _run(dev, lib().tt_cache_release, c, _index(slots, "slots", dev), n, _reach(window), _reach(sinks))


def cache_fork(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor,
               refs: torch.Tensor, parents: torch.Tensor, children: torch.Tensor) -> torch.Tensor:
    """Makes each (empty, distinct) child slot a copy of its parent: full pages are shared, a partial one is copied.

    All or nothing.  Returns an int32 status [1]: 0 done, > 0 pages missing, -1 a parent without
    its last page, -2 a bad slot, -3 a child that is not empty or occurs twice.
    """
    c = _cache(k_pages, v_pages, tables, lens, refs)
    dev = tables.get_device()
    _need(parents.shape == children.shape, "parents and children must have one length")
    n = parents.shape[0]
    buf = torch.empty(2 * n + 2, dtype=torch.int32, device=tables.device)
    status = buf[:1]
    _run(dev, lib().tt_cache_fork, c, _index(parents, "parents", dev), _index(children, "children", dev), n,
         buf.data_ptr() + 4, status.data_ptr())
    return status


def cache_compact(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor,
                  refs: torch.Tensor) -> torch.Tensor:
    """Moves the live pages to the front of the pool, tables and refs with them; returns their number, int32 [1]."""
    c = _cache(k_pages, v_pages, tables, lens, refs)
    buf = torch.empty(3 * c.n_pages + 3, dtype=torch.int32, device=tables.device)
    live = buf[:1]
    _run(tables.get_device(), lib().tt_cache_compact, c, buf.data_ptr() + 4, live.data_ptr())
    return live


def cache_copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor,
                     src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies pages src[i] -> dst[i] of every layer (no destination twice, none of them a source)."""
    c = _cache(k_pages, v_pages, tables, lens, None)
    dev = tables.get_device()
    _need(src.shape == dst.shape, "src and dst must have one length")
    _run(dev, lib().tt_cache_copy_pages, c, _index(src, "src", dev), _index(dst, "dst", dev), src.shape[0])


_paged_ws_bytes: Dict[tuple, int] = {}


def _paged_workspace_bytes(key: tuple) -> int:
    device, batch_small, rows, heads, kv_heads, *rest = key
    nbytes = c_size_t()
    with torch.cuda.device(device):
        check(lib().tt_paged_attention_workspace_bytes(
            heads, kv_heads, rest[0], rows // (heads // kv_heads) if batch_small else 0, *rest[1:], nbytes))
    _paged_ws_bytes[key] = int(nbytes.value)
    return int(nbytes.value)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                    lens: torch.Tensor, cu_q: torch.Tensor, *, slots: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, window: int = 0, sinks: int = 0, head_dim: Optional[int] = None,
                    max_q_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of new tokens over one layer's pages -> [tokens, heads * hd] in the pages' dtype.

    q [tokens, heads, hs] (dense features, any token and head strides of whole 16 bytes); heads a
    multiple of the pages' kv_heads.  The T new tokens of a sequence are its last T positions
    (``lens`` counts them).  ``scale`` (hd ** -0.5 by default) is any finite number; scaled
    scores are at most 2^26 (FP32 keeps less than whole units of larger ones).  With ``window``
    a query sees the last ``window`` keys, itself included, and the first ``sinks`` ones.  A row that
    sees no key, or belongs to no sequence, is zero.
    ``head_dim`` 8 takes pages stored 16 wide; ``max_q_len``, if known, bounds every T.
    What a page holds past its sequence's length is never used; an infinity or NaN among a sequence's
    own keys and values may reach each of its rows, those whose mask hides it included.
    """
    c = _cache(k_pages, v_pages, tables, lens, None)
    dev = tables.get_device()
    n, heads, hs = q.shape
    st = q.stride()
    if k_pages.dim() != 4:
        raise ValueError("attention reads one layer's pages")
    if hs != c.head_dim or (n > 0 and st[2] != 1):
        raise ValueError(f"q must be [tokens, heads, {c.head_dim}], dense in its features")
    dtype = q.dtype
    if dtype is not k_pages.dtype or q.get_device() != dev:
        raise ValueError("q must have the pages' dtype and device")
    if heads % c.kv_heads or not heads:
        raise ValueError(f"{heads} query heads are not a multiple of {c.kv_heads} KV heads")
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    if window > 1 << 30 or sinks > 1 << 30:
        window, sinks = _reach(window), _reach(sinks)
    hd = hs if head_dim is None else int(head_dim)
    cu, sl, batch = _batch(cu_q, slots, tables)
    if out is None:
        out = torch.empty(n, heads * hd, dtype=dtype, device=q.device)
    elif (out.shape != (n, heads * hd) or out.dtype is not dtype or out.get_device() != dev or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous [{n}, {heads * hd}] tensor of q's dtype on cuda:{dev}")
    bound = n if max_q_len is None or not 0 < max_q_len < n else max_q_len
    rows = bound * (heads // c.kv_heads)
    # (More rows than an item holds: the workspace no longer depends on them.)
    key = (dev, batch < 65536, rows if rows <= 16 else 1 << 20, heads, c.kv_heads, hd, window, sinks, c.table_width, c.page)
    need = _paged_ws_bytes.get(key)
    if need is None:
        need = _paged_workspace_bytes(key)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _run(dev, lib().tt_paged_attention, c, q.data_ptr(), st[0], st[1], cu, sl, batch, out.data_ptr(), n, heads, hd,
         dtype is torch.bfloat16, hd ** -0.5 if scale is None else scale, window, sinks, bound,
         ws.data_ptr() if need else None, need)
    return out
