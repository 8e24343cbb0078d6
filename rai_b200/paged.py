"""Paged KV caches on torch tensors: rotary positions with the store into
pages, attention of a ragged chunk of new tokens, and the page operations
(fork, resize, compact, copy), over the entry points of include/rai_gpu.h.

A cache is two tensors of pages per layer, K and V, each [pages, kv_heads,
page_size, head_dim] (any strides whose vectors start on 16 bytes; float32,
float16 or bfloat16), an int32 table [sequences, max_pages] that names each
sequence's pages, its int32 lengths, and int32 reference counts [pages]. rai-infer's own
cache (rai-infer/src/kv_cache.rs:143-304) is one contiguous window per stream.

Everything runs on the current torch stream of the tensors' device, without a
host synchronisation, and can be captured in a CUDA graph (after one call
outside of a capture). Wrong arguments raise ValueError or RaiError at the
call; page numbers, lengths and row ranges on the device that pass the given
bounds are cut to them and raise at the next `status()`.

    q = rope_append(q, k, v, k_pages, v_pages, table, kv_len, q_start, inv_freq)
    o = attention(q, k_pages, v_pages, table, kv_len, q_start, max_rows)
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from typing import Optional, Tuple

import numpy as np
import torch

from . import native
from .native import check

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_CHUNK = "2Q6q3Qq9I4x"
_ATTN = struct.Struct(_CHUNK + "3Q4q2I2f2Q")
_ROPE = struct.Struct(_CHUNK + "5Q8q4If4x")
_TABLE = struct.Struct("3Qq4I")
_POOL = struct.Struct("2Q5q2I")
ROPE_KINDS = {"plain": 0, "linear": 1, "ntk": 2, "llama3": 3, "yarn": 4}


def _dtype(t: torch.Tensor, name: str) -> int:
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"{name}: float32, float16 or bfloat16, not {t.dtype}")
    return d


def _device(first: torch.Tensor, *rest: torch.Tensor) -> int:
    """The CUDA device that all tensors are on."""
    dev = first.get_device()
    for t in rest:
        if t.get_device() != dev:
            dev = -1
    if dev < 0:
        raise ValueError("every tensor has to be on one CUDA device")
    return dev


_lib = None  # native.lib(), looked up once
_current_device = torch.cuda.current_device
# The handle of a device's current stream, without the wrapper object that
# torch.cuda.current_stream makes (1 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)


def lib():
    global _lib
    if _lib is None:
        _lib = native.lib()
    return _lib


def _launch(dev: int, fn, *args) -> None:
    """fn(*args, stream) with the tensors' device current, on its current
    torch stream."""
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        check(rc)


_INT = torch.int32


def _ints(name: str, t: torch.Tensor, n: int) -> int:
    """Address of an int32 vector of n elements."""
    if t.dtype is not _INT or t.shape != (n,):
        raise ValueError(f"{name}: an int32 vector that fits the other arguments ({n}), not {t.dtype} {tuple(t.shape)}")
    if n > 1 and not t.is_contiguous():
        raise ValueError(f"{name}: has to be contiguous")
    return t.data_ptr()


def _cells(name: str, t: torch.Tensor, n: int):
    """Address, row stride and columns of an int32 table of n rows."""
    shape = t.shape
    if t.dtype is not _INT or len(shape) != 2 or shape[0] != n:
        raise ValueError(f"{name}: an int32 table of {n} rows, not {t.dtype} {tuple(shape)}")
    if t.is_contiguous():
        return t.data_ptr(), shape[1], shape[1]
    if shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the last dimension has to be contiguous")
    # A one-row table may have any row stride.
    return t.data_ptr(), t.stride(0) if n > 1 else max(t.stride(0), shape[1]), shape[1]


def _rows3(name: str, t: torch.Tensor, heads: Optional[int], dim: int):
    """The strides of a tensor of rows."""
    shape, st = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name}: [rows, heads, head_dim] that fits the pages, not {tuple(shape)}")
    if st[2] != 1 and dim > 1:
        raise ValueError(f"{name}: head_dim has to be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: this operator has no gradient; call it under torch.no_grad()")
    return st


def _chunk(k_pages, v_pages, table, kv_len, q_start, rows: int, max_rows: int, dtype: int):
    shape = k_pages.shape
    if len(shape) != 4 or shape != v_pages.shape or k_pages.dtype is not v_pages.dtype:
        raise ValueError("k_pages, v_pages: two tensors [pages, kv_heads, page_size, head_dim] of one shape and type")
    n_pages, nkv, page, hd = shape
    ks, vs = k_pages.stride(), v_pages.stride()
    if hd > 1 and (ks[3] != 1 or vs[3] != 1):
        raise ValueError("k_pages, v_pages: head_dim has to be contiguous")
    n = kv_len.shape[0]
    at, row, width = _cells("page_table", table, n)
    return (k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
            at, _ints("kv_len", kv_len, n), _ints("q_start", q_start, n + 1),
            row, n, width, n_pages, page, nkv, hd, rows, max_rows, dtype)


@functools.lru_cache(maxsize=1024)
def _attn_workspace(dev: int, dtype: int, hd: int, nkv: int, heads: int, max_rows: int, max_pages: int, page: int,
                    seqs: int) -> int:
    a = native.PagedAttention()
    a.chunk.dtype, a.chunk.head_dim, a.chunk.n_kv_heads, a.chunk.max_rows = dtype, hd, nkv, max_rows
    a.chunk.max_pages, a.chunk.page_size, a.chunk.n_seqs = max_pages, page, seqs
    a.n_heads = heads
    with torch.cuda.device(dev):
        return native.lib().rai_gpu_paged_attention_workspace_bytes(C.byref(a))


def attention_workspace_bytes(q: torch.Tensor, k_pages: torch.Tensor, page_table: torch.Tensor, max_rows: int) -> int:
    """Bytes of the workspace that `attention` takes for these arguments."""
    return _attn_workspace(q.get_device(), _dtype(k_pages, "k_pages"), k_pages.shape[3], k_pages.shape[1], q.shape[1],
                           min(max_rows, q.shape[0]), page_table.shape[1], k_pages.shape[2], page_table.shape[0])


def attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
              kv_len: torch.Tensor, q_start: torch.Tensor, max_rows: int, *, scale: Optional[float] = None,
              softcap: float = 0.0, window: int = 0, out: Optional[torch.Tensor] = None,
              lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each sequence's new rows (q[q_start[s]:q_start[s+1]],
    the last of its kv_len[s] tokens, at most max_rows of them) over its pages
    (rai_gpu_paged_attention). q [rows, heads, head_dim] in the pages' type;
    heads a multiple of the pages' KV heads. softcap > 0 caps the scores by
    softcap * tanh(s / softcap), window > 0 keeps the last `window` tokens.
    Rows that no sequence has are left as they are in `out` (undefined when
    `out` is not given). lse (float32 [rows, heads]) receives the rows'
    log-sum-exp. A row that sees nothing gives 0 and -inf."""
    dtype = _dtype(k_pages, "k_pages")
    hd = k_pages.shape[-1]
    qs = _rows3("q", q, None, hd)
    if q.dtype is not k_pages.dtype:
        raise ValueError(f"q: {k_pages.dtype} as the pages, not {q.dtype}")
    rows, heads = q.shape[0], q.shape[1]
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((rows, heads, hd))
        os = out.stride()
    else:
        os = _rows3("out", out, heads, hd)
        if out.shape[0] != rows or out.dtype is not q.dtype:
            raise ValueError("out: shape and type of q")
    dev = _device(q, k_pages, v_pages, page_table, kv_len, q_start, out)
    if rows == 0 or kv_len.shape[0] == 0 or max_rows == 0:
        return out
    if max_rows > rows:
        max_rows = rows
    chunk = _chunk(k_pages, v_pages, page_table, kv_len, q_start, rows, max_rows, dtype)
    lse_at = 0
    if lse is not None:
        if lse.dtype != torch.float32 or lse.shape != (rows, heads) or not lse.is_contiguous() or lse.get_device() != dev:
            raise ValueError("lse: contiguous float32 [rows, heads] on q's device")
        lse_at = lse.data_ptr()
    ws_at = ws_bytes = 0
    if workspace is None:
        need = _attn_workspace(dev, dtype, hd, chunk[16], heads, max_rows, chunk[13], chunk[15], chunk[12])
        if need:
            workspace = q.new_empty((need,), dtype=torch.uint8)
            ws_at, ws_bytes = workspace.data_ptr(), need
    else:
        if workspace.get_device() != dev or not workspace.is_contiguous():
            raise ValueError("workspace: contiguous, on q's device")
        ws_at, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    args = _ATTN.pack(*chunk, q.data_ptr(), out.data_ptr(), lse_at, qs[0], qs[1], os[0], os[1], heads, window,
                      hd ** -0.5 if scale is None else scale, softcap, ws_at, ws_bytes)
    _launch(dev, lib().rai_gpu_paged_attention, args)
    return out


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                page_table: torch.Tensor, kv_len: torch.Tensor, q_start: torch.Tensor, inv_freq: torch.Tensor, *,
                interleaved: bool = False, mscale: float = 1.0, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate the chunk's q and k rows to their positions and store k and v in
    the pages (rai_gpu_rope_append). q [rows, heads, head_dim], k and v
    [rows, kv_heads, head_dim], views of one projection's output as well, in
    one type; the result and the pages in the pages' type. inv_freq (float32,
    device) has one frequency per pair; 2 * len(inv_freq) elements of a head
    turn. q_out may be q itself. Rows as in `attention`, kv_len counting them."""
    dtype, hd, nkv = _dtype(k_pages, "k_pages"), k_pages.shape[-1], k_pages.shape[1]
    qs, ks, vs = _rows3("q", q, None, hd), _rows3("k", k, nkv, hd), _rows3("v", v, nkv, hd)
    rows, heads = q.shape[0], q.shape[1]
    in_dtype = _dtype(q, "q")
    if k.dtype is not q.dtype or v.dtype is not q.dtype or k.shape[0] != rows or v.shape[0] != rows:
        raise ValueError("q, k, v: one type and one number of rows")
    if inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq: a contiguous float32 vector")
    if q_out is None:
        q_out = q.new_empty((rows, heads, hd), dtype=k_pages.dtype)
        os = q_out.stride()
    else:
        os = _rows3("q_out", q_out, heads, hd)
        if q_out.shape[0] != rows or q_out.dtype is not k_pages.dtype:
            raise ValueError("q_out: q's shape in the pages' type")
    dev = _device(q, k, v, k_pages, v_pages, page_table, kv_len, q_start, inv_freq, q_out)
    if rows == 0 or kv_len.shape[0] == 0:
        return q_out
    args = _ROPE.pack(*_chunk(k_pages, v_pages, page_table, kv_len, q_start, rows, rows, dtype), q.data_ptr(), k.data_ptr(),
                      v.data_ptr(), q_out.data_ptr(), inv_freq.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0],
                      os[1], heads, 2 * inv_freq.shape[0], 1 if interleaved else 0, in_dtype, mscale)
    _launch(dev, lib().rai_gpu_rope_append, args)
    return q_out


def rope_frequencies(rot_dim: int, theta: float = 10000.0, kind: str = "plain", *, factor: float = 1.0, low: float = 1.0,
                     high: float = 4.0, original: float = 8192.0) -> Tuple[np.ndarray, float]:
    """(inv_freq, mscale) for `rope_append` (rai_rope_frequencies): kind plain,
    linear, ntk, llama3 (rai-infer/src/layers.rs:760-808) or yarn, for
    contexts `factor` times the `original` positions."""
    if kind not in ROPE_KINDS:
        raise ValueError(f"kind: one of {', '.join(ROPE_KINDS)}")
    out = np.zeros(max(rot_dim, 0) // 2, np.float32)
    m = C.c_float()
    check(native.lib().rai_rope_frequencies(ROPE_KINDS[kind], rot_dim, theta, factor, low, high, original, out.ctypes.data,
                                            C.byref(m)))
    return out, m.value


def _table(table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, page_size: int) -> bytes:
    n, pages = lens.shape[0], refs.shape[0]
    at, row, width = _cells("page_table", table, n)
    return _TABLE.pack(at, _ints("lens", lens, n), _ints("refs", refs, pages), row, n, width, pages, page_size)


def _pool(k: torch.Tensor, v: torch.Tensor):
    """(bytes of rai_page_pool, page size) of the K and V pages of every
    layer: [layers, pages, kv_heads, page_size, head_dim], or one layer's four
    dimensions, a page being one dense block."""
    shape, kst, vst = k.shape, k.stride(), v.stride()
    if shape != v.shape or k.dtype is not v.dtype or len(shape) not in (4, 5):
        raise ValueError("k, v: two tensors [layers, pages, kv_heads, page_size, head_dim] of one shape and type")
    _dtype(k, "k")
    if len(shape) == 4:
        shape, kst, vst = (1, *shape), (0, *kst), (0, *vst)
    e = k.element_size()
    layers, pages, heads, slots, dim = shape
    n = heads * slots * dim
    if (kst[2], kst[3], kst[4]) != (slots * dim, dim, 1) or vst != kst:
        for st in (kst, vst):
            # A page's block may order its heads and slots either way.
            want = 1
            for s, m in sorted((s, m) for s, m in zip(st[2:], shape[2:]) if m > 1):
                if s != want:
                    raise ValueError("k, v: every page has to be one contiguous block")
                want *= m
    # The stride of a single page or layer means nothing.
    kl, vl = (kst[0] * e, vst[0] * e) if layers > 1 else (0, 0)
    kp, vp = (kst[1] * e, vst[1] * e) if pages > 1 else (n * e, n * e)
    return _POOL.pack(k.data_ptr(), v.data_ptr(), kl, kp, vl, vp, n * e, layers, pages), slots


def fork(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, page_size: int, *,
         out_table: Optional[torch.Tensor] = None, out_lens: Optional[torch.Tensor] = None):
    """Sequence i of the result takes the pages of sequence parents[i] (-1:
    none); returns (table, lens), in new memory or in out_table, out_lens
    (rai_gpu_kv_fork). refs is updated in place: sequences without children
    are freed, children of one parent share its pages. No page moves."""
    n = parents.shape[0]
    if n == 0 or page_table.shape[0] == 0:
        raise ValueError("fork: no sequences")
    if out_table is None:
        out_table = page_table.new_empty((n, page_table.shape[1]))
    if out_lens is None:
        out_lens = lens.new_empty((n,))
    dev = _device(page_table, lens, refs, parents, out_table, out_lens)
    _launch(dev, lib().rai_gpu_kv_fork, _table(page_table, lens, refs, page_size),
            _table(out_table, out_lens, refs, page_size), _ints("parents", parents, n))
    return out_table, out_lens


def resize(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
           delta: int = 0, new_lens: Optional[torch.Tensor] = None,
           workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Resize every sequence in place to new_lens, or by delta tokens
    (rai_gpu_kv_resize): what shrinks releases its pages (length 0 frees it),
    what grows takes the lowest free pages, copying a shared last page first
    that is partly filled. k, v: the pages of every layer. Returns an int32
    [1] on the device: 0, or the number of pages missing, when nothing grew."""
    pool, page = _pool(k, v)
    dev = _device(page_table, lens, refs, k, v, lens if new_lens is None else new_lens)
    n = lens.shape[0]
    status = lens.new_empty((1,))
    if workspace is None:
        workspace = lens.new_empty((lib().rai_gpu_kv_resize_workspace_bytes(n),), dtype=torch.uint8)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("workspace: contiguous, on the tables' device")
    _launch(dev, lib().rai_gpu_kv_resize, _table(page_table, lens, refs, page), pool,
            _ints("new_lens", new_lens, n) if new_lens is not None else None, delta, status.data_ptr(),
            workspace.data_ptr(), workspace.numel() * workspace.element_size())
    return status


def compact(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
            workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Move the pages in use to the front of the pool, in place; tables and
    refs follow (rai_gpu_kv_compact). Every sequence that holds pages of the
    pool has to be in page_table. Returns the number of pages in use, int32
    [1] on the device."""
    pool, page = _pool(k, v)
    dev = _device(page_table, lens, refs, k, v)
    used = refs.new_empty((1,))
    if workspace is None:
        workspace = refs.new_empty((lib().rai_gpu_kv_compact_workspace_bytes(refs.shape[0]),), dtype=torch.uint8)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("workspace: contiguous, on the tables' device")
    _launch(dev, lib().rai_gpu_kv_compact, _table(page_table, lens, refs, page), pool, used.data_ptr(),
            workspace.data_ptr(), workspace.numel() * workspace.element_size())
    return used


def copy_pages(k: torch.Tensor, v: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page src[i] to page dst[i] in every layer (rai_gpu_kv_copy_pages).
    No destination may occur twice or be a source."""
    pool, _ = _pool(k, v)
    dev = _device(k, v, src, dst)
    n = src.shape[0]
    _launch(dev, lib().rai_gpu_kv_copy_pages, pool, _ints("src", src, n), _ints("dst", dst, n), n)


def status(device=None) -> None:
    """Wait for the current stream and raise RaiError if a kernel-level call
    since the last query met a value on the device outside its tensors, or a
    device wait that gave up (rai_gpu_kernel_status)."""
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        check(native.lib().rai_gpu_kernel_status(torch.cuda.current_stream().cuda_stream))


__all__ = ["attention", "attention_workspace_bytes", "compact", "copy_pages", "fork", "resize", "rope_append",
           "rope_frequencies", "status"]
