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
from typing import Optional, Tuple

import numpy as np
import torch  # noqa: F401  (before the extension, which links its libraries)

from . import native
from .native import check

try:
    from . import _torch_ops as _ops
except ImportError as e:
    raise ImportError("rai_b200/_torch_ops.so is missing or does not fit this torch: build it with "
                      "`python -m rai_b200.build`") from e

ROPE_KINDS = {"plain": 0, "linear": 1, "ntk": 2, "llama3": 3, "yarn": 4}


def attention_workspace_bytes(q: torch.Tensor, k_pages: torch.Tensor, page_table: torch.Tensor, max_rows: int) -> int:
    """Bytes of the workspace that `attention` takes for these arguments."""
    return _ops.attention_workspace_bytes(q, k_pages, page_table, max_rows)


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
    return _ops.attention(q, k_pages, v_pages, page_table, kv_len, q_start, max_rows, scale, softcap, window, out, lse,
                          workspace)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                page_table: torch.Tensor, kv_len: torch.Tensor, q_start: torch.Tensor, inv_freq: torch.Tensor, *,
                interleaved: bool = False, mscale: float = 1.0, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate the chunk's q and k rows to their positions and store k and v in
    the pages (rai_gpu_rope_append). q [rows, heads, head_dim], k and v
    [rows, kv_heads, head_dim], views of one projection's output as well, in
    one type; the result and the pages in the pages' type. inv_freq (float32,
    device) has one frequency per pair; 2 * len(inv_freq) elements of a head
    turn. q_out may be q itself. Rows as in `attention`, kv_len counting them."""
    return _ops.rope_append(q, k, v, k_pages, v_pages, page_table, kv_len, q_start, inv_freq, interleaved, mscale, q_out)


def rope_frequencies(rot_dim: int, theta: float = 10000.0, kind: str = "plain", *, factor: float = 1.0, low: float = 1.0,
                     high: Optional[float] = None, original: float = 8192.0) -> Tuple[np.ndarray, float]:
    """(inv_freq, mscale) for `rope_append` (rai_rope_frequencies): kind plain,
    linear, ntk, llama3 (rai-infer/src/layers.rs:760-808) or yarn, for
    contexts `factor` times the `original` positions. `high` is 4 by default,
    for yarn 32 (the pairs that turn more often in `original` are kept)."""
    if kind not in ROPE_KINDS:
        raise ValueError(f"kind: one of {', '.join(ROPE_KINDS)}")
    if high is None:
        high = 32.0 if kind == "yarn" else 4.0
    out = np.zeros(max(rot_dim, 0) // 2, np.float32)
    m = C.c_float()
    check(native.lib().rai_rope_frequencies(ROPE_KINDS[kind], rot_dim, theta, factor, low, high, original, out.ctypes.data,
                                            C.byref(m)))
    return out, m.value


def fork(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, page_size: int, *,
         out_table: Optional[torch.Tensor] = None, out_lens: Optional[torch.Tensor] = None):
    """Sequence i of the result takes the pages of sequence parents[i] (-1:
    none); returns (table, lens), in new memory or in out_table, out_lens (as
    many rows as parents) (rai_gpu_kv_fork). refs is updated in place: sequences without children
    are freed, children of one parent share its pages. No page moves."""
    return _ops.fork(page_table, lens, refs, parents, page_size, out_table, out_lens)


def resize(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
           delta: int = 0, new_lens: Optional[torch.Tensor] = None,
           workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Resize every sequence in place to new_lens, or by delta tokens
    (rai_gpu_kv_resize): what shrinks releases its pages (length 0 frees it),
    what grows takes the lowest free pages, copying a shared last page first
    that is partly filled. k, v: the pages of every layer. Returns an int32
    [1] on the device: 0, or the number of pages missing, when nothing grew."""
    return _ops.resize(page_table, lens, refs, k, v, delta, new_lens, workspace)


def compact(page_table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
            workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Move the pages in use to the front of the pool, in place; tables and
    refs follow (rai_gpu_kv_compact). Every sequence that holds pages of the
    pool has to be in page_table. Returns the number of pages in use, int32
    [1] on the device."""
    return _ops.compact(page_table, lens, refs, k, v, workspace)


def copy_pages(k: torch.Tensor, v: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page src[i] to page dst[i] in every layer (rai_gpu_kv_copy_pages).
    No destination may occur twice or be a source."""
    _ops.copy_pages(k, v, src, dst)


def status(device=None) -> None:
    """Wait for the current stream and raise RaiError if a kernel-level call
    since the last query met a value on the device outside its tensors, or a
    device wait that gave up (rai_gpu_kernel_status). One word per device, that
    all threads and streams share: a report may be about another caller's call,
    and is not given twice."""
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        check(native.lib().rai_gpu_kernel_status(torch.cuda.current_stream().cuda_stream))


__all__ = ["attention", "attention_workspace_bytes", "compact", "copy_pages", "fork", "resize", "rope_append",
           "rope_frequencies", "status"]
