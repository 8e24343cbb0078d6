"""Beam search's choice on torch tensors (rai_gpu_beam_select): the best
continuations of every request's beams over the vocabulary. The parents it
returns are sequence numbers for rai_b200.paged.fork, which reorders the
beams' caches. rai-infer samples one stream at a time
(rai-infer/src/sampler.rs) and has no beam search.
"""
from __future__ import annotations

import functools
import struct
from typing import NamedTuple, Optional

import torch

from . import native
from .paged import _cells, _device, _dtype, _ints, _launch, lib

_ARGS = struct.Struct("2Qq6Q4Q2q5IiI4x2Q")


class BeamChoice(NamedTuple):
    cand_scores: torch.Tensor  # float32 [batch, keep], best first
    cand_beams: torch.Tensor   # int32: the candidate's beam within its request
    cand_tokens: torch.Tensor  # int32
    scores: torch.Tensor       # float32 [batch, beams]: the beams that go on
    parents: torch.Tensor      # int32: sequence number request * beams + beam, -1: none
    tokens: torch.Tensor       # int32
    history: Optional[torch.Tensor] = None
    hist_len: Optional[torch.Tensor] = None


@functools.lru_cache(maxsize=256)
def _workspace(dev: int, batch: int, beams: int, vocab: int, keep: int) -> int:
    with torch.cuda.device(dev):
        return native.lib().rai_gpu_beam_workspace_bytes(batch, beams, vocab, keep)


def select(logits: torch.Tensor, scores: torch.Tensor, *, keep: Optional[int] = None, eos: int = -1,
           history: Optional[torch.Tensor] = None, hist_len: Optional[torch.Tensor] = None,
           workspace: Optional[torch.Tensor] = None) -> BeamChoice:
    """Choose among the beams x vocabulary continuations of each request by
    scores + log_softmax(logits): the `keep` best (2 * beams by default, so
    that beams that end leave enough), and the first `beams` of them whose
    token is not eos. logits [batch, beams, vocab] (float32, float16 or
    bfloat16; rows evenly spaced), scores float32 [batch, beams] (-inf for
    beams that do not count). Candidates are ordered by score in 64 bits, then
    logit, then beam and token. With history (int32 [batch * beams, capacity])
    and hist_len the beams' token histories are reordered and extended."""
    dtype = _dtype(logits, "logits")
    if logits.dim() != 3:
        raise ValueError("logits: [batch, beams, vocab]")
    b, n, v = logits.shape
    if keep is None:
        keep = 2 * n
    if v > 1 and logits.stride(2) != 1:
        raise ValueError("logits: vocab has to be contiguous")
    row = logits.stride(1) if n > 1 else logits.stride(0) if b > 1 else v
    if n > 1 and b > 1 and logits.stride(0) != n * row:
        raise ValueError("logits: rows have to be evenly spaced")
    if scores.dtype != torch.float32 or scores.shape != (b, n) or not scores.is_contiguous():
        raise ValueError("scores: contiguous float32 [batch, beams]")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("logits: this operator has no gradient; call it under torch.no_grad()")
    dev = _device(logits, scores)
    if b == 0 or n == 0 or v == 0:
        raise ValueError("logits: a size is zero")
    cs, sc = scores.new_empty((b, keep)), torch.empty_like(scores)
    cb, ct = scores.new_empty((2, b, keep), dtype=torch.int32).unbind(0)
    pa, tk = scores.new_empty((2, b, n), dtype=torch.int32).unbind(0)
    hist = [0, 0, 0, 0, 0, 0, 0]
    out_h = out_n = None
    if history is not None:
        if hist_len is None:
            raise ValueError("hist_len: needed with history")
        _device(logits, history, hist_len)
        out_h = torch.empty_like(history, memory_format=torch.contiguous_format)
        out_n = torch.empty_like(hist_len)
        at, row_h, cap = _cells("history", history, b * n)
        hist = [at, _ints("hist_len", hist_len, b * n), out_h.data_ptr(), out_n.data_ptr(), row_h, max(cap, 1), cap]
    if workspace is None:
        workspace = scores.new_empty((_workspace(dev, b, n, v, keep),), dtype=torch.uint8)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("workspace: contiguous, on the logits' device")
    args = _ARGS.pack(logits.data_ptr(), scores.data_ptr(), row, cs.data_ptr(), cb.data_ptr(), ct.data_ptr(), sc.data_ptr(),
                      pa.data_ptr(), tk.data_ptr(), *hist, b, n, v, keep, eos, dtype, workspace.data_ptr(),
                      workspace.numel() * workspace.element_size())
    _launch(dev, lib().rai_gpu_beam_select, args)
    return BeamChoice(cs, cb, ct, sc, pa, tk, out_h, out_n)


__all__ = ["BeamChoice", "select"]
