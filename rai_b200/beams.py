"""Beam search's choice on torch tensors (rai_gpu_beam_select): the best
continuations of every request's beams over the vocabulary. The parents it
returns are sequence numbers for rai_b200.paged.fork, which reorders the
beams' caches. rai-infer samples one stream at a time
(rai-infer/src/sampler.rs) and has no beam search.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .paged import _ops


class BeamChoice(NamedTuple):
    cand_scores: torch.Tensor  # float32 [batch, keep], best first
    cand_beams: torch.Tensor   # int32: the candidate's beam within its request
    cand_tokens: torch.Tensor  # int32
    scores: torch.Tensor       # float32 [batch, beams]: the beams that go on
    parents: torch.Tensor      # int32: sequence number request * beams + beam, -1: none
    tokens: torch.Tensor       # int32
    history: Optional[torch.Tensor] = None
    hist_len: Optional[torch.Tensor] = None


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
    return BeamChoice(*_ops.select(logits, scores, keep, eos, history, hist_len, workspace))


__all__ = ["BeamChoice", "select"]
