"""Beam search's choice over the beams and the vocabulary (kernels: csrc/qmv_beam.cu; contract: include/nemicli_qmv.h,
qmv_beam_select), behind the vocabulary projection (`mmvq.mv`, `shard.RowShardedLinear`); `pages.reorder` then gives the beams
the tables they go on from.  The reference samples one sequence (ggufengine/sampling.py) and has no counterpart.
"""
from __future__ import annotations

import torch

from . import _lib


def select(logits: torch.Tensor, scores: torch.Tensor, n: int = 0):
    """The n best continuations of each request.  logits: (requests, beams, vocab) of float32, bfloat16 or float16, the values of a row
    side by side; scores: float32 (requests, beams), the beams' log probabilities so far (-inf: no such beam).  n: default the
    beams; twice as many leave room for beams that end; up to 64 of each.  -> scores float32, parents int32, tokens int32, each
    (requests, n), best first: scores[r, parents] + log_softmax(logits[r, parents])[tokens], the lowest (beam, token) first among
    equals (of a beam whose score is -inf or NaN its first tokens).  NaN counts as -inf, +inf as the largest float.  The
    same call gives the same bits; in a batch of another size a request's scores may differ in their last ones.  The three
    are parts of one allocation: clone what is kept for long, resize none.  Two launches."""
    return _lib.host().select(logits, scores, n)
