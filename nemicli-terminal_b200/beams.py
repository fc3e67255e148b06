"""Beam search's choice over the beams and the vocabulary (kernels: csrc/qmv_beam.cu; contract: include/nemicli_qmv.h,
qmv_beam_select), behind the vocabulary projection (`mmvq.mv`, `shard.RowShardedLinear`); `pages.reorder` then gives the beams
the tables they go on from.  The reference samples one sequence (ggufengine/sampling.py) and has no counterpart.
"""
from __future__ import annotations

import torch

from . import _lib

MOST = 64                                   # beams, and candidates a request
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def select(logits: torch.Tensor, scores: torch.Tensor, n: int = 0):
    """The n best continuations of each request.  logits: (requests, beams, vocab) of float32, bfloat16 or float16, the values of a row
    side by side; scores: float32 (requests, beams), the beams' log probabilities so far (-inf: no such beam).  n: default the
    beams; twice as many leave room for beams that end.  -> scores float32, parents int32, tokens int32, each (requests, n), best
    first: scores[r, parents] + log_softmax(logits[r, parents])[tokens], the lowest (beam, token) first among equals.  NaN counts as
    -inf, +inf as the largest float.  Two launches."""
    shape, dtype, device = logits.shape, _DTYPES.get(logits.dtype), logits.device
    if len(shape) != 3 or dtype is None or not logits.is_cuda:
        raise RuntimeError(f"beams.select: logits (requests, beams, vocab) of float32, bfloat16 or float16 on a CUDA device expected, "
                           f"got {logits.dtype} {tuple(shape)} on {device}")
    reqs, k, vocab = shape
    if scores.shape != (reqs, k) or scores.dtype is not torch.float32 or scores.device != device or not scores.is_contiguous():
        raise RuntimeError(f"beams.select: scores contiguous float32 ({reqs}, {k}) on {device} expected, got {scores.dtype} "
                           f"{tuple(scores.shape)} on {scores.device}")
    n = n or k
    if not 0 < k <= MOST or not 0 < n <= MOST or not 0 < vocab <= 1 << 30 or n > k * vocab or reqs * k > 65535:
        raise RuntimeError(f"beams.select: {reqs} requests of {k} beams over {vocab} tokens, {n} best: up to {MOST} beams and candidates, "
                           f"65535 beams in all")
    parents = torch.empty((reqs, n), dtype=torch.int32, device=device)
    tokens, out = torch.empty_like(parents), torch.empty((reqs, n), dtype=torch.float32, device=device)
    if reqs == 0:
        return out, parents, tokens
    by_req, by_beam, apart = logits.stride()
    if apart != 1 and vocab > 1 or k > 1 and by_beam < vocab or reqs > 1 and by_req != k * by_beam:
        logits = logits.contiguous()
        by_beam = vocab
    stride = by_beam if k > 1 else (by_req if reqs > 1 else vocab)
    lib = _lib.load()
    with _lib.on_device(device):
        nbytes = lib.qmv_beam_workspace_bytes(reqs, k, vocab, n)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        st = lib.qmv_beam_select(logits.data_ptr(), dtype, stride, reqs, k, vocab, scores.data_ptr(), n, out.data_ptr(),
                                 parents.data_ptr(), tokens.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_of(device))
    if st:
        _lib.check(st, "qmv_beam_select")
    return out, parents, tokens
