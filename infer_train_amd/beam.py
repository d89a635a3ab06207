"""Beam search's step: the best continuations of each request's beams
(it_beam_select), and their states put in the selected order (it_beam_reorder;
KvManager.reorder for the sequences' blocks).  The reference carries one
hypothesis (src/inference/forward.rs:765-796)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._lib import call
from .kv import _check, _grad_on, _on, _raw_stream, _refuse_gradient, _written, torch_dtype_id

__all__ = ["beam_select", "beam_select_workspace", "beam_reorder"]


def _launch(index: int, fn, *args) -> None:
    if torch._C._cuda_getDevice() == index:
        _check(fn(*args))
    else:
        with torch.cuda.device(index):
            _check(fn(*args))


def beam_select_workspace(n_groups: int, n_beams: int, vocab: int, n_out: int, device) -> torch.Tensor:
    """A workspace for `beam_select` (calls that overlap in time need one each)."""
    return torch.empty(call.it_beam_select_workspace(n_groups, n_beams, vocab, n_out), dtype=torch.uint8, device=device)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n_out: Optional[int] = None,
                ws: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """logits [n_groups * n_beams, vocab] (float32, float16 or bfloat16, any row
    stride), scores float32 [n_groups, n_beams] the beams' log-probabilities so
    far (-inf: a beam that is not in use, as all but one are at the start).
    Returns of each group's n_out best continuations (n_beams by default; twice
    as many leave enough beside those that end) their scores float32, parents
    int32 (the beam in its group) and tokens int32, [n_groups, n_out] each, best
    first, equal ones by the lower beam, larger logit and lower token; -inf, -1,
    -1 where there are no more.  The scores carry no gradient: logits and scores
    that require one are refused, unless gradients are off."""
    if _grad_on() and (logits.requires_grad or scores.requires_grad):
        _refuse_gradient("beam_select")
    strides, index = logits.stride(), logits.get_device()
    if len(strides) != 2 or (strides[1] != 1 and logits.shape[1] != 1):
        raise ValueError("logits must be [n_groups * n_beams, vocab] with contiguous rows")
    if index < 0:
        raise ValueError("device tensor expected")
    rows, vocab = logits.shape
    if scores.dtype != torch.float32 or scores.dim() != 2 or scores.numel() != rows:
        raise TypeError("scores must be float32 [n_groups, n_beams], one per row of logits")
    groups, beams = scores.shape
    n = beams if n_out is None else int(n_out)
    at_scores = _on(scores, index)
    device = logits.device
    if ws is None:
        ws = beam_select_workspace(groups, beams, vocab, n, device)
    best = torch.empty((3, groups, n), dtype=torch.int32, device=device)
    at, part = best.data_ptr(), 4 * groups * n
    _launch(index, call.it_beam_select, logits.data_ptr(), torch_dtype_id(logits.dtype), strides[0], groups, beams, vocab,
            at_scores, n, at, at + part, at + 2 * part, _on(ws, index), ws.nbytes, _raw_stream(index))
    best_scores, parents, tokens = best.unbind()
    return best_scores.view(torch.float32), parents, tokens


def beam_reorder(x: torch.Tensor, parents: torch.Tensor, dim: int = 0) -> torch.Tensor:
    """Per-beam states x (contiguous, any dtype; n_groups * n_beams rows along
    `dim`) put in the order of int32 parents [n_groups, n_beams], in place: row
    g * n_beams + j becomes what row g * n_beams + parents[g, j] was; a parent
    below 0 leaves it.  Block tables, token histories, recurrent states.
    Returns x."""
    if parents.dtype != torch.int32 or parents.dim() != 2:
        raise TypeError("parents must be int32 [n_groups, n_beams]")
    if x.requires_grad and _grad_on():
        _refuse_gradient("beam_reorder")
    if not -x.dim() <= dim < x.dim():
        raise ValueError(f"dim {dim} of a tensor of {x.dim()} dimensions")
    dim %= x.dim()
    if x.shape[dim] != parents.numel():
        raise ValueError(f"{x.shape[dim]} rows, {parents.numel()} parents")
    if not x.is_cuda:
        raise ValueError("device tensor expected")
    index = x.get_device()
    at, rows = _on(x, index), x.shape[dim]
    outer = 1
    for s in x.shape[:dim]:
        outer *= s
    row = x.element_size() * (x.numel() // (outer * rows) if outer * rows else 0)
    _launch(index, call.it_beam_reorder, at, row, row, outer, row * rows, parents.shape[0], parents.shape[1], _on(parents, index),
            _raw_stream(index))
    _written(x)
    return x
