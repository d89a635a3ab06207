"""The next token of every row of logits (it_sample): temperature, min-p,
top-k and top-p from given uniform numbers.  The reference's step ends with
ForwardExecutor::sample (src/inference/forward.rs:765-796)."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ._lib import call
from .kv import _check, _ptr, _raw_stream, torch_dtype_id

__all__ = ["sample", "sample_workspace"]


def sample_workspace(n_rows: int, vocab: int, device) -> torch.Tensor:
    """A workspace for `sample` (calls that overlap in time need one each)."""
    return torch.empty(call.it_sample_workspace(n_rows, vocab), dtype=torch.uint8, device=device)


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
           top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
           min_p: Union[float, torch.Tensor] = 0.0, tokens: Optional[torch.Tensor] = None,
           probs: Optional[torch.Tensor] = None, ws: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """logits [n_rows, vocab] (float32, float16 or bfloat16, any row stride),
    u float32 [n_rows] in [0, 1); temperature, top_k, top_p and min_p one
    number for all rows or a device tensor with one per row (float32; top_k
    int32).  Returns tokens int32 [n_rows] (-1 where a row holds nothing above
    -inf) and the probability float32 [n_rows] of each among the tokens kept."""
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] != 1):
        raise ValueError("logits must be [n_rows, vocab] with contiguous rows")
    if not logits.is_cuda:
        raise ValueError("device tensor expected")
    n, vocab = logits.shape
    arrays, numbers = [], []
    for name, x, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if isinstance(x, torch.Tensor):
            if x.dtype != dtype or x.numel() != n:
                raise TypeError(f"{name} must be {dtype}, one per row")
            arrays.append(_ptr(x))
            numbers.append(0)
        else:
            arrays.append(None)
            numbers.append(x)
    if u.dtype != torch.float32 or u.numel() != n:
        raise TypeError("u must be float32, one per row")
    if tokens is None:
        tokens = torch.empty(n, dtype=torch.int32, device=logits.device)
    elif tokens.dtype != torch.int32 or tokens.numel() != n:
        raise TypeError("tokens must be int32, one per row")
    if probs is None:
        probs = torch.empty(n, dtype=torch.float32, device=logits.device)
    elif probs.dtype != torch.float32 or probs.numel() != n:
        raise TypeError("probs must be float32, one per row")
    if ws is None:
        ws = sample_workspace(n, vocab, logits.device)
    index = logits.device.index
    args = (logits.data_ptr(), torch_dtype_id(logits.dtype), logits.stride(0), n, vocab, _ptr(u), *arrays,
            float(numbers[0]), int(numbers[1]), float(numbers[2]), float(numbers[3]), _ptr(tokens), _ptr(probs), _ptr(ws),
            ws.numel() * ws.element_size(), _raw_stream(index))
    if torch.cuda.current_device() == index:
        _check(call.it_sample(*args))
    else:
        with torch.cuda.device(index):
            _check(call.it_sample(*args))
    return tokens, probs
