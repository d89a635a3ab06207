"""The next token of every row of logits (it_sample): temperature, min-p,
top-k and top-p from given uniform numbers.  The reference's step ends with
ForwardExecutor::sample (src/inference/forward.rs:765-796)."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ._lib import call
from .kv import _check, _on, _raw_stream, torch_dtype_id

__all__ = ["sample", "sample_workspace"]


def sample_workspace(n_rows: int, vocab: int, device) -> torch.Tensor:
    """A workspace for `sample` (calls that overlap in time need one each);
    empty for short rows and large batches, which need none."""
    return torch.empty(call.it_sample_workspace(n_rows, vocab), dtype=torch.uint8, device=device)


def _per_row(t: torch.Tensor, name: str, dtype: torch.dtype, n: int, index: int) -> int:
    if t.dtype != dtype or t.numel() != n:
        raise TypeError(f"{name} must be {dtype}, one per row")
    if t.get_device() != index or not t.is_contiguous():
        return _on(t, index)  # which raises
    return t.data_ptr()


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
           top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
           min_p: Union[float, torch.Tensor] = 0.0, tokens: Optional[torch.Tensor] = None,
           probs: Optional[torch.Tensor] = None, ws: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """logits [n_rows, vocab] (float32, float16 or bfloat16, any row stride; at
    most 65535 rows of 262144 tokens),
    u float32 [n_rows] in [0, 1); temperature, top_k, top_p and min_p one
    number for all rows or a device tensor with one per row (float32; top_k
    int32).  Returns tokens int32 [n_rows] (-1 where a row holds nothing above
    -inf) and the probability float32 [n_rows] of each among the tokens kept."""
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] != 1):
        raise ValueError("logits must be [n_rows, vocab] with contiguous rows")
    if not logits.is_cuda:
        raise ValueError("device tensor expected")
    n, vocab = logits.shape
    index = logits.get_device()
    temperatures = top_ks = top_ps = min_ps = None
    if isinstance(temperature, torch.Tensor):
        temperatures, temperature = _per_row(temperature, "temperature", torch.float32, n, index), 1.0
    if isinstance(top_k, torch.Tensor):
        top_ks, top_k = _per_row(top_k, "top_k", torch.int32, n, index), 0
    else:  # no row has more than 2^18 tokens: a count past the parameter's width keeps them all
        top_k = min(max(int(top_k), 0), 2 ** 31 - 1)
    if isinstance(top_p, torch.Tensor):
        top_ps, top_p = _per_row(top_p, "top_p", torch.float32, n, index), 1.0
    if isinstance(min_p, torch.Tensor):
        min_ps, min_p = _per_row(min_p, "min_p", torch.float32, n, index), 0.0
    us = _per_row(u, "u", torch.float32, n, index)
    if tokens is None:
        tokens = torch.empty_like(u, dtype=torch.int32)
        at_tokens = tokens.data_ptr()
    else:
        at_tokens = _per_row(tokens, "tokens", torch.int32, n, index)
    if probs is None:
        probs = torch.empty_like(u)
        at_probs = probs.data_ptr()
    else:
        at_probs = _per_row(probs, "probs", torch.float32, n, index)
    need = 0
    if ws is None:
        need = call.it_sample_workspace(n, vocab)
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=logits.device)
    else:
        need = ws.nbytes
    args = (logits.data_ptr(), torch_dtype_id(logits.dtype), logits.stride(0), n, vocab, us, temperatures, top_ks, top_ps, min_ps,
            float(temperature), top_k, float(top_p), float(min_p), at_tokens, at_probs,
            None if ws is None else _on(ws, index), need, _raw_stream(index))
    if torch._C._cuda_getDevice() == index:
        _check(call.it_sample(*args))
    else:
        with torch.cuda.device(index):
            _check(call.it_sample(*args))
    return tokens, probs
