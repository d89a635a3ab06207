"""Latent attention and beam selection carry no gradient, and say so."""
import pytest
import torch

from infer_train_amd import F32
from infer_train_amd.beam import beam_select
from infer_train_amd.kv import Rotary
from infer_train_amd.latent import LatentKvCache, latent_prefill
from test_gpu_latent import DEV, gen, normal

pytestmark = pytest.mark.gpu


def test_inputs_that_require_gradients_are_refused():
    """No call here carries one: what would be lost in silence is refused, unless gradients are off."""
    g, n = gen(23), 6
    z = lambda *s: normal(g, *s).to(DEV)  # noqa: E731
    c = LatentKvCache(4, 16, 64, 32, F32)
    slots, rotary, pos = torch.arange(n, device=DEV), Rotary(32), torch.arange(n, dtype=torch.int32, device=DEV)
    append = lambda kv, w, q, out=None, rows=None: c.append(kv, slots, rotary, pos, weight=w, q_rope=q, q_out=out, rows_out=rows)  # noqa: E731
    tables, lens = torch.zeros(n, 1, dtype=torch.int32, device=DEV), torch.ones(n, dtype=torch.int32, device=DEV)
    decode = lambda ql, qr, out=None: c.decode(ql, qr, tables, lens, 16, 0.1, out=out)  # noqa: E731
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    prefill = lambda q, k, v, r, out=None: latent_prefill(q, k, v, r, cu, cu, n, n, 0.1, out=out)  # noqa: E731
    calls = ((append, (z(n, 96), z(64), z(n, 2, 32), z(n, 2, 32), z(n, 96))), (decode, (z(n, 2, 64), z(n, 2, 32), z(n, 2, 64))),
             (prefill, (z(n, 2, 96), z(n, 2, 64), z(n, 2, 64), z(n, 32), z(n, 2, 64))), (beam_select, (z(n, 100), z(3, 2))))
    for fn, args in calls:
        fn(*args)
        for i in range(len(args)):
            leaf = [a.clone().requires_grad_() if j == i else a for j, a in enumerate(args)]
            with pytest.raises(ValueError, match="gradient"):
                fn(*leaf)
            with torch.no_grad():
                fn(*leaf)
            with torch.inference_mode():
                fn(*leaf)


def test_outputs_given_by_the_caller_show_that_they_changed():
    """A tensor saved for a backward pass and then written here is found out."""
    g, n = gen(24), 3
    z = lambda *s: normal(g, *s).to(DEV)  # noqa: E731
    c = LatentKvCache(4, 16, 64, 32, F32)
    slots = torch.arange(n, device=DEV)
    tables, lens = torch.zeros(n, 1, dtype=torch.int32, device=DEV), torch.ones(n, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    q = z(n, 2, 32)
    rows, out, pre = z(n, 96), z(n, 2, 64), z(n, 2, 64)
    for t, fn in ((q, lambda: c.append(z(n, 96), slots, q_rope=q, q_out=q)), (rows, lambda: c.append(z(n, 96), slots, rows_out=rows)),
                  (out, lambda: c.decode(z(n, 2, 64), z(n, 2, 32), tables, lens, 16, 0.1, out=out)),
                  (pre, lambda: latent_prefill(z(n, 2, 96), z(n, 2, 64), z(n, 2, 64), z(n, 32), cu, cu, n, n, 0.1, out=pre))):
        w = torch.ones_like(t, requires_grad=True)
        loss = (w * t).sum()
        version = t._version
        fn()
        assert t._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.inference_mode():
            fn()
