"""Edges of the rotary, sampling and move calls that the tests of their numerics leave out."""
import numpy as np
import pytest

from kvutil import to_dev

pytestmark = pytest.mark.gpu


def test_no_tokens_in_any_layout():
    """Of a tensor without tokens the strides mean nothing: whatever they are, the result is empty and the cache as it was."""
    import torch
    from infer_train_amd import F32
    from infer_train_amd.kv import PagedKvCache, Rotary

    r, pos, slots = Rotary(64), to_dev(np.zeros(0, np.int32)), to_dev(np.zeros(0, np.int64))
    cache = PagedKvCache(2, 16, 2, 64, F32)
    for x in (torch.zeros(2, 64, 5, device="cuda").permute(2, 0, 1)[:0], torch.zeros(1, 1, 1, device="cuda").expand(0, 2, 64)):
        assert x.shape == (0, 2, 64)
        assert r.apply(x, pos).shape == x.shape and r.apply(x, pos, out=x) is x
        assert cache.append_rotary(r, x, x, x, slots, pos).shape == x.shape
    assert not cache.k_pool.any()


def test_counts_past_the_parameter_keep_all():
    """top_k is 32 bits wide at the library: a larger number is no small one."""
    import torch
    from infer_train_amd.sampling import sample

    z = torch.from_numpy(np.random.default_rng(15).standard_normal((4, 5003)).astype(np.float32)).cuda()
    u = torch.tensor([0.1, 0.6, 0.99, 0.9999]).cuda()
    want = sample(z, u)
    for k in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 10 ** 30, -1, -2 ** 32 + 1):
        got = sample(z, u, top_k=k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k
