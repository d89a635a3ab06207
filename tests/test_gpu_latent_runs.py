"""Absorbed decode of more sequences than are divided into whole numbers of workgroups:
runs in which a workgroup ends one sequence and begins others."""
import numpy as np
import pytest
import torch

from infer_train_amd import BF16
from infer_train_amd.latent import LatentKvCache
from test_gpu_latent import DEV, decode_case, gen, normal

pytestmark = pytest.mark.gpu


def ragged(n, most, seed):
    """Lengths 0 to most: empty ones, single tokens, whole and broken tiles, one after another."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, most, n)
    lens[rng.random(n) < 0.15] = 0
    lens[rng.random(n) < 0.1] = 1
    lens[rng.random(n) < 0.1] = 64
    return [int(x) for x in lens[:-1]] + [most]


@pytest.mark.parametrize("dtype,latent,rope,heads,q_len,bound", [
    # one, two, four and eight groups of 16 queries a workgroup
    (torch.bfloat16, 512, 64, 28, 1, 0), (torch.bfloat16, 512, 64, 28, 1, 4096), (torch.float16, 512, 64, 64, 1, 0),
    (torch.bfloat16, 512, 64, 64, 1, 4096), (torch.bfloat16, 512, 64, 128, 1, 4096), (torch.float16, 512, 64, 128, 1, 0),
    # narrow rows, one and two
    (torch.float16, 256, 32, 40, 1, 0), (torch.float16, 256, 32, 40, 1, 4096), (torch.bfloat16, 256, 64, 64, 1, 4096),
    (torch.bfloat16, 128, 64, 48, 1, 4096),
    # drafted tokens
    (torch.bfloat16, 512, 64, 12, 4, 0), (torch.bfloat16, 512, 64, 32, 3, 4096), (torch.bfloat16, 512, 64, 48, 3, 4096),
    (torch.float16, 256, 32, 12, 5, 4096)])
@pytest.mark.parametrize("n", [65, 130])
def test_decode_many_sequences_in_runs(dtype, latent, rope, heads, q_len, bound, n):
    """A worker ends one sequence and begins others in its run."""
    decode_case(dtype, latent, rope, heads, ragged(n, 290, n + heads), q_len=q_len, poison=True, bound=bound, seed=n)


@pytest.mark.parametrize("heads,bound", [(28, 0), (64, 1 << 14), (128, 1 << 14)])
def test_decode_long_and_short_sequences_in_runs(heads, bound):
    """Sequences that several workers share, beside many that one takes; windows among them."""
    lens = ragged(80, 100, heads)
    for i, x in ((0, 2500), (33, 4000), (79, 1500)):
        lens[i] = x
    start = [x // 3 if i % 3 == 0 else 0 for i, x in enumerate(lens)]
    decode_case(torch.bfloat16, 512, 64, heads, lens, poison=True, bound=bound, start=start)


def test_decode_repeats_itself():
    """The same call gives the same bits: no sum depends on which workgroup is first."""
    g = gen(21)
    c = LatentKvCache(400, 16, 512, 64, BF16)
    c.view().copy_(normal(g, 400, 16, 576).to(torch.bfloat16))
    for n, heads in ((1, 28), (7, 64), (100, 28), (100, 128)):
        lens = torch.randint(0, 64 * 400 // (16 * n) if n < 8 else 300, (n,), generator=g, dtype=torch.int32).to(DEV)
        tables = torch.randint(0, 400, (n, 256), generator=g, dtype=torch.int32).to(DEV)
        q = normal(g, n, heads, 576).to(torch.bfloat16).to(DEV)
        first = c.decode(q[..., :512], q[..., 512:], tables, lens, 4096, 0.07)
        for _ in range(5):
            assert torch.equal(c.decode(q[..., :512], q[..., 512:], tables, lens, 4096, 0.07), first)
