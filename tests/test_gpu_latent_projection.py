"""Queries turned inside a projection that holds the latent rows too."""
import pytest
import torch

from infer_train_amd import BF16, InvalidInput
from infer_train_amd.kv import Rotary
from infer_train_amd.latent import LatentKvCache
from test_gpu_latent import DEV, IDS, gen, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 2, 67])
@pytest.mark.parametrize("dtype,heads,nope,rope,latent,first", [(torch.bfloat16, 12, 128, 64, 512, "q"), (torch.bfloat16, 12, 128, 64, 512, "kv"),
                                                                (torch.float16, 1, 40, 32, 256, "q"), (torch.float32, 5, 64, 32, 128, "kv"),
                                                                (torch.bfloat16, 3, 30, 24, 72, "q")])
def test_append_turns_queries_inside_a_projection_that_holds_the_rows(n, dtype, heads, nope, rope, latent, first):
    g = gen(n + heads)
    width = heads * (nope + rope)
    one = normal(g, n, width + latent + rope + 8).to(dtype).to(DEV)

    def parts(x):
        at = 0 if first == "q" else latent + rope
        kv = x[:, width:width + latent + rope] if first == "q" else x[:, :latent + rope]
        return kv, x[:, at:at + width].unflatten(1, (heads, nope + rope))[..., nope:]

    caches = [LatentKvCache(8, 16, latent, rope, IDS[dtype]) for _ in range(2)]
    rotary, pos = Rotary(rope, layout="half"), torch.arange(n, dtype=torch.int32, device=DEV) * 37
    slots = torch.randperm(8 * 16, generator=g)[:n].to(DEV)
    kv, q = parts(one)
    want = caches[0].append(kv.clone(), slots, rotary, pos, q_rope=q.clone())
    before = one.clone()
    assert caches[1].append(kv, slots, rotary, pos, q_rope=q, q_out=q) is q
    assert torch.equal(q, want) and torch.equal(caches[0].view(), caches[1].view())
    parts(before)[1].copy_(want)
    assert torch.equal(one, before)  # nothing else in the projection changed
    # Out of one projection's queries into another part of it, the rows between.
    if n > 1 and first == "q":
        wide = torch.cat((before, before), 1)
        q = wide[:, :width].unflatten(1, (heads, nope + rope))[..., nope:]
        out = wide[:, width + latent + rope + 8:][:, :width].unflatten(1, (heads, nope + rope))[..., nope:]
        kv = wide[:, width:width + latent + rope]
        want = caches[0].append(kv.clone(), slots, rotary, pos, q_rope=q.clone())
        caches[1].append(kv, slots, rotary, pos, q_rope=q, q_out=out)
        assert torch.equal(out, want) and torch.equal(caches[0].view(), caches[1].view())


def test_append_still_refuses_what_overlaps():
    n, heads, rope, latent = 5, 4, 32, 256
    c = LatentKvCache(4, 16, latent, rope, BF16)
    slots, rotary, pos = torch.arange(n, device=DEV), Rotary(rope), torch.arange(n, dtype=torch.int32, device=DEV)
    one = torch.zeros(n + 2, 1024, dtype=torch.bfloat16, device=DEV)
    kv, q = one[:n, 512:512 + latent + rope], one[:n, :512].unflatten(1, (heads, 128))[..., :rope]
    flat = one.view(-1)
    at = lambda off, token=1024, head=128, h=heads: flat.as_strided((n, h, rope), (token, head, 1), off)  # noqa: E731
    for out, why in ((at(8), "a head onto a part of itself"), (at(128 - 31), "onto the next head"), (at(384), "the last heads onto the rows"),
                     (at(512 + latent - 8, h=2), "onto the row's rope part"), (at(1024 - 144), "onto the next token's queries"),
                     (at(700, head=64), "inside the row")):
        queries = q[:, :out.shape[1]]
        with pytest.raises(InvalidInput, match="overlap"):
            c.append(kv, slots, rotary, pos, q_rope=queries, q_out=out)
    rows = flat.as_strided((n, latent + rope), (latent + rope, 1), 600)
    with pytest.raises(InvalidInput, match="overlap"):
        c.append(kv, slots, rotary, pos, q_rope=q, rows_out=rows)
    c.append(kv, slots, rotary, pos, q_rope=q, q_out=at(32))  # between a head's elements and the next's
