"""Infinite values in the expanded form: in every sum that they belong to, and in no
other, wherever their keys stand among the blocks."""
import pytest
import torch

from infer_train_amd.latent import latent_prefill
from test_gpu_latent import DEV, INF, gen, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,nope,rope,v_dim", [(torch.bfloat16, 128, 64, 128), (torch.float16, 64, 32, 64), (torch.float16, 128, 32, 64),
                                                   (torch.float32, 64, 32, 64), (torch.bfloat16, 96, 16, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_infinite_values_are_summed_wherever_they_stand(dtype, nope, rope, v_dim, causal):
    """In V alone: a query that sees an infinite value has it in its sum, one of either sign or a NaN makes NaN, and
    so does a weight of zero (a score far below the others'); no other query and no other column changes."""
    g, n, heads = gen(22), 330, 3
    q, k, v, kr = normal(g, n, heads, nope + rope), normal(g, n, heads, nope), normal(g, n, heads, v_dim), normal(g, n, rope)
    q[..., nope:] = q[..., nope:].abs() + 0.1
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    dev = lambda x: x.to(dtype).to(DEV)  # noqa: E731
    run = lambda kr, v: latent_prefill(dev(q), dev(k), dev(v), dev(kr), cu, cu, n, n, 0.07, causal=causal)  # noqa: E731
    clean = run(kr, v)
    sees = lambda at: torch.arange(n, device=DEV) >= (at if causal else 0)  # noqa: E731
    # key, others: in a block that all, some or (under the queries' own) few see
    for at, also in ((5, 3), (127, 64), (128, 100), (140, 2), (191, 192), (200, 201), (329, 300)):
        bad, want = v.clone(), clean.clone()
        plus, minus, nan, both = 1, 8, 21, v_dim - 1
        bad[at, :, plus], bad[at, :, minus], bad[at, :, nan] = INF, -INF, float("nan")
        bad[at, :, both], bad[also, :, both] = INF, -INF
        want[sees(at), :, plus], want[sees(at), :, minus], want[sees(at), :, nan] = INF, -INF, float("nan")
        want[sees(at), :, both] = INF
        want[sees(also), :, both] = -INF
        want[sees(at) & sees(also), :, both] = float("nan")
        got = run(kr, bad)
        assert torch.equal(got.isnan(), want.isnan()), at
        assert torch.equal(got.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0)), at
        far = kr.clone()
        far[at] = -200.0  # a score below -200 * 0.07 * 0.1 * rope and far below the others
        q_far = 40 * q[..., nope:]
        base = latent_prefill(dev(torch.cat((q[..., :nope], q_far), -1)), dev(k), dev(v), dev(far), cu, cu, n, n, 0.07, causal=causal)
        got = latent_prefill(dev(torch.cat((q[..., :nope], q_far), -1)), dev(k), dev(bad), dev(far), cu, cu, n, n, 0.07, causal=causal)
        seen = sees(at)
        if causal:
            seen = seen & (torch.arange(n, device=DEV) > 0)
        assert got[seen][..., [plus, minus, nan]].isnan().all(), at
        assert torch.equal(got[~sees(at)][..., [plus, minus, nan]], base[~sees(at)][..., [plus, minus, nan]]), at
        others = [d for d in range(v_dim) if d not in (plus, minus, nan, both)]
        assert torch.equal(got[..., others], base[..., others]), at
