"""Beam scores of rows with extreme logits: the group's value of a continuation is
its beam's score plus log_softmax of its row in 64 bits, however large the logits
are.  Chosen beams and tokens must be equal; a score is one fp64 value rounded to
fp32 (2^-24 of it), whose own error is below 2^-40 of its terms (at most 64 where
the value is small)."""
import numpy as np
import pytest
import torch

from infer_train_amd.beam import beam_select

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain_select(logits, scores, n):
    """log_softmax is shifted by the row's maximum; of a row at +inf the tokens there share the row."""
    z = torch.where(logits.isnan(), -INF, logits.double())
    top = z.amax(-1, keepdim=True)
    flat = torch.where(top == INF, torch.where(z == INF, 0.0, -INF), z)
    lp = torch.log_softmax(flat, -1).nan_to_num(nan=-INF, neginf=-INF)  # a row without a token: none
    g, b = scores.shape
    v = (scores.double().nan_to_num(nan=-INF, neginf=-INF)[..., None] + lp.view(g, b, -1)).numpy()
    z = z.view(g, b, -1).numpy()
    out = np.full((g, n), -np.inf), np.full((g, n), -1), np.full((g, n), -1)
    for i in range(g):
        beam, token = np.nonzero(v[i] > -np.inf)
        order = np.lexsort((token, -z[i, beam, token], beam, -v[i, beam, token]))[:n]
        for j, o in enumerate(order):
            out[0][i, j], out[1][i, j], out[2][i, j] = v[i, beam[o], token[o]], beam[o], token[o]
    return out


def check(logits, scores, n):
    got = [x.cpu().numpy() for x in beam_select(logits.to(DEV), scores.to(DEV), n)]
    want = plain_select(logits, scores, n)
    assert np.array_equal(got[1], want[1]), "parents"
    assert np.array_equal(got[2], want[2]), "tokens"
    fin, one = np.isfinite(want[0]), np.nan_to_num(want[0], neginf=0.0, posinf=0.0)
    assert np.array_equal(np.isfinite(got[0]), fin) and np.array_equal(got[0][~fin], want[0][~fin])
    diff = np.abs(np.where(fin, got[0], 0.0) - one)
    assert (diff[fin] <= (2.0 ** -24 * np.abs(one) + 2.0 ** -40 * np.maximum(np.abs(one), 64.0))[fin]).all()
    return got


def rows(seed, n, vocab, dtype, spread=3.0):
    g = torch.Generator()
    g.manual_seed(seed)
    return (spread * torch.randn(n, vocab, generator=g)).to(dtype), -20 * torch.rand(n, generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_all_at_the_lowest_value_does_not_outrank_a_live_beam(dtype):
    """A grammar without a token left for a beam: its row is flat, its score log(1 / vocab) lower."""
    z, _ = rows(1, 2, 1000, dtype)
    z[0] = torch.finfo(dtype).min
    got = check(z, torch.tensor([[-19.0, -4.0]]), 4)
    assert (got[1] == 1).all()
    got = check(z[:1], torch.tensor([[-19.0]]), 4)
    assert np.allclose(got[0], -19 - np.log(1000), atol=1e-5) and got[2].tolist() == [[0, 1, 2, 3]]


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_token_at_the_largest_value_keeps_its_beams_score(dtype):
    z, _ = rows(2, 2, 5000, dtype)
    z[0, 77] = torch.finfo(dtype).max
    got = check(z, torch.tensor([[-19.0, -30.0]]), 4)
    assert got[0][0, 0] == -19 and got[2][0, 0] == 77


@pytest.mark.parametrize("size", [1e3, 1e10, 1e30])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_rows_far_from_zero(size, sign):
    """Rows shifted as a whole: a row's log-probabilities are those of its differences."""
    z, s = rows(3, 6, 9001, torch.float32, spread=1.0)
    z = (z.double() * size * 2.0 ** -20 + sign * size).float()
    check(z, s.view(2, 3), 12)
    check(z, s.view(6, 1), 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows(dtype):
    """Rows with few tokens, one, none; the type's lowest and largest values; infinities and NaN."""
    z, s = rows(4, 12, 9001, dtype)
    g = torch.Generator()
    g.manual_seed(5)
    out = torch.rand(z.shape, generator=g) < 0.999
    z[0] = z[0].masked_fill(out[0], -INF)
    z[1] = -INF
    z[2] = -INF
    z[2, 8500] = -70.0
    z[3] = z[3].masked_fill(out[3], torch.finfo(dtype).min)
    z[4] = torch.finfo(dtype).min
    z[5] = z[5].masked_fill(~out[5], float("nan"))
    z[6] = float("nan")
    z[7, [77, 8999, 4000]] = INF
    z[8, 3] = torch.finfo(dtype).max
    z[9, 100:] = torch.finfo(dtype).min
    z[9, :100] = -INF
    check(z, s.view(3, 4), 16)
    check(z, s.view(1, 12), 24)
    check(z, s.view(12, 1), 64)


def test_flat_and_peaked_rows():
    z, s = rows(6, 4, 100003, torch.float32, spread=1e-3)
    check(z, s.view(1, 4), 8)
    z, s = rows(7, 4, 100003, torch.float32, spread=30.0)
    check(z, s.view(2, 2), 4)
    check(z.double().mul(1e36).float(), s.view(2, 2), 4)


def test_several_slices_of_which_one_is_extreme():
    """The row's maximum is in another slice than most of its tokens, or than all that are not masked."""
    z, s = rows(8, 4, 40000, torch.float32)
    z[0, :39000] = torch.finfo(torch.float32).min
    z[1, 35000] = 3e38
    z[2] = torch.finfo(torch.float32).min
    z[2, 20000:20003] = torch.tensor([-3e38, -2e38, -2e38])
    check(z, s.view(1, 4), 32)
    check(z, s.view(4, 1), 32)
