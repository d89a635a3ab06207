"""it_sample on the GPU against its definition in 64 bits.

Tokens are equal (borders are hit by chance with a probability below 1e-6 a row:
masses are off by 2^-45 of the largest weight each).  The probability w / kept
is fp32: half a unit, 2^-24 of it; and the weights' rounding to 2^-44 units, at
most 2^-45 each in w and n 2^-45 in a kept mass of at least 1."""
import math

import numpy as np
import pytest

from kvutil import to_dev

pytestmark = pytest.mark.gpu


def reference(z, u, t, k, p, m):
    """(token, probability, tokens kept) of one row."""
    z = np.where(np.isnan(z), -np.inf, np.asarray(z, np.float64))
    order = np.argsort(-z, kind="stable")
    order = order[z[order] > -np.inf]
    if order.size == 0:
        return -1, 0.0, 0
    if not t > 0:
        return int(order[0]), 1.0, 1
    top = z[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(z[order] == top, 1.0, np.exp((z[order] - top) / t)) if top < np.inf else (z[order] == top).astype(float)
    w = w[w >= max(2.0 ** -45, min(m, 1.0) if m > 0 else 0.0)]
    if k > 0:
        w = w[:k]
    c = np.cumsum(w)
    n = w.size
    if p < 1:
        n = max(1, int(np.count_nonzero(np.concatenate([[0.0], c[:-1]]) < p * c[-1])))
    at = int(np.count_nonzero(c[:n] <= (min(max(u, 0.0), 1.0) if u == u else 0.0) * c[n - 1]))
    at = min(at, n - 1)
    return int(order[at]), w[at] / c[n - 1], n


def run(z, u, t=1.0, k=0, p=1.0, m=0.0, dtype=None):
    """z, u and settings (numbers or arrays) through the library; every row against the reference."""
    import torch
    from infer_train_amd.sampling import sample

    logits = z if isinstance(z, torch.Tensor) else torch.from_numpy(np.asarray(z, np.float32)).cuda()
    if dtype is not None:
        logits = logits.to(dtype)
    dev = lambda x, dt: to_dev(np.asarray(x, dt)) if isinstance(x, (np.ndarray, list)) else x  # noqa: E731
    tokens, probs = sample(logits, to_dev(np.asarray(u, np.float32)), dev(t, np.float32), dev(k, np.int32), dev(p, np.float32),
                           dev(m, np.float32))
    tokens, probs, host = tokens.cpu().numpy(), probs.cpu().numpy(), logits.double().cpu().numpy()
    n = len(host)
    full = lambda x, dt: np.broadcast_to(np.asarray(x, dt), (n,))  # noqa: E731
    for r, (zz, uu, tt, kk, pp, mm) in enumerate(zip(host, full(u, np.float32), full(t, np.float32), full(k, np.int32),
                                                     full(p, np.float32), full(m, np.float32))):
        token, prob, _ = reference(zz, float(uu), float(tt), int(kk), float(pp), float(mm))
        assert tokens[r] == token, (r, tokens[r], token, float(probs[r]), prob)
        assert abs(float(probs[r]) - prob) <= 2.0 ** -24 * prob + 2.0 ** -45 * (1 + host.shape[1] * prob), (r, probs[r], prob)
    return tokens, probs


def logits(seed, rows, vocab, scale=2.5):
    rng = np.random.default_rng(seed)
    return (scale * rng.standard_normal((rows, vocab)) + 8 * rng.random((rows, vocab)) ** 30).astype(np.float32)


@pytest.mark.parametrize("dtype", ("float32", "float16", "bfloat16"))
@pytest.mark.parametrize("vocab", (1, 2, 7, 63, 64, 65, 513, 4096, 4097, 32768, 32769, 100003, 262144))
def test_settings(vocab, dtype):
    """Every setting alone and together, rows of odd lengths (each starts at another alignment)."""
    import torch

    t, k, p, m = zip(*((1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.2, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.02),
                       (0.0, 5, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (1.5, 1000, 0.99, 0.0), (0.3, 0, 0.5, 0.0), (1.0, 3000, 1.0, 0.0)))
    u = np.random.default_rng(vocab).random(len(t))
    run(logits(vocab, len(t), vocab), u, np.array(t), np.array(k), np.array(p), np.array(m), getattr(torch, dtype))


@pytest.mark.parametrize("u", (0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, math.nan))
def test_uniform_numbers(u):
    for vocab in (5000, 50000):
        z = logits(1, 4, vocab)
        run(z, [u] * 4)
        run(z, [u] * 4, t=0.9, k=30, p=0.9, m=0.01)


@pytest.mark.parametrize("vocab", (3, 500, 20000, 70000))
def test_equal_tokens(vocab):
    """All tokens equal, or two values: the lower token first, at the borders of every filter, past what is listed."""
    same = np.full((6, vocab), 1.25, np.float32)
    u = np.array([0.0, 0.25, 0.5, 0.75, 0.999, 0.1])
    run(same, u)
    run(same, u, k=vocab // 2 + 1)
    run(same, u, p=0.5)
    run(same, u, k=vocab - 1, p=0.3, m=1.0)
    two = np.where(np.random.default_rng(2).random((6, vocab)) < 0.5, 3.0, 2.5).astype(np.float32)
    for kw in (dict(), dict(k=vocab // 4 + 1), dict(p=0.9), dict(m=0.9), dict(k=vocab // 2 + 2, p=0.7)):
        run(two, u, **kw)
    zero = np.where(np.arange(6 * vocab).reshape(6, vocab) % 2 == 0, 0.0, -0.0).astype(np.float32)
    assert run(zero, [0.0] * 6, k=1)[0].tolist() == [0] * 6  # -0 equals +0


@pytest.mark.parametrize("vocab", (9001, 33001))
def test_masked_rows(vocab):
    """Rows with -inf, the type's lowest value, NaN, +inf, and nothing left."""
    import torch

    rng = np.random.default_rng(3)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        z = torch.from_numpy(logits(4, 12, vocab)).cuda().to(dtype)
        z[0, 1:] = -math.inf
        z[1] = -math.inf
        z[2, rng.random(vocab) < 0.9] = -math.inf
        z[3, rng.random(vocab) < 0.9] = torch.finfo(dtype).min
        z[4] = torch.finfo(dtype).min
        z[5] = math.nan
        z[6, ::2] = math.nan
        z[7, [5, 70, 8000]] = math.inf
        z[8] = math.inf
        z[9, 10:] = -math.inf
        z[10] = torch.finfo(dtype).max
        z[11, :vocab - 2] = -math.inf
        u = rng.random(12)
        for kw in (dict(), dict(t=0.0), dict(k=20), dict(p=0.8), dict(m=0.1), dict(t=0.5, k=1500, p=0.95, m=0.001)):
            tokens, probs = run(z, u, **kw)
            assert tokens[1] == -1 and probs[1] == 0 and tokens[5] == -1 and tokens[0] == 0


@pytest.mark.parametrize("vocab", (3001, 40001))
def test_extreme_settings(vocab):
    z = logits(5, 8, vocab)
    u = np.random.default_rng(6).random(8)
    run(z, u, t=np.array([1e-30, 1e-6, 1e30, math.inf, 1e-45, -1.0, math.nan, 100.0]))
    run(z, u, p=np.array([0.0, -1.0, 1e-9, 1e-45, 0.5, 1.0, 2.0, math.nan]))
    run(z, u, m=np.array([0.0, -1.0, 1e-30, 1.0, 5.0, 1e-9, 0.999, math.nan]))
    run(z, u, k=np.array([0, -3, 1, vocab - 1, vocab, vocab + 1, 2 ** 31 - 1, -2 ** 31]))
    tiny = np.full((2, vocab), 1e-40, np.float32)
    tiny[:, 7] = 2e-40
    run(tiny, [0.3, 0.9])
    run(tiny * 1e38, [0.3, 0.9], t=1e-3, k=300)
    wide = np.linspace(-3e38, 3e38, vocab, dtype=np.float32)[None]
    run(wide, [0.4])
    run(wide, [0.4], t=np.array([1e38]))


@pytest.mark.parametrize("vocab,stride,offset", ((5003, 5003, 0), (5003, 5003, 3), (5003, 5008, 1), (5003, 6000, 0),
                                                 (33333, 33333, 5), (33333, 40000, 2)))
def test_row_strides(vocab, stride, offset):
    import torch

    base = torch.from_numpy(logits(7, 1, offset + 9 * stride)[0]).cuda()
    for dtype in (torch.float32, torch.bfloat16):
        z = base.to(dtype)[offset:].as_strided((9, vocab), (stride, 1), offset)
        run(z, np.linspace(0.05, 0.95, 9), t=0.9, p=0.9)
    one = torch.from_numpy(logits(8, 700, 1)).cuda().t()  # [1, 700], any row stride
    run(one, [0.5])


@pytest.mark.parametrize("kw", (dict(), dict(k=60), dict(p=0.92), dict(t=0.6, k=400, p=0.9, m=0.003)))
def test_a_row_does_not_depend_on_its_batch(kw):
    """One row is divided among many workgroups, 5 and 40 rows likewise, 3000 take one each: the same token and the same
    bits."""
    import torch
    from infer_train_amd.sampling import sample

    z, u = torch.from_numpy(logits(9, 5, 70001)).cuda(), torch.rand(5, generator=torch.Generator().manual_seed(1)).cuda()
    names = dict(t="temperature", k="top_k", p="top_p", m="min_p")
    kw = {names[a]: b for a, b in kw.items()}
    tokens, probs = sample(z, u, **kw)
    for r in range(5):
        a, b = sample(z[r:r + 1], u[r:r + 1], **kw)
        assert a[0] == tokens[r] and b[0] == probs[r]
    for n in (8, 600):
        a, b = sample(z.repeat(n, 1), u.repeat(n), **kw)
        assert torch.equal(a, tokens.repeat(n)) and torch.equal(b, probs.repeat(n))


def test_distribution():
    """20000 draws of one row, evenly spread u: each token as often as its probability, to a token's two ends."""
    import torch
    from infer_train_amd.sampling import sample

    n, z = 20000, logits(10, 1, 40, 1.0)
    u = (torch.arange(n).float() / n).cuda()
    tokens, _ = sample(torch.from_numpy(z).cuda().expand(n, 40).contiguous(), u, top_k=20)
    order = np.argsort(-z[0], kind="stable")[:20]
    w = np.exp(z[0].astype(np.float64)[order])
    got = np.bincount(tokens.cpu().numpy(), minlength=40)
    assert got.sum() == got[order].sum() and (np.abs(got[order] - n * w / w.sum()) <= 2).all()


def test_captured_with_a_shared_and_a_dirty_workspace():
    """Replays of a captured draw with new logits, eager draws between them, over a workspace that starts as rubbish;
    two graphs in turn on one workspace."""
    import torch
    from infer_train_amd.sampling import sample, sample_workspace

    z, u = torch.from_numpy(logits(11, 6, 40011)).cuda(), torch.rand(6).cuda()
    z2, u2 = torch.from_numpy(logits(12, 3, 50000)).cuda().half(), torch.rand(3).cuda()
    ws = sample_workspace(6, 40011, z.device)
    ws.fill_(0xA5)
    want = sample(z, u, top_p=0.9)
    got = sample(z, u, top_p=0.9, ws=ws)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out, out2 = [torch.empty_like(x) for x in want], [torch.empty(3, dtype=torch.int32).cuda(), torch.empty(3).cuda()]
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        sample(z, u, top_p=0.9, tokens=out[0], probs=out[1], ws=ws)
    with torch.cuda.graph(graphs[1]):
        sample(z2, u2, temperature=0.8, top_k=30, tokens=out2[0], probs=out2[1], ws=ws)
    for i in range(4):
        z.copy_(torch.from_numpy(logits(20 + i, 6, 40011)))
        z2.copy_(torch.from_numpy(logits(30 + i, 3, 50000)))
        u.copy_(torch.rand(6))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        a, b = sample(z, u, top_p=0.9), sample(z2, u2, temperature=0.8, top_k=30)
        assert torch.equal(out[0], a[0]) and torch.equal(out[1], a[1]), i
        assert torch.equal(out2[0], b[0]) and torch.equal(out2[1], b[1]), i


def test_two_streams_at_once():
    import torch
    from infer_train_amd.sampling import sample

    z, u = torch.from_numpy(logits(13, 40, 50021)).cuda(), torch.rand(40).cuda()
    want = sample(z, u, top_p=0.8)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(sample(z, u, top_p=0.8))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_sample_refusals():
    import torch
    from infer_train_amd import InvalidInput, NotImplementedOp
    from infer_train_amd.sampling import sample

    z, u = torch.zeros(3, 50, device="cuda"), torch.zeros(3, device="cuda")
    for bad in (dict(temperature=-1.0), dict(temperature=math.inf), dict(top_p=math.nan), dict(min_p=2.0),
                ):
        with pytest.raises(InvalidInput):
            sample(z, u, **bad)
    with pytest.raises(InvalidInput):
        sample(torch.zeros(3, 40000, device="cuda"), u, ws=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(NotImplementedOp):
        sample(torch.zeros(1, 262145, device="cuda"), u[:1])
    for bad in (dict(temperature=u.double()), dict(top_k=u), dict(min_p=u[:2]), dict(tokens=u), dict(probs=u.int())):
        with pytest.raises(TypeError):
            sample(z, u, **bad)
    with pytest.raises(TypeError):
        sample(z, u[:2])
    with pytest.raises(TypeError):
        sample(z.double(), u)
    for bad in (z[0], z.t(), z.cpu()):
        with pytest.raises(ValueError):
            sample(bad, u)
    tokens, probs = sample(z[:0], u[:0])
    assert tokens.numel() == probs.numel() == 0


def test_batcher_draws_for_its_requests():
    import torch
    from infer_train_amd import ContinuousBatcher, SamplingParams

    settings = [SamplingParams(), SamplingParams(0.0), SamplingParams(0.7, 40, 0.9, 0.01)]
    b = ContinuousBatcher(8)
    for i, s in enumerate(settings):
        b.add_request(i, [1], 4, s)
    b.schedule()
    z, u = logits(14, 3, 7001), np.array([0.3, 0.6, 0.9], np.float32)
    got = b.sample(torch.from_numpy(z).cuda(), to_dev(u))
    for i, s in enumerate(settings):
        want = reference(z[i], float(u[i]), float(np.float32(s.temperature)), s.top_k, float(np.float32(s.top_p)), float(np.float32(s.min_p)))[0]
        assert got[i] == want and b.requests[i].generated_tokens == [want]
    z[1] = -math.inf
    with pytest.raises(ValueError):
        b.sample(torch.from_numpy(z).cuda(), to_dev(u))
    assert [len(r.generated_tokens) for r in b.requests.values()] == [1, 1, 1]
