"""Latent attention on the device against plain forms in 64 bits: rows stored,
gathered, moved and copied, absorbed attention over pages, expanded attention
over contiguous keys, and a step of them together.

Tolerances: u = finfo(type).eps / 2 is a rounding.  Attention's weights are
rounded to the cache's type for the matrix cores (u each, so 2 u of the
weighted sum of |values|, numerator and denominator), a score's fp32 sum takes
at most 160 roundings of 2^-24 of the sum of its terms' magnitudes, and the
result is rounded once (half a step: u, or half a subnormal one)."""
import numpy as np
import pytest
import torch

from infer_train_amd import BF16, F16, F32, BlockPool, InvalidInput, KvManager, NotImplementedOp
from infer_train_amd.kv import PagedKvCache, Rotary
from infer_train_amd.latent import LatentKvCache, latent_prefill

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
IDS = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
INF = float("inf")


def u(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(dtype, x):
    """What rounding x to dtype changes at most: half a step, u of x; below the smallest normal number
    (tiny) steps are tiny * eps all the way down."""
    f = torch.finfo(dtype)
    return (u(dtype) * x.abs()).clamp(min=f.tiny * f.eps / 2)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape):
    return torch.randn(shape, generator=g)


def angles(rotary, pos):
    return pos.double()[:, None] * torch.from_numpy(rotary.inv_freq)


def turn(x, ang, layout, magnitude=1.0):
    """x [n, heads, d] float64 with all of its pairs rotated."""
    c, s = (ang.cos() * magnitude)[:, None], (ang.sin() * magnitude)[:, None]
    y = torch.empty_like(x)
    d = x.shape[-1]
    a, b = (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else (x[..., :d // 2], x[..., d // 2:])
    first, second = a * c - b * s, a * s + b * c
    if layout == "interleaved":
        y[..., 0::2], y[..., 1::2] = first, second
    else:
        y[..., :d // 2], y[..., d // 2:] = first, second
    return y


def within(got, want, tol, what=""):
    got, want = got.detach().cpu().double(), want.cpu().double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    ok = ~torch.isnan(want)
    err = torch.where(ok, (got - want).abs(), torch.zeros_like(want))
    bad = err > torch.where(ok, tol.cpu().double().expand_as(want), torch.zeros_like(want))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, at {bad.nonzero()[0].tolist()}, most {err.max():.3g}"


# ---- append ------------------------------------------------------------------
@pytest.mark.parametrize("src,cache,latent,rope,heads,layout,odd", [
    (torch.bfloat16, torch.bfloat16, 512, 64, 28, "interleaved", False),
    (torch.float16, torch.float16, 256, 32, 5, "half", False),
    (torch.float32, torch.bfloat16, 512, 64, 16, "half", False),
    (torch.float32, torch.float32, 1024, 64, 1, "interleaved", False),
    (torch.bfloat16, torch.float32, 128, 16, 40, "interleaved", False),
    (torch.bfloat16, torch.bfloat16, 72, 24, 33, "half", False),  # pairs that do not fall into vectors
    (torch.float16, torch.bfloat16, 512, 64, 3, "interleaved", True),  # strides that no vector is aligned to
])
@pytest.mark.parametrize("n", [1, 2, 67])
def test_append(src, cache, latent, rope, heads, layout, odd, n):
    g, bs = gen(n + latent), 16
    nb = -(-n // bs) + 2
    c = LatentKvCache(nb, bs, latent, rope, IDS[cache])
    before = normal(g, nb, bs, latent + rope).to(cache)
    c.view().copy_(before)
    rotary = Rotary(rope, layout=layout, magnitude=1.25)
    extra = 1 if odd else 8
    kv = (3 * normal(g, n, latent + rope + extra)).to(src).to(DEV)[:, :latent + rope]
    proj = normal(g, n, heads, 40 + rope + extra).to(src).to(DEV)
    q = proj[..., 40:40 + rope]
    weight = (1 + 0.3 * normal(g, latent)).to(torch.float32 if heads % 2 else src).to(DEV)
    pos = torch.randint(0, 1 << 20, (n,), generator=g, dtype=torch.int32)
    slots = torch.randperm(nb * bs, generator=g)[:n]
    if n > 2:
        slots[n // 2] = -1
    rows = torch.full((n, latent + rope), -7.0, dtype=cache, device=DEV)
    out = c.append(kv, slots.to(DEV), rotary, pos.to(DEV), weight=weight, eps=1e-5, q_rope=q, rows_out=rows)
    c.check()
    x, w = kv.cpu().double(), weight.cpu().double()
    lat = x[:, :latent] * torch.rsqrt(x[:, :latent].square().mean(1, keepdim=True) + 1e-5) * w
    turned = turn(x[:, None, latent:], angles(rotary, pos), layout, 1.25)[:, 0]
    want = torch.cat((lat, turned), 1)
    # the norm: a sum of squares in fp32 (at most 26 roundings), a root, a quotient, two products
    size = torch.cat((lat.abs(), 1.25 * 1.5 * x[:, latent:].abs().amax(1, keepdim=True).expand(-1, rope)), 1)
    tol = rounding(cache, want) + 32 * 2.0 ** -24 * size + 1e-12
    within(rows, want, tol, "rows")
    pool = before.double().view(-1, latent + rope).clone()
    live = slots >= 0
    pool[slots[live]] = rows.cpu().double()[live]
    assert torch.equal(c.view().cpu().double().view(-1, latent + rope), pool)  # and nothing else changed
    wq = turn(q.cpu().double(), angles(rotary, pos), layout, 1.25)
    within(out, wq, rounding(src, wq) + 8 * 2.0 ** -24 * 2 * q.cpu().double().abs().amax(), "q")
    same = c.append(kv, slots.to(DEV), rotary, pos.to(DEV), weight=weight, eps=1e-5, q_rope=q, q_out=q)
    assert same is q and torch.equal(same.cpu(), out.cpu())  # in place, inside the projection
    assert torch.equal(proj[..., :40].cpu(), proj.cpu()[..., :40])


@pytest.mark.parametrize("src,cache,heads,layout", [(torch.bfloat16, torch.bfloat16, 3, "interleaved"), (torch.float16, torch.float16, 8, "half"),
                                                    (torch.float32, torch.bfloat16, 1, "half")])
def test_append_many_tokens_of_few_heads(src, cache, heads, layout):
    test_append(src, cache, 256, 64, heads, layout, False, 4500)


def test_append_without_norm_rotation_or_queries():
    g = gen(3)
    c = LatentKvCache(4, 8, 128, 32, BF16)
    kv = normal(g, 9, 160).to(torch.bfloat16).to(DEV)
    kv[4, 7], kv[4, 150] = INF, float("nan")
    slots = torch.arange(9, device=DEV) + 3
    assert c.append(kv, slots) is None
    got = c.view().view(-1, 160)[3:12].cpu()
    assert torch.equal(got.view(torch.int16), kv.cpu().view(torch.int16))


def test_append_bad_positions_and_slots_are_latched():
    g = gen(4)
    c = LatentKvCache(2, 8, 64, 32, F16)
    kv = normal(g, 3, 96).half().to(DEV)
    rotary = Rotary(32)
    q = normal(g, 3, 2, 32).half().to(DEV)
    out = torch.full_like(q, 9.0)
    c.append(kv, torch.tensor([0, 1, 2], device=DEV), rotary, torch.tensor([5, -1, 7], dtype=torch.int32, device=DEV), q_rope=q, q_out=out)
    with pytest.raises(InvalidInput, match="position"):
        c.check()
    assert (out[1] == 9).all() and not (out[0] == 9).any() and (c.view()[0, 1] == 0).all() and not (c.view()[0, 2] == 0).all()
    c.append(kv, torch.tensor([16, -1, 3], device=DEV))
    with pytest.raises(InvalidInput, match="slot"):
        c.check()
    c.check()


def test_append_many_layers_and_moves():
    """A cache of three layers: appended by layer, its blocks copied and
    cleared, its rows moved (the rope part turned), tables kept, in all."""
    g, bs, latent, rope = gen(5), 8, 64, 32
    for dtype in (torch.bfloat16, torch.float32):
        c = LatentKvCache(6, bs, latent, rope, IDS[dtype], n_layers=3)
        data = normal(g, 3, 6 * bs, latent + rope).to(dtype)
        slots = torch.arange(6 * bs, device=DEV)
        for i in range(3):
            c.layer(i).append(data[i].to(DEV), slots)
        with pytest.raises(InvalidInput):
            c.append(data[0].to(DEV), slots)
        c.copy_blocks(torch.tensor([1], dtype=torch.int32, device=DEV), torch.tensor([5], dtype=torch.int32, device=DEV))
        c.evict(torch.tensor([2], dtype=torch.int32, device=DEV))
        data = data.view(3, 6, bs, -1)
        data[:, 5], data[:, 2] = data[:, 1], 0
        data = data.view(3, 6 * bs, -1)
        for i in range(3):
            assert torch.equal(c.layer(i).view().cpu().view(6 * bs, -1), data[i])
        for layout in ("interleaved", "half"):
            rotary = Rotary(rope, layout=layout)
            src, dst = torch.tensor([1, 2, 9, 40, -1]), torch.tensor([17, 18, 19, 40, 20])
            delta = torch.tensor([-5, 0, 100003, 7, 1], dtype=torch.int32)
            c.move(src.to(DEV), dst.to(DEV), rotary, delta.to(DEV))
            c.check()
            for i in range(3):
                old = data[i].double()
                turned = turn(old[src[:4], None, latent:], angles(rotary, delta[:4]), layout)[:, 0]
                want = data[i].double().clone()
                want[dst[:4]] = torch.cat((old[src[:4], :latent], turned), 1)
                got = c.layer(i).view().cpu().double().view(6 * bs, -1)
                tol = torch.zeros_like(want)
                tol[dst[:4], latent:] = rounding(dtype, turned) + 8 * 2.0 ** -24 * 2 * old[src[:4], latent:].abs().amax()
                tol[18] = 0  # not turned: the same bytes
                within(got, want, tol, f"move {layout} {dtype}")
                data[i] = got.to(dtype)
        c.move(torch.tensor([3], device=DEV), torch.tensor([23], device=DEV))
        for i in range(3):
            data[i, 23] = data[i, 3]
            assert torch.equal(c.layer(i).view().cpu().view(6 * bs, -1), data[i])


def test_gather_rows():
    g, bs = gen(6), 16
    c = LatentKvCache(12, bs, 96, 32, F16)
    c.view().copy_(normal(g, 12, bs, 128).half())
    tables = torch.randperm(12, generator=g).int()[:9].view(3, 3)
    ctx, start = torch.tensor([33, 0, 48]), torch.tensor([0, 0, 17])
    cu = torch.tensor([0, 33, 33])
    out = torch.zeros(70, 128, dtype=torch.float16, device=DEV)
    c.gather(tables.to(DEV), ctx.int().to(DEV), start.int().to(DEV), cu.to(DEV), 48, out)
    flat, want = c.view().cpu().view(-1, 128), []
    for b in range(3):
        p = torch.arange(int(start[b]), int(ctx[b]))
        want.append(flat[tables[b][p // bs].long() * bs + p % bs])
    assert torch.equal(out.cpu()[:64], torch.cat(want)) and (out[64:] == 0).all()


# ---- decode --------------------------------------------------------------------
def exact_decode(q, flat, slots, seen, latent, scale):
    """q [heads, row], the rows of `slots`, `seen` [n] of them visible: float64 result and the
    magnitudes that bound its error: sum of p |v|, and a score's sum of |terms|."""
    rows = flat[slots[seen]].double()
    if rows.shape[0] == 0:
        z = torch.zeros(q.shape[0], latent, dtype=torch.float64)
        return z, z, 0.0
    s = q.double() @ rows.t() * scale
    p = torch.softmax(s, 1)
    terms = (q.double().abs() @ rows.abs().t() * abs(scale)).nan_to_num(0, 0, 0).amax().item()
    return p @ rows[:, :latent], p @ rows[:, :latent].abs(), terms


def decode_case(dtype, latent, rope, heads, lens, q_len=1, bs=16, start=None, seed=0, poison=False, split_q=False, out_dtype=None,
                spread=1.0, bound=0):
    g = gen(seed + heads + sum(lens))
    held = [-(-n // bs) for n in lens]
    blocks = sum(held) + 3
    order = torch.randperm(blocks, generator=g).int()
    tables = torch.full((len(lens), max(held) + 2), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(held):
        tables[i, :m] = order[at:at + m]
        at += m
    c = LatentKvCache(blocks, bs, latent, rope, IDS[dtype])
    flat = normal(g, blocks * bs, latent + rope)
    used = torch.zeros(blocks * bs, dtype=torch.bool)
    slots = []
    for i, n in enumerate(lens):
        p = torch.arange(n)
        slots.append(tables[i][p // bs].long() * bs + p % bs)
        lo = 0 if start is None else start[i]
        used[slots[i][lo:]] = True
    if poison:  # what no query may see
        flat[~used] = torch.tensor([float("nan"), INF, -INF])[torch.randint(0, 3, (int((~used).sum()), 1), generator=g)]
    if start is not None:  # entries of blocks wholly below the window are not read
        for i, lo in enumerate(start):
            tables[i, :lo // bs] = -1
    flat = flat.to(dtype)
    c.view().copy_(flat.view(blocks, bs, -1))
    n = len(lens) * q_len
    q = (spread * normal(g, n, heads, latent + rope)).to(dtype)
    scale = 1.0 / (128 + rope) ** 0.5
    qd = q.to(DEV)
    ql, qr = qd[..., :latent], qd[..., latent:]
    if split_q:
        ql, qr = ql.contiguous(), qr.contiguous()
    longest = max([m - (0 if start is None else start[i] & ~31) for i, m in enumerate(lens)] + [bound])
    out = c.decode(ql, qr, tables.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), longest, scale,
                   start_pos=None if start is None else torch.tensor(start, dtype=torch.int32, device=DEV), q_len=q_len,
                   out_dtype=out_dtype)
    c.check()
    odt = out_dtype or dtype
    for i, m in enumerate(lens):
        for j in range(q_len):
            p = torch.arange(m)
            seen = (p < m - q_len + 1 + j) & (p >= (0 if start is None else start[i]))
            want, mag, terms = exact_decode(q[i * q_len + j], flat, slots[i], seen, latent, scale)
            weights = 2 * (u(dtype) if dtype != torch.float32 else 0.0) + 2 * 160 * 2.0 ** -24 * terms + 2.0 ** -20
            within(out[i * q_len + j], want, rounding(odt, want) + weights * mag + 1e-30, f"seq {i} row {j}")
    return c, out


@pytest.mark.parametrize("dtype,latent,rope", [(torch.bfloat16, 512, 64), (torch.float16, 512, 64), (torch.float16, 256, 32),
                                               (torch.bfloat16, 256, 64), (torch.float32, 512, 64), (torch.float32, 64, 16),
                                               (torch.bfloat16, 128, 64), (torch.float16, 96, 24)])
@pytest.mark.parametrize("heads,q_len", [(1, 1), (12, 4), (28, 1), (40, 1), (16, 3)])
def test_decode(dtype, latent, rope, heads, q_len):
    decode_case(dtype, latent, rope, heads, [1 + q_len, 0, 31, 32, 33, 130, 257], q_len=q_len, poison=True)


@pytest.mark.parametrize("heads", [64, 80, 128])
@pytest.mark.parametrize("dtype,latent,rope", [(torch.bfloat16, 512, 64), (torch.float16, 256, 32)])
def test_decode_many_heads(dtype, latent, rope, heads):
    decode_case(dtype, latent, rope, heads, [700, 0, 45, 1025], poison=True)


@pytest.mark.parametrize("bound", [1 << 15, 1 << 17])
@pytest.mark.parametrize("heads,q_len", [(28, 1), (64, 1), (80, 1), (128, 1), (40, 3), (24, 6)])
@pytest.mark.parametrize("dtype,latent,rope", [(torch.bfloat16, 512, 64), (torch.float16, 256, 32), (torch.bfloat16, 128, 64),
                                               (torch.float16, 256, 64)])
def test_decode_under_a_bound_far_above(dtype, latent, rope, heads, q_len, bound):
    """The bound, not the lengths, chooses how many queries share a workgroup."""
    decode_case(dtype, latent, rope, heads, [700, 0, 45, 1025, 31], q_len=q_len, poison=True, bound=bound, start=[3, 0, 40, 900, 0])


@pytest.mark.parametrize("bs", [1, 4, 8, 16, 64, 256])
def test_decode_page_sizes(bs):
    decode_case(torch.bfloat16, 512, 64, 16, [5, 300, 64, 129], bs=bs, poison=True)
    decode_case(torch.float16, 256, 32, 40, [5, 300, 64, 129], bs=bs, q_len=2, poison=True)


@pytest.mark.parametrize("n", [1, 2, 300])
def test_decode_batches(n):
    """One sequence to more sequences than workgroups, lengths 0 to 200."""
    rng = np.random.default_rng(n)
    decode_case(torch.bfloat16, 256, 32, 4, [int(x) for x in rng.integers(0, 200, n - 1)] + [190], poison=True)


def test_decode_one_long_sequence_beside_short_ones():
    decode_case(torch.bfloat16, 512, 64, 8, [3, 9000, 1, 64], poison=True)
    decode_case(torch.float16, 512, 64, 128, [1, 5000], poison=True, split_q=True)


@pytest.mark.parametrize("heads,q_len", [(12, 1), (40, 3), (128, 1)])
def test_decode_windows(heads, q_len):
    """Starts inside and at the edges of pages and key tiles, and at the context's end."""
    lens = [100, 333, 64, 500, 40, 70]
    decode_case(torch.bfloat16, 512, 64, heads, lens, q_len=q_len, start=[1, 200, 32, 499, 0, 70], poison=True)


def test_decode_out_types_and_large_scores():
    decode_case(torch.bfloat16, 512, 64, 20, [77, 400], out_dtype=torch.float32, spread=6.0)
    decode_case(torch.float16, 512, 64, 20, [77, 400], out_dtype=torch.float32, spread=6.0)


def test_decode_more_new_tokens_than_context():
    """Rows of new tokens that see nothing are zero."""
    c, out = decode_case(torch.bfloat16, 256, 32, 3, [2, 5], q_len=4)
    assert (out[:2] == 0).all() and (out[2:4] != 0).any()


def test_decode_values_that_later_tokens_bring():
    """A drafted token's infinities and NaN do not reach the tokens before it, and
    reach those that see it as a sum would."""
    wide = [(h, b, 512, 64) for h in (12, 32, 48) for b in (0, 1 << 17, 1 << 20)]
    for heads, bound, latent, rope in [(2, 0, 256, 32), (12, 0, 256, 32), (32, 0, 256, 32), (48, 0, 256, 32), (48, 1 << 20, 256, 32)] + wide:
        g, bs, n, t = gen(heads), 16, 70, 4
        c = LatentKvCache(8, bs, latent, rope, BF16)
        flat = normal(g, 8 * bs, latent + rope).to(torch.bfloat16)
        flat[n - 2, 3] = INF  # token 2 of the four
        flat[n - 1, 200] = float("nan")
        c.view().copy_(flat.view(8, bs, -1))
        q = normal(g, t, heads, latent + rope).to(torch.bfloat16)
        q[..., 3] = -q[..., 3].abs() - 0.5  # an infinite latent element scores -inf: its weight is 0, and 0 * inf NaN
        tables = torch.arange(8, dtype=torch.int32, device=DEV)[None]
        out = c.decode(q.to(DEV)[..., :latent], q.to(DEV)[..., latent:], tables, torch.tensor([n], dtype=torch.int32, device=DEV),
                       max(n, bound), 0.1, q_len=t)
        for j in range(2):
            want, mag, terms = exact_decode(q[j], flat, torch.arange(n), torch.arange(n) < n - t + 1 + j, latent, 0.1)
            within(out[j], want, u(torch.bfloat16) * (want.abs() + 2 * mag) + 2 * 160 * 2.0 ** -24 * terms * mag + 1e-5 * mag, f"token {j}")
        assert torch.isnan(out[2, :, 3]).all() and torch.isnan(out[3]).all()


def test_decode_bad_tables_and_lengths_are_latched():
    g = gen(8)
    c = LatentKvCache(4, 16, 256, 32, BF16)
    c.view().copy_(normal(g, 4, 16, 288).to(torch.bfloat16))
    q = normal(g, 2, 4, 288).to(torch.bfloat16).to(DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    run = lambda tables, lens, most, start=None: c.decode(q[..., :256], q[..., 256:], tables, lens, most, 0.1, start_pos=start)  # noqa: E731
    good = run(torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV), i32(20, 30), 32)
    c.check()
    out = run(torch.tensor([[0, 9], [2, 3]], dtype=torch.int32, device=DEV), i32(20, 30), 32)
    with pytest.raises(InvalidInput, match="block"):
        c.check()
    assert torch.equal(out[1], good[1])
    for lens, most, start, word in ((i32(20, 65), 32, None, "ctx"), (i32(20, 40), 64, None, "table"), (i32(20, 30), 32, i32(0, -3), "start")):
        out = run(torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV), lens, most, start)
        with pytest.raises(InvalidInput, match=word):
            c.check()
        assert torch.equal(out[0], good[0]) and (out[1] == 0).all()


def test_decode_replayed_from_a_graph():
    """Captured once, replayed with other lengths, tables and rows between eager
    calls; two captured graphs with a workspace each."""
    g, bs = gen(9), 16
    c = LatentKvCache(64, bs, 512, 64, BF16)
    c.view().copy_(normal(g, 64, bs, 576).to(torch.bfloat16))
    q = normal(g, 3, 16, 576).to(torch.bfloat16).to(DEV)
    tables = torch.randperm(64, generator=g).int()[:60].view(3, 20).to(DEV)
    lens = torch.tensor([100, 320, 7], dtype=torch.int32, device=DEV)
    eager = lambda: c.decode(q[..., :512], q[..., 512:], tables, lens, 320, 0.07)  # noqa: E731
    eager()
    graphs = []
    for _ in range(2):
        ws, out = c.decode_workspace(3, 16, 320), torch.empty(3, 16, 512, dtype=torch.bfloat16, device=DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.decode(q[..., :512], q[..., 512:], tables, lens, 320, 0.07, out=out, ws=ws)
        graphs.append((graph, out, ws))
    for turn_ in range(4):
        lens.copy_(torch.tensor([[100, 320, 7], [1, 0, 319], [64, 65, 320], [320, 320, 320]][turn_], dtype=torch.int32))
        q.mul_(-1.01)
        want = eager()
        torch.cuda.synchronize()
        for graph, out, _ in graphs:
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for _, out, _ in graphs:
            assert torch.equal(out, want)


def test_decode_on_two_streams():
    """Overlapping calls, each with its own workspace, equal the calls one after another."""
    g = gen(10)
    c = LatentKvCache(400, 16, 512, 64, BF16)
    c.view().copy_(normal(g, 400, 16, 576).to(torch.bfloat16))
    q = [normal(g, 2, 32, 576).to(torch.bfloat16).to(DEV) for _ in range(2)]
    tables = torch.randperm(400, generator=g).int().view(2, 200).to(DEV)
    lens = torch.tensor([3000, 3200], dtype=torch.int32, device=DEV)
    call = lambda x, **kw: c.decode(x[..., :512], x[..., 512:], tables, lens, 3200, 0.07, **kw)  # noqa: E731
    want = [call(x) for x in q]
    ws = [c.decode_workspace(2, 32, 3200) for _ in q]
    outs = [[torch.empty(2, 32, 512, dtype=torch.bfloat16, device=DEV) for _ in range(4)] for _ in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for r in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                call(q[i], ws=ws[i], out=outs[i][r])
    torch.cuda.synchronize()
    for i in range(2):
        for r in range(4):
            assert torch.equal(outs[i][r], want[i])


# ---- prefill -------------------------------------------------------------------
def prefill_case(dtype, heads, nope, rope, v_dim, q_lens, k_lens, causal=True, seed=0, fused=True, out_dtype=None, behind=3, spread=1.0):
    g = gen(seed + heads + sum(q_lens) + sum(k_lens))
    nq, nk = sum(q_lens) + behind, sum(k_lens) + behind
    q = (spread * normal(g, nq, heads, nope + rope)).to(dtype)
    kv = normal(g, nk, heads, nope + v_dim).to(dtype)
    rows = normal(g, nk, 40 + rope).to(dtype)
    kv[sum(k_lens):], rows[sum(k_lens):] = float("nan"), float("nan")
    kd, rd = kv.to(DEV), rows.to(DEV)
    k, v, kr = kd[..., :nope], kd[..., nope:], rd[:, 40:]
    if not fused:
        k, v, kr = k.contiguous(), v.contiguous(), kr.contiguous()
    cu = lambda x: torch.tensor([0] + list(np.cumsum(x)), dtype=torch.int32, device=DEV)  # noqa: E731
    out = torch.full((nq, heads, v_dim), 7.0, dtype=out_dtype or dtype, device=DEV)
    scale = 1.0 / (nope + rope) ** 0.5
    latent_prefill(q.to(DEV), k, v, kr, cu(q_lens), cu(k_lens), max(q_lens), max(k_lens), scale, causal=causal, out=out)
    torch.cuda.synchronize()
    aq = ak = 0
    for m, n in zip(q_lens, k_lens):
        if m:
            qq = q[aq:aq + m].double().transpose(0, 1)
            kk = torch.cat((kv[ak:ak + n, :, :nope].double(), rows[ak:ak + n, None, 40:].double().expand(-1, heads, -1)), -1).permute(1, 2, 0)
            vv = kv[ak:ak + n, :, nope:].double().transpose(0, 1)
            s = qq @ kk * scale
            hidden = torch.arange(n)[None] > n - m + torch.arange(m)[:, None]
            if causal:
                s = s.masked_fill(hidden, -INF)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            want, mag = (p @ vv).transpose(0, 1), (p @ vv.abs()).transpose(0, 1)
            terms = (qq.abs() @ kk.abs() * scale).amax().item() if n else 0.0
            weights = 2 * (u(dtype) if dtype != torch.float32 else 0.0) + 2 * 160 * 2.0 ** -24 * terms + 2.0 ** -20
            within(out[aq:aq + m], want, rounding(out.dtype, want) + weights * mag + 1e-30, f"rows {aq}..{aq + m} over {n}")
        aq, ak = aq + m, ak + n
    assert (out[aq:] == 7).all()  # rows behind the last sequence
    return out


@pytest.mark.parametrize("dtype,nope,rope,v_dim", [(torch.bfloat16, 128, 64, 128), (torch.float16, 128, 64, 128), (torch.float16, 64, 32, 64),
                                                   (torch.bfloat16, 128, 32, 64), (torch.float32, 128, 64, 128), (torch.bfloat16, 96, 16, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill(dtype, nope, rope, v_dim, causal):
    prefill_case(dtype, 3, nope, rope, v_dim, [1, 0, 33, 64, 130, 5], [1, 7, 33, 200, 131, 70], causal=causal)
    prefill_case(dtype, 1, nope, rope, v_dim, [65], [65], causal=causal, fused=False, out_dtype=torch.float32)


@pytest.mark.parametrize("dtype,nope,rope,v_dim", [(torch.bfloat16, 128, 64, 128), (torch.float16, 64, 32, 64), (torch.float16, 128, 32, 64)])
def test_prefill_long(dtype, nope, rope, v_dim):
    prefill_case(dtype, 2, nope, rope, v_dim, [300, 511, 1], [1300, 511, 2049])
    prefill_case(dtype, 9, nope, rope, v_dim, [257], [257], spread=5.0)


def test_prefill_more_queries_than_keys():
    """Queries that see nothing give 0; no keys at all too."""
    out = prefill_case(torch.bfloat16, 2, 128, 64, 128, [9, 4], [5, 0])
    assert (out[:4] == 0).all() and (out[9:13] == 0).all()


def test_prefill_masked_values_do_not_spread():
    """Keys that only later queries see may hold infinities and NaN."""
    g, n, heads = gen(12), 150, 2
    q, kv, kr = (normal(g, n, heads, 192).to(torch.bfloat16), normal(g, n, heads, 256).to(torch.bfloat16), normal(g, n, 64).to(torch.bfloat16))
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    run = lambda x: latent_prefill(q.to(DEV), x.to(DEV)[..., :128], x.to(DEV)[..., 128:], kr.to(DEV), cu, cu, n, n, 0.07)  # noqa: E731
    clean = run(kv)
    for at in (149, 140, 100, 64, 63, 37):
        bad = kv.clone()
        bad[at, :, 128 + 5], bad[at, :, 128 + 77], bad[at, :, 3] = INF, float("nan"), float("nan")
        out = run(bad)
        assert torch.equal(out[:at], clean[:at]), at
        assert torch.isnan(out[at:]).all(), at


def test_prefill_lengths_outside_the_tensors_are_not_computed():
    g = gen(13)
    q, k, kr, v = (normal(g, 40, 2, 96).half().to(DEV), normal(g, 50, 2, 64).half().to(DEV), normal(g, 50, 32).half().to(DEV),
                   normal(g, 50, 2, 64).half().to(DEV))
    cu = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    run = lambda cq, ck, mq, mk: latent_prefill(q, k, v, kr, cq, ck, mq, mk, 0.1, out=torch.full((40, 2, 64), 7.0, dtype=torch.float16, device=DEV))  # noqa: E731
    good = run(cu(0, 20, 40), cu(0, 20, 50), 20, 30)
    for cq, ck, mq, mk in ((cu(0, 20, 41), cu(0, 20, 50), 30, 30), (cu(0, 20, 40), cu(0, 20, 51), 20, 40), (cu(0, 20, 40), cu(0, 20, 50), 20, 29),
                           (cu(0, 20, 5), cu(0, 20, 50), 20, 30)):
        out = run(cq, ck, mq, mk)
        assert torch.equal(out[:20], good[:20]) and (out[20:] == 7).all()


def test_prefill_replayed_from_a_graph():
    g = gen(14)
    q, k, kr, v = (normal(g, 100, 4, 192).to(torch.bfloat16).to(DEV), normal(g, 300, 4, 128).to(torch.bfloat16).to(DEV),
                   normal(g, 300, 64).to(torch.bfloat16).to(DEV), normal(g, 300, 4, 128).to(torch.bfloat16).to(DEV))
    cq, ck = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 40, 100], [0, 40, 300]))
    run = lambda out=None: latent_prefill(q, k, v, kr, cq, ck, 100, 300, 0.07, out=out)  # noqa: E731
    run()
    out, graph = torch.empty(100, 4, 128, dtype=torch.bfloat16, device=DEV), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out)
    for lens in ((0, 40, 100), (0, 0, 100), (0, 100, 100), (0, 1, 2)):
        cq.copy_(torch.tensor(lens, dtype=torch.int32))
        q.mul_(-1.01)
        out.fill_(3)
        want = run(torch.full_like(out, 3))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---- together --------------------------------------------------------------------
def test_prompt_then_steps_equal_one_long_prefill():
    """A prompt stored and attended expanded, then tokens one and two at a time in
    absorbed form: each step's result, projected up, is the expanded attention of
    its position over everything before."""
    g, heads, latent, nope, rope, v_dim, bs = gen(15), 4, 256, 64, 32, 64, 16
    dt = torch.bfloat16
    pool = BlockPool(40, BF16)
    mgr = KvManager(pool, bs, 2, 20)
    c = LatentKvCache(40, bs, latent, rope, BF16)
    rotary = Rotary(rope, layout="interleaved")
    w_k, w_v = (normal(g, heads, d, latent).to(dt).to(DEV) / latent ** 0.5 for d in (nope, v_dim))
    scale = 1.0 / (nope + rope) ** 0.5
    prompts, steps = [37, 90], [1, 2, 1]
    total = [p + sum(steps) for p in prompts]
    kv = [normal(g, n, latent + rope).to(dt).to(DEV) for n in total]
    q = [normal(g, n, heads, nope + rope).to(dt).to(DEV) for n in total]
    weight = torch.ones(latent, dtype=dt, device=DEV)
    tables = torch.full((2, 20), -1, dtype=torch.int32, device=DEV)

    def store(plan, kvs, qs):
        to = lambda a: torch.from_numpy(a).to(DEV)  # noqa: E731
        slots, pos = to(plan.slots), to(plan.token_pos)
        rows = torch.empty(slots.numel(), latent + rope, dtype=dt, device=DEV)
        turned = c.append(kvs, slots, rotary, pos, weight=weight, q_rope=qs[..., nope:], rows_out=rows)
        c.sync_tables(tables, to(plan.token_seq), pos, slots)
        return torch.cat((qs[..., :nope], turned), -1), rows, to(plan.ctx_lens)

    def up(rows):  # the projection: keys and values of each head
        x = rows[:, :latent].float()
        k = torch.stack([x @ w.float().t() for w in w_k], 1).to(dt)
        v = torch.stack([x @ w.float().t() for w in w_v], 1).to(dt)
        return k, v, rows[:, latent:]

    plan = mgr.append([0, 1], prompts)
    qs, rows, _ = store(plan, torch.cat([kv[i][:p] for i, p in enumerate(prompts)]), torch.cat([q[i][:p] for i, p in enumerate(prompts)]))
    cu = torch.tensor([0, prompts[0], sum(prompts)], dtype=torch.int32, device=DEV)
    k, v, kr = up(rows)
    got = [[x] for x in latent_prefill(qs, k, v, kr, cu, cu, 90, 90, scale).split(prompts)]
    done = list(prompts)
    for n in steps:
        plan = mgr.append([0, 1], n)
        qs, _, ctx = store(plan, torch.cat([kv[i][d:d + n] for i, d in enumerate(done)]), torch.cat([q[i][d:d + n] for i, d in enumerate(done)]))
        absorbed = torch.stack([qs[:, h, :nope].float() @ w_k[h].float() for h in range(heads)], 1).to(dt)
        lat = c.decode(absorbed, qs[..., nope:], tables, ctx, int(ctx.max()), scale, q_len=n, out_dtype=torch.float32)
        out = torch.stack([lat[:, h] @ w_v[h].float().t() for h in range(heads)], 1)
        for i in range(2):
            got[i].append(out[i * n:(i + 1) * n])
            done[i] += n
    c.check()
    ctx = torch.tensor(total, dtype=torch.int32, device=DEV)
    rows = torch.empty(sum(total), latent + rope, dtype=dt, device=DEV)
    c.gather(tables, ctx, None, torch.tensor([0, total[0]], device=DEV), max(total), rows)
    k, v, kr = up(rows)
    qr = [torch.cat((q[i][..., :nope], rotary.apply(q[i][..., nope:].contiguous(), torch.arange(total[i], dtype=torch.int32, device=DEV))), -1)
          for i in range(2)]
    cu = torch.tensor([0, total[0], sum(total)], dtype=torch.int32, device=DEV)
    want = latent_prefill(torch.cat(qr), k, v, kr, cu, cu, max(total), max(total), scale, out_dtype=torch.float32).split(total)
    for i in range(2):
        a, b = torch.cat([x.float() for x in got[i]]), want[i]
        # Keys and queries rounded at other places: a score of d = 64 terms moves by about 2 u sqrt(sum of squares) <
        # 3 x 2^-8, values by u, weights by 2 u: a norm's bound, not an element's.
        assert ((a - b).norm(dim=-1) <= 16 * 2.0 ** -8 * v.float().abs().amax()).all(), i


# ---- refusals --------------------------------------------------------------------
def test_refusals_on_the_device():
    c = LatentKvCache(4, 16, 256, 32, BF16)
    kv, slots = torch.zeros(3, 288, dtype=torch.bfloat16, device=DEV), torch.arange(3, device=DEV)
    rotary, pos = Rotary(32), torch.arange(3, dtype=torch.int32, device=DEV)
    q = torch.zeros(3, 4, 32, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(TypeError):
        c.append(kv, slots.int())
    with pytest.raises(ValueError):
        c.append(kv[:, :-8], slots)
    with pytest.raises(ValueError):
        c.append(kv.t().contiguous().t(), slots)
    with pytest.raises(TypeError):
        c.append(kv, slots, rotary)
    with pytest.raises(TypeError):
        c.append(kv, slots, rotary, pos, q_rope=q.float())
    with pytest.raises(ValueError):
        c.append(kv, slots, rotary, pos, q_rope=q[..., :16])
    with pytest.raises(InvalidInput):
        c.append(kv, slots, Rotary(64), pos)
    with pytest.raises(InvalidInput):  # heads of zero stride
        c.append(kv, slots, rotary, pos, q_rope=q, q_out=q[:, :1].expand(-1, 4, -1))
    with pytest.raises(InvalidInput):  # shifted by a head
        big = torch.zeros(3, 5, 32, dtype=torch.bfloat16, device=DEV)
        c.append(kv, slots, rotary, pos, q_rope=big[:, :4], q_out=big[:, 1:])
    with pytest.raises(InvalidInput):
        c.append(kv, slots, weight=torch.ones(256, device=DEV), eps=-1.0)
    with pytest.raises(InvalidInput):  # latent caches hold no K and V rows
        PagedKvCache.append(c, kv, kv, slots)
    with pytest.raises(InvalidInput):
        PagedKvCache.decode(c, kv[:, None], torch.zeros(3, 1, dtype=torch.int32, device=DEV), pos, None, 16)
    ordinary = PagedKvCache(4, 16, 1, 288, BF16)
    with pytest.raises(InvalidInput):
        ordinary.latent_dim, ordinary.rope_dim = 256, 32
        LatentKvCache.append(ordinary, kv, slots)
    tables, lens = torch.zeros(3, 1, dtype=torch.int32, device=DEV), torch.ones(3, dtype=torch.int32, device=DEV)
    ql, qr = torch.zeros(3, 4, 256, dtype=torch.bfloat16, device=DEV), q
    with pytest.raises(NotImplementedOp):
        c.decode(ql.half(), qr.half(), tables, lens, 16, 0.1)
    with pytest.raises(NotImplementedOp):
        c.decode(ql, qr, tables, lens, 16, 0.1, out_dtype=torch.float16)
    with pytest.raises(InvalidInput):
        c.decode(ql, qr, tables, lens, 16, float("nan"))
    with pytest.raises(ValueError):
        c.decode(ql, qr[:, :3], tables, lens, 16, 0.1)
    with pytest.raises(ValueError):
        c.decode(ql, qr, tables, lens, 16, 0.1, q_len=2)
    with pytest.raises(InvalidInput):
        c.decode(ql.expand(3, 4, 256).repeat(65, 1, 1)[:65 * 3], qr.repeat(65, 1, 1), tables, lens, 16, 0.1, q_len=65)
    with pytest.raises(InvalidInput):  # 2^31 runs of 32 tokens
        many = LatentKvCache(2, 1024, 8, 8, BF16)
        z = torch.zeros(65535, 1, 8, dtype=torch.bfloat16, device=DEV)
        many.decode(z, z, torch.zeros(65535, 1024, dtype=torch.int32, device=DEV), torch.zeros(65535, dtype=torch.int32, device=DEV), 1 << 20, 0.1)
    with pytest.raises(InvalidInput):
        c.move(slots, slots + 8, Rotary(64), pos)
    k = torch.zeros(5, 4, 64, dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        latent_prefill(ql, k, k, q[:, 0], cu, cu, 3, 3, 0.1)
    with pytest.raises(InvalidInput):
        latent_prefill(torch.zeros(3, 4, 76, dtype=torch.bfloat16, device=DEV), k, k, torch.zeros(5, 12, dtype=torch.bfloat16, device=DEV), cu, cu, 3, 5, 0.1)
