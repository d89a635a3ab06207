"""it_kv_move on the GPU: rows between slots of every format, keys turned.

Float rows against the formula (tolerances as in test_gpu_rotary); quantised
rows against the same row dequantised on the host, turned in fp64 and compared
as values: the quantiser rounds to within half a step of its grid (Q8_0: scale /
2; 4- and 5-bit: the grid's step d / 2, or a whole step at the end that the
formats clamp), and its fp16 scale, taken again from the turned row, is off by
2^-11 of itself times the code."""
import numpy as np
import pytest

import oracle as orc
from kvutil import from_dev, to_dev
from test_gpu_rotary import CACHE, check, exact_turn, torch_dtype, values

pytestmark = pytest.mark.gpu
QUANT = ("q8_0", "q4_0", "q4_1", "q5_0", "q5_1")


def filled(cname, nb, bs, h, d, layers, seed):
    """A cache whose rows hold random values in its format."""
    import torch
    from infer_train_amd.kv import PagedKvCache

    cache = PagedKvCache(nb, bs, h, d, CACHE[cname], n_layers=layers)
    slots = to_dev(np.arange(nb * bs, dtype=np.int64))
    for i in range(layers):
        x = torch.from_numpy(values(seed + i, 2, nb * bs, h, d)).cuda()
        x = x if cname in QUANT else x.to(torch_dtype(cname))
        (cache.layer(i) if layers > 1 else cache).append(x[0].contiguous(), x[1].contiguous(), slots)
    cache.check()
    return cache


def rows_of(cache, which, layer):
    """(values float64 [slots, heads, d], raw bytes per row [slots, heads, row_bytes], step [slots, heads, d]) of a layer."""
    c = cache.layer(layer) if cache.n_layers > 1 else cache
    nb, h, bs, d = c.num_blocks, c.n_kv_heads, c.block_size, c.head_dim
    flat = lambda a: a.swapaxes(1, 2).reshape((nb * bs, h) + a.shape[3:])  # noqa: E731
    if c.dtype in (0, 1, 30):
        t = c.view(which)
        x = t.double().cpu().numpy()
        import torch

        raw = t.contiguous().view(torch.uint8).view(nb, h, bs, -1).cpu().numpy()
        return flat(x), flat(raw), None
    half = lambda t: t.cpu().numpy().view(np.float16).astype(np.float64)  # noqa: E731
    if c.dtype == CACHE["q8_0"]:
        qs, sc = c.q8_planes(which)
        q, s = qs.cpu().numpy().astype(np.float64), half(sc)
        raw = np.concatenate([qs.cpu().numpy().view(np.uint8), sc.cpu().numpy().view(np.uint8).reshape(nb, h, bs, -1)], -1)
        step = np.repeat(s, 32, -1)
        return flat(q * step), flat(raw), flat(np.abs(step))
    planes = c.q5_planes(which) if c.dtype in (CACHE["q5_0"], CACHE["q5_1"]) else c.q4_planes(which)
    qs, meta = planes[0].cpu().numpy().reshape(nb, h, bs, d // 32, 16), half(planes[-1])
    q = np.concatenate([qs & 15, qs >> 4], -1).astype(np.float64)
    parts = [planes[0].cpu().numpy()]
    if len(planes) == 3:
        qh = planes[1].cpu().numpy().view(np.uint32)
        q += 16.0 * ((qh[..., None] >> np.arange(32, dtype=np.uint32)) & 1)
        parts.append(qh.view(np.uint8).reshape(nb, h, bs, -1))
    parts.append(planes[-1].cpu().numpy().view(np.uint8).reshape(nb, h, bs, -1))
    if c.dtype in (CACHE["q4_1"], CACHE["q5_1"]):
        x, s = q * meta[..., :1] + meta[..., 1:], meta[..., 0]
    else:
        x, s = (q - (8 if c.dtype == CACHE["q4_0"] else 16)) * meta[..., None], meta
    shape = (nb, h, bs, d)
    return flat(x.reshape(shape)), flat(np.concatenate(parts, -1)), flat(np.abs(np.repeat(s, 32, -1)).reshape(shape))


CASES = [  # cache, bs, heads, D, n_dims, layout, layers
    ("bf16", 16, 4, 128, 128, "half", 1), ("bf16", 16, 2, 128, 64, "half", 5), ("f16", 8, 3, 96, 32, "half", 2),
    ("f32", 32, 1, 256, 256, "interleaved", 3), ("bf16", 16, 2, 24, 24, "half", 2), ("f16", 4, 5, 40, 6, "interleaved", 1),
    ("f32", 16, 2, 64, 20, "half", 1), ("bf16", 1, 2, 64, 64, "interleaved", 1), ("f32", 16, 7, 80, 80, "half", 1),
    ("q8_0", 16, 2, 128, 128, "half", 2), ("q8_0", 32, 3, 256, 64, "interleaved", 1), ("q4_0", 16, 2, 64, 64, "half", 2),
    ("q4_1", 16, 2, 96, 96, "interleaved", 1), ("q5_0", 8, 2, 32, 10, "half", 3), ("q5_1", 16, 2, 128, 128, "half", 1),
]


@pytest.mark.parametrize("n", (1, 50, 333))
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_move(case, n):
    import torch
    from infer_train_amd.kv import Rotary

    cname, bs, h, d, rot, layout, layers = case
    nb = 2 * (-(-n // bs)) + 3
    cache = filled(cname, nb, bs, h, d, layers, 30)
    rng = np.random.default_rng(n)
    perm = rng.permutation(nb * bs)
    src, dst = perm[:n].astype(np.int64), perm[n:2 * n].astype(np.int64)
    if n > 4:
        src[1], dst[2] = -1, -7  # skipped
    delta = rng.integers(-5000, 50, n).astype(np.int32)
    delta[::3] = 0
    before = [[rows_of(cache, w, l) for l in range(layers)] for w in "kv"]
    r = Rotary(rot, layout, magnitude=1.3)  # a move does not apply it again
    live = (src >= 0) & (dst >= 0)

    cache.move(to_dev(src), to_dev(dst), r, to_dev(delta))
    cache.check()
    for w, which in enumerate("kv"):
        for l in range(layers):
            x, raw, _ = before[w][l]
            gx, graw, gstep = rows_of(cache, which, l)
            want = raw.copy()
            still = live if w else live & (delta == 0)
            want[dst[still]] = raw[src[still]]
            turned = np.flatnonzero(live & ~still)
            rest = np.ones(nb * bs, bool)
            rest[dst[turned]] = False
            assert np.array_equal(graw[rest], want[rest]), (which, l)  # byte for byte: copied rows and those not named
            if not turned.size:
                continue
            y, tol = exact_turn(x[src[turned]], delta[turned], r.inv_freq, 1.0, layout)
            got = gx[dst[turned]]
            if cname in QUANT:
                step = gstep[dst[turned]]
                low = cname in ("q4_0", "q5_0")  # the grid ends one step short on the side opposite to its largest element
                bound = step * (1.0 if low else 0.5) * (1 + 2.0 ** -6) + 2.0 ** -10 * np.abs(y) + step * 2.0 ** -5 + tol
                assert (np.abs(got - y) <= bound).all(), (which, l, np.abs(got - y).max())
            else:
                check(torch.from_numpy(got), y, tol, cname, f"{which} layer {l}")

    plain = filled(cname, nb, bs, h, d, layers, 30)
    plain.move(to_dev(src), to_dev(dst))
    plain.check()
    for w, which in enumerate("kv"):
        for l in range(layers):
            want = before[w][l][1].copy()
            want[dst[live]] = want[src[live]]
            assert np.array_equal(rows_of(plain, which, l)[1], want), (which, l, "copied")


@pytest.mark.parametrize("cname", ("bf16", "f32", "q8_0", "q5_1"))
@pytest.mark.parametrize("d,rot,layout", ((128, 128, "half"), (64, 22, "interleaved"), (64, 20, "half")))
def test_shift_in_place_equals_a_move(cname, d, rot, layout):
    """src == dst: rows are turned where they are (some of them past a lane's or a wave's end), as if moved elsewhere."""
    from infer_train_amd.kv import Rotary

    bs, nb, h, n = 16, 12, 3, 90
    a, b = filled(cname, nb, bs, h, d, 2, 50), filled(cname, nb, bs, h, d, 2, 50)
    r = Rotary(rot, layout)
    at = np.arange(n, dtype=np.int64)
    delta = np.full(n, -13, np.int32)
    delta[5] = 0
    a.move(to_dev(at), to_dev(at), r, to_dev(delta))
    b.move(to_dev(at), to_dev(at + 100), r, to_dev(delta))
    for which in "kv":
        for l in range(2):
            got, want = rows_of(a, which, l)[1], rows_of(b, which, l)[1]
            assert np.array_equal(got[:n], want[100:100 + n]) and np.array_equal(got[100:], rows_of(filled(cname, nb, bs, h, d, 2, 50), which, l)[1][100:])


def test_moves_refused_and_latched():
    import torch
    from infer_train_amd import InvalidInput
    from infer_train_amd.kv import Rotary

    cache = filled("bf16", 4, 16, 2, 64, 2, 60)
    keep = cache.k_pool.clone()
    r = Rotary(64)
    one = lambda x, dt=np.int64: to_dev(np.array([x], dt))  # noqa: E731
    for src, dst in ((64, 0), (0, 64), (1 << 40, 0)):
        cache.move(one(src), one(dst), r, one(3, np.int32))
        with pytest.raises(InvalidInput):
            cache.check()
        cache.move(one(src), one(dst))
        with pytest.raises(InvalidInput):
            cache.check()
    assert torch.equal(cache.k_pool, keep)
    with pytest.raises(InvalidInput):
        cache.move(one(0), one(1), Rotary(128), one(3, np.int32))
    for args in ((one(0), one(1), r, None), (one(0), one(1), None, one(3, np.int32)), (one(0, np.int32), one(1)),
                 (one(0), to_dev(np.zeros(2, np.int64))), (one(0), one(1), r, one(3))):
        with pytest.raises(TypeError):
            cache.move(*args)
    empty = to_dev(np.zeros(0, np.int64))
    cache.move(empty, empty)
    assert torch.equal(cache.k_pool, keep)


def test_layer_view_and_graph():
    """A layer's view moves that layer alone; a captured move replayed with new slots equals eager ones."""
    import torch
    from infer_train_amd.kv import Rotary

    cache, ref = filled("f16", 8, 16, 2, 64, 3, 70), filled("f16", 8, 16, 2, 64, 3, 70)
    r = Rotary(64)
    src, dst, delta = (to_dev(np.arange(5, dtype=np.int64)), to_dev(np.arange(5, dtype=np.int64) + 64),
                       to_dev(np.full(5, -9, np.int32)))
    cache.layer(1).move(src, dst, r, delta)
    for l, moved in ((0, False), (1, True), (2, False)):
        a, b = rows_of(cache, "v", l)[1], rows_of(ref, "v", l)[1]
        assert np.array_equal(a[64:69], b[0:5] if moved else b[64:69])
    ref.layer(1).move(src, dst, r, delta)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.move(src, dst, r, delta)
    for i in range(3):
        src.add_(5)
        dst.add_(5)
        delta.sub_(1)
        graph.replay()
        torch.cuda.synchronize()
        ref.move(src, dst, r, delta)
        assert torch.equal(cache.k_pool, ref.k_pool) and torch.equal(cache.v_pool, ref.v_pool), i
