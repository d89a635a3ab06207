"""Rotary positions on the GPU (it_rotary_apply, it_kv_append_rotary) against
the formula in 64 bits (angles in 80).

Tolerance of an output element of a pair (a, b): the angle is off by 2^-51 of
itself (frequency / 2 pi, its product with the position: a rounding of 2^-53
each and the constant's) and by 2^-25 where it is rounded to fp32; cosine and
sine by 2^-24 each, their product with the magnitude 2^-24, the two products and
their sum 2^-24 each: together below 2^-21 + |angle| 2^-51 of magnitude (|a| +
|b|).  Then half a step of the output's type, eps / 2 of the value, and half
fp16's smallest step."""
import math

import numpy as np
import pytest

import oracle as orc
from kvutil import from_dev, to_dev

pytestmark = pytest.mark.gpu
DTYPES = {"f32": 0, "f16": 1, "bf16": 30}


def torch_dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def exact_turn(x, pos, freqs, m, layout, transpose=False):
    """x [n, heads, d] float64 -> (rotated, tolerance before the output's rounding)."""
    rot = 2 * len(freqs)
    two_pi = np.longdouble("6.283185307179586476925286766559")
    angle = np.asarray(pos, np.longdouble)[:, None] * np.asarray(freqs, np.longdouble)
    a64 = (angle - two_pi * np.rint(angle / two_pi)).astype(np.float64)[:, None, :]
    size = np.abs(angle).astype(np.float64)[:, None, :]
    c, s = m * np.cos(a64), m * np.sin(a64) * (-1 if transpose else 1)
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    a, b = x[..., first], x[..., second]
    y, tol = x.copy(), np.zeros_like(x)
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    tol[..., first] = tol[..., second] = m * (np.abs(a) + np.abs(b)) * (2.0 ** -21 + size * 2.0 ** -51)
    return y, tol


def eps_half(name):
    import torch

    return torch.finfo(torch_dtype(name)).eps / 2


def check(got, want, tol, name, what=""):
    got = got.double().cpu().numpy()
    bound = tol + eps_half(name) * (np.abs(want) + tol) + (2.0 ** -25 if name == "f16" else 0.0)
    bad = np.abs(got - want) > bound
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], want[bad][:3], bound[bad][:3])


def values(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


CASES = [  # tokens, heads, head_dim, n_dims, layout, dtype
    (1, 1, 2, 2, "half", "f32"), (1, 28, 128, 128, "half", "bf16"), (3, 5, 128, 64, "half", "bf16"),
    (7, 3, 96, 32, "half", "f16"), (5, 9, 80, 80, "interleaved", "bf16"), (2, 4, 80, 20, "half", "f16"),
    (65, 2, 64, 64, "interleaved", "f32"), (4, 3, 256, 128, "interleaved", "f16"), (9, 2, 24, 24, "half", "bf16"),
    (6, 3, 40, 6, "interleaved", "f32"), (2, 2, 1024, 1024, "half", "f32"), (2, 2, 2048, 1024, "interleaved", "f32"),
    (300, 16, 128, 128, "half", "f32"), (1200, 33, 64, 32, "half", "bf16"), (2, 1, 30, 14, "half", "f16"),
    (3, 200, 112, 112, "interleaved", "bf16"),
]


@pytest.mark.parametrize("transpose", (False, True))
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_apply(case, transpose):
    import torch
    from infer_train_amd.kv import Rotary

    n, h, d, rot, layout, name = case
    r = Rotary(rot, layout, magnitude=1.25)
    x = torch.from_numpy(values(1, n, h, d)).cuda().to(torch_dtype(name))
    pos = np.random.default_rng(2).integers(-300, 200000, n).astype(np.int32)
    got = r.apply(x, to_dev(pos), transpose=transpose)
    want, tol = exact_turn(x.double().cpu().numpy(), pos, r.inv_freq, 1.25, layout, transpose)
    check(got, want, tol, name)
    assert torch.equal(got[..., rot:], x[..., rot:])  # passes through
    same = x.clone()
    assert r.apply(same, to_dev(pos), out=same, transpose=transpose) is same and torch.equal(same, got)  # in place


@pytest.mark.parametrize("name", ("f32", "bf16"))
@pytest.mark.parametrize("offset,stride", ((0, 700), (3, 700), (8, 704), (0, 512), (1, 513)))
def test_apply_strides_and_alignment(name, offset, stride):
    """Token strides and addresses that are no multiple of 16 bytes, inputs and outputs; elements between tokens are
    left as they were."""
    import torch
    from infer_train_amd.kv import Rotary

    n, h, d = 5, 4, 128
    r = Rotary(d)
    base = torch.from_numpy(values(3, offset + n * stride)).cuda().to(torch_dtype(name))
    view = lambda t: t[offset:].as_strided((n, h, d), (stride, d, 1), t.storage_offset() + offset)  # noqa: E731
    x, pos = view(base), to_dev(np.arange(n, dtype=np.int32) * 1000)
    buf = torch.full_like(base, 7.0)
    out = view(buf)
    got = r.apply(x, pos, out=out)
    assert got is out and torch.equal(out, r.apply(x.contiguous(), pos))
    mask = torch.ones_like(buf, dtype=torch.bool)
    view(mask).fill_(False)
    assert bool((buf[mask] == 7.0).all())


def test_positions_of_any_size():
    """Positions from -2^31 to 2^31 - 1, a custom frequency of 2^20 radians, and scaled frequencies."""
    import torch
    from infer_train_amd.kv import Rotary

    pos = np.array([-2 ** 31, -1, 0, 1, 2, 1000003, 2 ** 24 + 1, 2 ** 31 - 1], np.int32)
    x = torch.from_numpy(values(4, len(pos), 2, 64)).cuda()
    for r in (Rotary(64), Rotary(64, scaling="linear", factor=4.0), Rotary(64, scaling="base", factor=40.0),
              Rotary(64, scaling="parts", factor=16.0, original_ctx=4096, magnitude=1.277)):
        want, tol = exact_turn(x.double().cpu().numpy(), pos, r.inv_freq, r.magnitude, "half")
        check(r.apply(x, to_dev(pos)), want, tol, "f32")
    fast = Rotary(64, inv_freq=np.linspace(0.0, 2.0 ** 20, 32))
    small = np.arange(8, dtype=np.int32) * 1000
    want, tol = exact_turn(x.double().cpu().numpy(), small, fast.inv_freq, 1.0, "half")
    check(fast.apply(x, to_dev(small)), want, tol, "f32")


def test_position_zero_and_special_values():
    import torch
    from infer_train_amd.kv import Rotary

    for layout in ("half", "interleaved"):
        x = torch.from_numpy(values(5, 2, 2, 64)).cuda()
        assert torch.equal(Rotary(64, layout).apply(x, to_dev(np.zeros(2, np.int32))), x)
        part = torch.from_numpy(values(6, 1, 1, 64)).cuda()
        part[..., 40:] = float("inf")
        part[..., 41] = float("nan")
        out = Rotary(32, layout).apply(part, to_dev(np.array([77], np.int32)))
        assert torch.equal(out[..., 40:].nan_to_num(5.0), part[..., 40:].nan_to_num(5.0)) and bool(out[..., :40].isfinite().all())


@pytest.mark.parametrize("layout", ("half", "interleaved"))
def test_transpose_is_the_gradient(layout):
    """<g, R x> differentiated: against R^T g of the formula (as in test_apply) and against differences.  R is linear, so
    a central difference is exact but for fp32's rounding of the two forward outputs: each is within 2^-21 + |angle|
    2^-51 of its pair's |a| + |b| <= 12, and half a unit; the sum over 2 elements of |g| <= 6, over a step of 2."""
    import torch
    from infer_train_amd.kv import Rotary

    n, h, d, rot = 3, 2, 32, 24
    r = Rotary(rot, layout, magnitude=1.5)
    x, g = torch.from_numpy(values(7, n, h, d)).cuda(), torch.from_numpy(values(8, n, h, d)).cuda()
    assert float(x.abs().max()) < 5 and float(g.abs().max()) < 5
    pos = to_dev(np.array([0, 17, 4095], np.int32))
    grad = r.apply(g, pos, transpose=True)
    for t, i, e in ((0, 0, 0), (1, 1, 5), (2, 0, 11), (2, 1, 23), (1, 0, 31)):
        up, down = x.clone(), x.clone()
        up[t, i, e] += 1.0
        down[t, i, e] -= 1.0
        step = float(up[t, i, e].double() - down[t, i, e].double())
        diff = float(((r.apply(up, pos).double() - r.apply(down, pos).double()) * g.double()).sum()) / step
        # Forward outputs 1.5 (|a| + |b|) <= 18 with 2^-20.5 each, two of them, times |g| < 5 over two elements, over 2.
        assert abs(diff - float(grad[t, i, e])) < 2 * 2 * 5 * 18 * 2.0 ** -20 / 2 + 2.0 ** -20 * 15
    plain = Rotary(rot, layout)
    back = plain.apply(plain.apply(x, pos), pos, transpose=True)  # magnitude 1: the inverse
    assert float((back - x).abs().max()) < 2 * 10 * 2.0 ** -20


# ---- with the append ---------------------------------------------------------
APPEND = [  # cache, source, hq, hkv, D, n_dims, layout
    ("bf16", "bf16", 28, 4, 128, 128, "half"), ("f16", "f16", 6, 3, 96, 32, "half"), ("f32", "f32", 8, 2, 64, 64, "interleaved"),
    ("bf16", "f32", 4, 4, 128, 96, "interleaved"), ("f32", "bf16", 2, 1, 256, 256, "half"), ("f16", "bf16", 2, 2, 24, 10, "half"),
    ("f32", "f16", 0, 3, 20, 20, "interleaved"),
    ("q8_0", "bf16", 8, 2, 128, 128, "half"), ("q8_0", "f32", 8, 2, 256, 128, "half"), ("q4_0", "f16", 2, 2, 64, 64, "interleaved"),
    ("q4_1", "f32", 2, 2, 96, 96, "half"), ("q5_0", "bf16", 4, 2, 128, 32, "half"), ("q5_1", "f32", 2, 1, 128, 128, "interleaved"),
    ("q4_0", "bf16", 3, 3, 32, 6, "half"),
]
CACHE = {"f32": 0, "f16": 1, "bf16": 30, "q8_0": 8, "q4_0": 2, "q4_1": 3, "q5_0": 6, "q5_1": 7}


@pytest.mark.parametrize("n", (1, 37, 700))
@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c)))
def test_append_rotary(case, n):
    """q_out and float pages against the formula.  Quantised pages: byte for byte what the plain append makes of the same
    fp32 rotated rows, which it_rotary_apply gives in float32 from the widened input (bit-equal arithmetic: the same
    products and sums of the same angles)."""
    import torch
    from infer_train_amd.kv import PagedKvCache, Rotary

    cname, sname, hq, hkv, d, rot, layout = case
    bs, nb = 16, n // 16 + 8
    r = Rotary(rot, layout, magnitude=1.125)
    rng = np.random.default_rng(n)
    x = torch.from_numpy(values(9, n, hq + 2 * hkv, d)).cuda().to(torch_dtype(sname))
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    pos = rng.integers(0, 100000, n).astype(np.int32)
    slots = rng.permutation(nb * bs)[:n].astype(np.int64)
    slots[::5] = -1  # padding
    cache = PagedKvCache(nb, bs, hkv, d, CACHE[cname])
    for p in (cache.k_pool, cache.v_pool):
        p.fill_(0x3C)
    out = cache.append_rotary(r, q if hq else None, k, v, to_dev(slots), to_dev(pos))
    cache.check()
    if hq:
        want, tol = exact_turn(q.double().cpu().numpy(), pos, r.inv_freq, 1.125, layout)
        check(out, want, tol, sname, "q")
        other = cache.append_rotary(r, q, k, v, to_dev(slots), to_dev(pos), q_out_dtype=torch.float32)
        check(other, want, tol, "f32", "q in float32")
    ref = PagedKvCache(nb, bs, hkv, d, CACHE[cname])
    for p in (ref.k_pool, ref.v_pool):
        p.fill_(0x3C)
    kr = r.apply(k.float().contiguous(), to_dev(pos))
    if cname in ("f32", "f16", "bf16"):
        ref.append(kr.to(torch_dtype(cname)), v.to(torch_dtype(cname)).contiguous(), to_dev(slots))
        live = np.flatnonzero(slots >= 0)
        at = torch.from_numpy(slots[live]).cuda()
        got = cache.view("k")[at // bs, :, at % bs]
        want, tol = exact_turn(k.double().cpu().numpy()[live], pos[live], r.inv_freq, 1.125, layout)
        check(got, want, tol, cname, "k")
        untouched = torch.ones((nb, bs), dtype=torch.bool, device="cuda")
        untouched[at // bs, at % bs] = False
        kc, kf = cache.view("k").transpose(1, 2), ref.view("k").transpose(1, 2)
        assert torch.equal(kc[untouched], kf[untouched])
    else:
        ref.append(kr, v.float().contiguous(), to_dev(slots))
        assert torch.equal(cache.k_pool, ref.k_pool)
    assert torch.equal(cache.v_pool, ref.v_pool)


def test_append_rotary_layer_view_and_latches():
    import torch
    from infer_train_amd import InvalidInput
    from infer_train_amd.kv import PagedKvCache, Rotary

    cache = PagedKvCache(4, 16, 2, 64, CACHE["bf16"], n_layers=2)
    r = Rotary(64)
    x = torch.from_numpy(values(10, 3, 6, 64)).cuda().bfloat16()
    q, k, v = x[:, :2], x[:, 2:4], x[:, 4:]
    pos, slots = to_dev(np.array([1, 2, 3], np.int32)), to_dev(np.array([0, 1, 2], np.int64))
    with pytest.raises(InvalidInput):
        cache.append_rotary(r, q, k, v, slots, pos)  # takes a layer's view
    cache.layer(1).append_rotary(r, q, k, v, slots, pos)
    lb = cache.k_pool.numel() // 2
    assert not cache.k_pool[:lb].any() and cache.k_pool[lb:].any()
    cache.check()
    view = cache.layer(0)
    out = torch.full((3, 2, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    view.append_rotary(r, q, k, v, slots, to_dev(np.array([1, -2, 3], np.int32)), q_out=out)
    assert bool((out[1] == 9.0).all()) and not bool((out[0] == 9.0).any())
    rows = view.view("k")[0].transpose(0, 1)
    assert not rows[1].any() and rows[0].any() and rows[2].any()
    with pytest.raises(InvalidInput):
        cache.check()
    cache.check()
    view.append_rotary(r, q, k, v, to_dev(np.array([5, 64, 6], np.int64)), pos)
    with pytest.raises(InvalidInput):
        cache.check()


def test_refusals_on_device():
    import torch
    from infer_train_amd import InvalidInput, NotImplementedOp
    from infer_train_amd.kv import PagedKvCache, Rotary

    r, x = Rotary(64), torch.zeros(4, 2, 64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(InvalidInput):
        r.apply(torch.zeros(4, 2, 32, device="cuda"), pos)  # n_dims > head_dim
    flat = torch.zeros(5 * 128, device="cuda")
    a, b = flat[:512].view(4, 2, 64), flat[128:].view(4, 2, 64)
    with pytest.raises(InvalidInput):
        r.apply(a, pos, out=b)  # overlaps, and is not x
    with pytest.raises(InvalidInput):
        r.apply(x.as_strided((4, 2, 64), (64, 64, 1)), pos)  # tokens overlap
    with pytest.raises(TypeError):
        r.apply(x, pos.long())
    with pytest.raises(TypeError):
        r.apply(x.to(torch.float64), pos)
    with pytest.raises(ValueError):
        r.apply(x.transpose(1, 2), pos)
    with pytest.raises(ValueError):
        r.apply(x.cpu(), pos)
    with pytest.raises(ValueError):
        Rotary(64, layout="spiral")
    with pytest.raises(ValueError):
        Rotary(64, inv_freq=[1.0])
    assert r.apply(x[:0], pos[:0]).shape == (0, 2, 64)
    cache = PagedKvCache(2, 16, 2, 64, CACHE["f32"])
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(InvalidInput):
        cache.append_rotary(r, torch.zeros(4, 3, 64, device="cuda"), x, x, slots, pos)  # 3 heads over 2
    with pytest.raises(InvalidInput):
        cache.append_rotary(r, x, x, x.clone(), slots, pos, q_out=x)  # q_out is k too
    with pytest.raises(InvalidInput):
        cache.append_rotary(Rotary(128), x, x, x, slots, pos)
    with pytest.raises(TypeError):
        cache.append_rotary(r, x.half(), x, x, slots, pos)
    with pytest.raises(ValueError):
        cache.append_rotary(r, x, x[:3], x, slots, pos)
    with pytest.raises(NotImplementedOp):
        from infer_train_amd._lib import check as raise_for, lib
        raise_for(lib.it_rotary_apply(r._h, x.data_ptr(), 8, 128, pos.data_ptr(), 4, 2, 64, 0, x.data_ptr(), 128, None))


def test_append_rotary_captured_and_on_another_stream():
    import torch
    from infer_train_amd.kv import PagedKvCache, Rotary

    r, d, hkv, n = Rotary(128), 128, 2, 9
    cache, ref = PagedKvCache(4, 16, hkv, d, CACHE["bf16"]), PagedKvCache(4, 16, hkv, d, CACHE["bf16"])
    x = torch.from_numpy(values(11, n, 8, d)).cuda().bfloat16()
    pos, slots = to_dev(np.arange(n, dtype=np.int32)), to_dev(np.arange(n, dtype=np.int64) + 3)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    want = ref.append_rotary(r, q, k, v, slots, pos)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append_rotary(r, q, k, v, slots, pos, q_out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and torch.equal(cache.k_pool, ref.k_pool)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append_rotary(r, q, k, v, slots, pos, q_out=out)
    for i in range(3):
        x.copy_(torch.from_numpy(values(20 + i, n, 8, d)).cuda())
        pos.add_(100)
        graph.replay()
        torch.cuda.synchronize()
        want = ref.append_rotary(r, q, k, v, slots, pos)
        assert torch.equal(out, want) and torch.equal(cache.k_pool, ref.k_pool) and torch.equal(cache.v_pool, ref.v_pool), i


def test_rows_past_four_gibibytes():
    """The last block of pools of 4.5 GiB: appended to, moved out of, moved into; nothing else is touched."""
    import torch
    from infer_train_amd.kv import PagedKvCache, Rotary

    h, d, bs, nb = 8, 128, 16, 150000
    cache = PagedKvCache(nb, bs, h, d, CACHE["bf16"])
    assert cache.k_pool.numel() > 9 << 29
    r, n = Rotary(d), 5
    x = torch.from_numpy(values(12, n, 3 * h, d)).cuda().bfloat16()
    q, k, v = x[:, :h], x[:, h:2 * h], x[:, 2 * h:]
    last = (nb - 1) * bs
    slots, pos = to_dev(np.arange(n, dtype=np.int64) + last), to_dev(np.arange(n, dtype=np.int32))
    cache.append_rotary(r, q, k, v, slots, pos)
    want = r.apply(k, pos)
    assert torch.equal(cache.view("k")[-1, :, :n].transpose(0, 1), want) and torch.equal(cache.view("v")[-1, :, :n].transpose(0, 1), v)
    delta = to_dev(np.full(n, 100, np.int32))
    cache.move(slots, slots - last, r, delta)
    cache.move(slots - last, slots + 8)
    cache.check()
    turned = r.apply(want, delta)
    assert torch.equal(cache.view("k")[0, :, :n].transpose(0, 1), turned) and torch.equal(cache.view("k")[-1, :, 8:8 + n].transpose(0, 1), turned)
    assert torch.equal(cache.view("v")[-1, :, 8:8 + n].transpose(0, 1), v)
    assert not cache.k_pool[h * bs * d * 2:-h * bs * d * 2].any() and not cache.v_pool[h * bs * d * 2:-h * bs * d * 2].any()
