"""Rotary.apply under autograd: the gradient of <g, R x> is R^T g, which the
library computes by the same kernel with its flag turned.

Against the formula in 64 bits with test_gpu_rotary's tolerances (its head note)
and, elementwise, against differences: R is linear, so that a central difference
over a step of 2 is exact but for the rounding of fp32 outputs."""
import numpy as np
import pytest

from kvutil import to_dev
from test_gpu_rotary import check, exact_turn, torch_dtype, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("transpose", (False, True))
@pytest.mark.parametrize("layout,d,rot,name", (("half", 128, 128, "f32"), ("interleaved", 80, 80, "f32"), ("half", 96, 20, "bf16"),
                                               ("interleaved", 64, 32, "f16")))
def test_backward(layout, d, rot, name, transpose):
    import torch
    from infer_train_amd.kv import Rotary

    n, h = 7, 3
    r = Rotary(rot, layout, magnitude=1.5)
    x = torch.from_numpy(values(1, n, h, d)).cuda().to(torch_dtype(name)).requires_grad_()
    g = torch.from_numpy(values(2, n, h, d)).cuda().to(torch_dtype(name))
    pos = np.random.default_rng(3).integers(-50, 100000, n).astype(np.int32)
    y = r.apply(x, to_dev(pos), transpose=transpose)
    assert y.requires_grad and y.grad_fn is not None
    with torch.no_grad():
        assert torch.equal(r.apply(x, to_dev(pos), transpose=transpose), y)
    y.backward(g)
    assert torch.equal(x.grad, r.apply(g, to_dev(pos), transpose=not transpose))
    want, tol = exact_turn(g.double().cpu().numpy(), pos, r.inv_freq, 1.5, layout, not transpose)
    check(x.grad, want, tol, name)


def test_backward_against_differences():
    """Outputs of a pair are below 1.5 (|a| + |b|) <= 18 and off by 2^-20.5 of that, two of them times |g| < 5 over a step of
    2; the gradient itself by 2^-20 of 15 (as in test_gpu_rotary's test of the transpose)."""
    import torch
    from infer_train_amd.kv import Rotary

    r = Rotary(24, "half", magnitude=1.5)
    x, g = torch.from_numpy(values(7, 3, 2, 32)).cuda().requires_grad_(), torch.from_numpy(values(8, 3, 2, 32)).cuda()
    assert float(x.detach().abs().max()) < 5 and float(g.abs().max()) < 5
    pos = to_dev(np.array([0, 17, 4095], np.int32))
    (r.apply(x, pos) * g).sum().backward()
    with torch.no_grad():
        for t, i, e in ((0, 0, 0), (1, 1, 5), (2, 0, 11), (2, 1, 23), (1, 0, 31)):
            up, down = x.clone(), x.clone()
            up[t, i, e] += 1.0
            down[t, i, e] -= 1.0
            step = float(up[t, i, e].double() - down[t, i, e].double())
            diff = float(((r.apply(up, pos).double() - r.apply(down, pos).double()) * g.double()).sum()) / step
            assert abs(diff - float(x.grad[t, i, e])) < 2 * 2 * 5 * 18 * 2.0 ** -20 / 2 + 2.0 ** -20 * 15


def test_gradients_of_views_and_broadcasts():
    """Slices of a fused projection collect their gradients in it; broadcast and strided gradients are taken; a gradient of the
    gradient is the rotation again."""
    import torch
    from infer_train_amd.kv import Rotary

    r, n, hq, hkv, d = Rotary(64), 5, 4, 2, 64
    pos = to_dev(np.arange(n, dtype=np.int32) * 37)
    qkv = torch.from_numpy(values(4, n, hq + 2 * hkv, d)).cuda().requires_grad_()
    q, k = r.apply(qkv[:, :hq], pos), r.apply(qkv[:, hq:hq + hkv], pos)
    (q.sum() + (k * 2).sum()).backward()  # the gradient of sum() has no strides
    ones = torch.ones(n, hq + hkv, d, device="cuda")
    ones[:, hq:] = 2.0
    want = torch.cat((r.apply(ones[:, :hq].contiguous(), pos, transpose=True),
                      r.apply(ones[:, hq:].contiguous(), pos, transpose=True), torch.zeros(n, hkv, d, device="cuda")), 1)
    assert torch.equal(qkv.grad, want)
    x = torch.from_numpy(values(5, n, hq, d)).cuda().requires_grad_()
    for g in (torch.ones(n, 1, d, device="cuda").expand(n, hq, d), torch.ones(1, hq, d, device="cuda").expand(n, hq, d),
              torch.ones(n, d, hq, device="cuda").transpose(1, 2), torch.ones(n, hq + 3, d, device="cuda")[:, :hq],
              torch.ones(n, hq, 2 * d, device="cuda")[..., ::2]):
        grad, = torch.autograd.grad(r.apply(x, pos), x, g)
        assert torch.equal(grad, r.apply(g.contiguous(), pos, transpose=True))
    one = torch.from_numpy(values(6, 1, 1, d)).cuda().requires_grad_()
    grad, = torch.autograd.grad(r.apply(one, pos[:1]).sum(), one)
    assert grad.shape == one.shape
    empty = x[:0]
    assert torch.autograd.grad(r.apply(empty, pos[:0]).sum(), x)[0].eq(0).all()
    g = torch.from_numpy(values(9, n, hq, d)).cuda().requires_grad_()
    grad, = torch.autograd.grad(r.apply(x, pos), x, g, create_graph=True)
    again, = torch.autograd.grad(grad, g, x.detach())
    assert torch.equal(again, r.apply(x.detach(), pos))


def test_out_and_autograd():
    """out under autograd is refused; a tensor or positions saved for a backward pass and changed since are found out."""
    import torch
    from infer_train_amd.kv import Rotary

    r, pos = Rotary(64), to_dev(np.arange(3, dtype=np.int32))
    x = torch.from_numpy(values(5, 3, 2, 64)).cuda()
    leaf, buf = x.clone().requires_grad_(), torch.empty_like(x)
    for a, out in ((leaf, buf), (leaf, leaf), (x, leaf)):
        with pytest.raises(ValueError):
            r.apply(a, pos, out=out)
    assert torch.equal(leaf.detach(), x)
    with torch.no_grad():
        assert r.apply(leaf, pos, out=buf) is buf
    with torch.inference_mode():
        y = x.clone()
        assert r.apply(y, pos, out=y) is y and torch.equal(y, buf)
    w = x.clone().requires_grad_()
    kept = x.clone()
    loss = (w * kept).sum()  # saves kept
    r.apply(kept, pos, out=kept)
    with pytest.raises(RuntimeError):
        loss.backward()
    y = r.apply(leaf, pos)
    pos.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_training_step_captured():
    """Forward and backward in a graph, replayed with new inputs, against eager steps after the replays."""
    import torch
    from infer_train_amd.kv import Rotary

    r, pos = Rotary(128), to_dev(np.arange(9, dtype=np.int32))
    x = torch.from_numpy(values(1, 9, 4, 128)).cuda().requires_grad_()
    g = torch.from_numpy(values(2, 9, 4, 128)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(r.apply(x, pos), x, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = r.apply(x, pos)
        grad, = torch.autograd.grad(y, x, g)
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.from_numpy(values(10 + i, 9, 4, 128)))
        g.copy_(torch.from_numpy(values(20 + i, 9, 4, 128)))
        pos.add_(1000)
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(y, r.apply(x, pos)) and torch.equal(grad, r.apply(g, pos, transpose=True)), i
