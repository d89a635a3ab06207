"""Beam search's selection and reordering on the device against a plain form in
64 bits, and a search over a paged cache against one over copied states.

Chosen beams and tokens must be equal; a score is one fp64 value rounded to
fp32 (finfo.eps / 2), whose own error is below 2^-40 of its terms."""
import math

import numpy as np
import pytest
import torch

from infer_train_amd import BF16, BlockPool, InvalidInput, KvManager
from infer_train_amd.beam import beam_reorder, beam_select, beam_select_workspace
from infer_train_amd.latent import LatentKvCache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")


def plain_select(logits, scores, n):
    z = logits.double().cpu().numpy().reshape(scores.shape[0], scores.shape[1], -1)
    z = np.where(np.isnan(z), -np.inf, z)
    sc = scores.double().cpu().numpy()
    out = np.full((z.shape[0], n), -np.inf), np.full((z.shape[0], n), -1), np.full((z.shape[0], n), -1)
    for g in range(z.shape[0]):
        cands = []
        for b in range(z.shape[1]):
            row = z[g, b]
            top = row.max()
            if top == -np.inf or not sc[g, b] > -np.inf:
                continue
            if top == np.inf:
                live = np.flatnonzero(row == np.inf)
                values = np.full(live.size, sc[g, b] - math.log(live.size))
            else:
                live = np.flatnonzero(row > -np.inf)
                values = (sc[g, b] - (top + math.log(math.fsum(np.exp(row[live] - top).tolist())))) + row[live]
            keep = np.argsort(-row[live], kind="stable")[:n]  # equal values of a beam: the larger logit first
            cands += [(-values[i], b, -row[live[i]], int(live[i])) for i in keep]
        for j, (v, b, _, i) in enumerate(sorted(cands)[:n]):
            out[0][g, j], out[1][g, j], out[2][g, j] = -v, b, i
    return out


def check(logits, scores, n, **kw):
    got = [x.cpu().numpy() for x in beam_select(logits.to(DEV), scores.to(DEV), n, **kw)]
    want = plain_select(logits, scores, n)
    assert np.array_equal(got[1], want[1]), "parents"
    assert np.array_equal(got[2], want[2]), "tokens"
    fin, one = np.isfinite(want[0]), np.nan_to_num(want[0], neginf=0.0, posinf=0.0)
    assert np.array_equal(np.isfinite(got[0]), fin) and np.array_equal(got[0][~fin], want[0][~fin])
    big, diff = np.maximum(np.abs(one), 64.0), np.abs(np.where(fin, got[0], 0.0) - one)
    assert (diff[fin] <= (2.0 ** -24 * np.abs(one) + 2.0 ** -40 * big)[fin]).all()
    return got


def logits_of(seed, rows, vocab, dtype, spread=3.0):
    g = torch.Generator()
    g.manual_seed(seed)
    return (spread * torch.randn(rows, vocab, generator=g)).to(dtype), -20 * torch.rand(rows, generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("groups,beams,vocab,n", [(1, 1, 1, 1), (1, 4, 3, 8), (2, 3, 63, 6), (3, 5, 8192, 10), (2, 4, 8193, 64), (5, 8, 32001, 16),
                                                  (1, 64, 1000, 64), (2, 2, 262144, 4)])
def test_select(dtype, groups, beams, vocab, n):
    z, s = logits_of(vocab + n, groups * beams, vocab, dtype)
    check(z, s.view(groups, beams), n)


def test_select_first_step_and_unused_beams():
    """All beams alike but one in use; none in use; a score of NaN."""
    z, _ = logits_of(1, 3, 5000, torch.float32)
    z = z.repeat_interleave(4, 0)
    s = torch.tensor([[0.0, -INF, -INF, -INF], [-INF] * 4, [float("nan"), -INF, -3.0, -INF]])
    got = check(z, s, 8)
    assert (got[1][0] == 0).all() and (got[1][1] == -1).all() and (got[1][2] == 2).all()


def test_select_ties_go_to_the_lower_beam_and_token():
    """Equal beams, equal logits (more than any list holds), and both zeros."""
    check(torch.zeros(4, 20000), torch.zeros(1, 4), 64)
    check(torch.full((3, 9000), -2.5), torch.tensor([[0.0, 0.0, 1.0]]), 7)
    z, _ = logits_of(2, 1, 3000, torch.bfloat16)
    check(z.repeat(6, 1), torch.zeros(2, 3), 12)
    z = torch.full((2, 10000), -1.0)
    z[:, 5000:] = 0.0
    z[:, 7001::2] = -0.0
    check(z, torch.tensor([[0.0, 0.0]]), 64)


def test_select_masked_rows():
    """Rows with few tokens, one, none; the type's lowest value; infinities and NaN."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        z, s = logits_of(3, 12, 9001, dtype)
        g = torch.Generator()
        g.manual_seed(4)
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
        check(z, s.view(3, 4), 16)
        check(z, s.view(1, 12), 24)
        check(z, s.view(12, 1), 64)


def test_select_flat_and_peaked_rows():
    z, s = logits_of(5, 4, 100003, torch.float32, spread=1e-3)
    check(z, s.view(1, 4), 8)
    z, s = logits_of(6, 4, 100003, torch.float32, spread=30.0)
    check(z, s.view(2, 2), 4)
    check(z.double().mul(1e36).float(), s.view(2, 2), 4)


def test_select_strides_and_batches():
    """Rows inside a wider tensor, at odd offsets; a group's result is its own in any batch."""
    z, s = logits_of(7, 6, 5003, torch.float16)
    wide = torch.zeros(6, 6001, dtype=torch.float16)
    wide[:, 5:5008] = z
    whole = check(wide[:, 5:5008], s.view(3, 2), 6)
    d = wide.to(DEV)[:, 5:5008]
    got = [x.cpu().numpy() for x in beam_select(d, s.view(3, 2).to(DEV), 6)]
    for a, b in zip(whole, got):
        assert np.array_equal(a, b)
    one = [x.cpu().numpy() for x in beam_select(d[2:4], s[2:4].view(1, 2).to(DEV), 6)]
    for a, b in zip(whole, one):
        assert np.array_equal(a[1:2], b)
    assert [x.shape for x in beam_select(d[:0], s[:0].view(0, 2).to(DEV), 6)] == [(0, 6)] * 3


def test_select_replayed_from_a_graph():
    z, s = logits_of(8, 8, 30000, torch.bfloat16)
    zd, sd = z.to(DEV), s.view(2, 4).to(DEV)
    beam_select(zd, sd, 8)
    graph, ws = torch.cuda.CUDAGraph(), beam_select_workspace(2, 4, 30000, 8, DEV)
    with torch.cuda.graph(graph):
        out = beam_select(zd, sd, 8, ws=ws)
    for i in range(4):
        zd.mul_(-1.0 if i % 2 else 0.5)
        sd.sub_(1.0)
        want = beam_select(zd, sd, 8)
        for o in out:
            o.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


# ---- reorder -------------------------------------------------------------------
def reordered(x, parents, dim):
    rows = torch.arange(parents.numel()).view(parents.shape)
    base = rows - rows % parents.shape[1]
    ok = (parents >= 0) & (parents < parents.shape[1])
    return x.index_select(dim, torch.where(ok, base + parents, rows).view(-1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.int32, torch.bfloat16, torch.uint8, torch.int64])
@pytest.mark.parametrize("groups,beams", [(1, 1), (3, 2), (2, 4), (5, 5), (1, 8), (2, 16), (3, 17), (1, 33), (1, 64)])
def test_reorder(dtype, groups, beams):
    g = torch.Generator()
    g.manual_seed(groups * 100 + beams)
    for shape, dim in (((groups * beams, 2048), 0), ((3, groups * beams, 7, 5), 1), ((2, 2, groups * beams), 2), ((groups * beams, 33), -2)):
        x = torch.randint(0, 100, shape, generator=g).to(dtype)
        parents = torch.randint(-1, beams, (groups, beams), generator=g, dtype=torch.int32)
        parents[0, 0] = beams + 3  # no beam: it stays
        d = x.to(DEV)
        assert beam_reorder(d, parents.to(DEV), dim=dim) is d
        assert torch.equal(d.cpu(), reordered(x, parents, dim))


def test_reorder_part_of_a_tensor():
    """An offset that no vector is aligned to; what is around it stays."""
    x = torch.arange(1000, dtype=torch.int16)
    d = x.to(DEV)
    parents = torch.tensor([[2, 2, 0], [1, 0, 0]], dtype=torch.int32)
    beam_reorder(d[1:1 + 6 * 13].view(6, 13), parents.to(DEV))
    want = x.clone()
    want[1:79] = reordered(x[1:79].view(6, 13), parents, 0).view(-1)
    assert torch.equal(d.cpu(), want)
    empty = torch.zeros(6, 0, device=DEV)
    assert beam_reorder(empty, parents.to(DEV)).numel() == 0
    assert beam_reorder(torch.zeros(0, 4, device=DEV), torch.zeros(0, 3, dtype=torch.int32, device=DEV)).numel() == 0


# ---- together --------------------------------------------------------------------
def test_beams_over_a_latent_cache():
    """A search of three requests, four beams each, over one paged latent cache:
    blocks shared and copied on write, tables and histories reordered on the
    device.  Each step's attention equals that over every beam's own copied rows,
    and the pool ends where it began."""
    groups, beams, heads, latent, rope, bs, vocab, steps = 3, 4, 4, 256, 32, 8, 500, 21
    g = torch.Generator()
    g.manual_seed(1)
    n = groups * beams
    pool = BlockPool(120, BF16)
    mgr = KvManager(pool, bs, n, 12)
    c = LatentKvCache(120, bs, latent, rope, BF16, n_layers=2)
    layers = [c.layer(0), c.layer(1)]
    tables = torch.full((n, 12), -1, dtype=torch.int32, device=DEV)
    table_w = torch.randn(vocab, latent + rope, generator=g)  # a token's row, and its logits' weights
    head_w = torch.randn(latent, vocab, generator=g) * 0.3
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    copies = [torch.zeros(0, 2, latent + rope, dtype=torch.bfloat16) for _ in range(n)]

    def write(plan, rows):  # rows [tokens, 2, row]
        if plan.cow_src.size:
            c.copy_blocks(to(plan.cow_src), to(plan.cow_dst))
        slots = to(plan.slots)
        for i, layer in enumerate(layers):
            layer.append(rows[:, i].to(DEV), slots)
        c.sync_tables(tables, to(plan.token_seq), to(plan.token_pos), slots)
        return to(plan.ctx_lens)

    def rows_of(tokens):
        x = table_w[tokens]
        return torch.stack((x, -0.5 * x.flip(-1)), 1).to(torch.bfloat16)

    prompts = [torch.randint(0, vocab, (m,), generator=g) for m in (5, 16, 11)]
    first = [i * beams for i in range(groups)]
    ctx = write(mgr.append(first, [len(p) for p in prompts]), torch.cat([rows_of(p) for p in prompts]))
    for i in range(groups):
        copies[first[i]] = rows_of(prompts[i])
        for b in range(1, beams):
            mgr.fork(first[i], first[i] + b)
            copies[first[i] + b] = copies[first[i]]
    parents0 = torch.zeros(groups, beams, dtype=torch.int32, device=DEV)
    beam_reorder(tables, parents0)
    ctx = torch.from_numpy(mgr.positions()).to(DEV)
    scores = torch.full((groups, beams), -INF, device=DEV)
    scores[:, 0] = 0.0
    history = torch.zeros(n, steps, dtype=torch.int32, device=DEV)
    lists = [[] for _ in range(n)]
    shared = 0
    for step in range(steps):
        q = torch.randn(n, heads, latent + rope, generator=g).to(torch.bfloat16)
        q[:] = q[::beams].repeat_interleave(beams, 0)
        outs = [layer.decode(q.to(DEV)[..., :latent], q.to(DEV)[..., latent:], tables, ctx, int(ctx.max()), 0.06, out_dtype=torch.float32)
                for layer in layers]
        for i in range(2):
            for s in range(n):
                rows = copies[s][:, i].double()
                p = torch.softmax(q[s].double() @ rows.t() * 0.06, 1)
                want, mag = p @ rows[:, :latent], p @ rows[:, :latent].abs()
                # weights to bf16 (2^-8 each, in sum and result), scores to 160 roundings of fp32
                terms = (q[s].double().abs() @ rows.abs().t() * 0.06).amax()
                assert ((outs[i][s].cpu().double() - want).abs() <= (2 * 2.0 ** -8 + 320 * 2.0 ** -24 * terms + 2.0 ** -20) * mag).all(), (step, i, s)
        logits = (outs[0].mean(1) - outs[1].mean(1)).cpu() @ head_w * 8
        best, parents, tokens = beam_select(logits.to(DEV), scores, 2 * beams)
        want = plain_select(logits, scores, 2 * beams)
        assert np.array_equal(parents.cpu().numpy(), want[1]) and np.array_equal(tokens.cpu().numpy(), want[2])
        keep = torch.tensor([i for i in range(2 * beams) if (i + step) % 3 != 2][:beams])  # as if some had ended
        keep = keep.to(DEV)
        scores, parents, tokens = best[:, keep].contiguous(), parents[:, keep].contiguous(), tokens[:, keep]
        evicted = mgr.reorder(list(range(n)), (parents.cpu() + torch.tensor(first)[:, None]).view(-1).tolist())
        if evicted.size:
            c.evict(to(evicted))
        beam_reorder(tables, parents)
        beam_reorder(history, parents)
        history[:, step] = tokens.reshape(-1)
        flat = [first[j // beams] + int(p) for j, p in enumerate(parents.cpu().view(-1).tolist())]
        copies = [copies[p] for p in flat]
        lists = [lists[p] + [int(t)] for p, t in zip(flat, tokens.cpu().reshape(-1).tolist())]
        seqs = list(range(n))
        shared += mgr.needs_cow(seqs)
        if mgr.needs_cow(seqs):
            with pytest.raises(InvalidInput):
                mgr.append(seqs, 1)
        new = rows_of(tokens.cpu().reshape(-1).long())
        ctx = write(mgr.append(seqs, 1, cow=True), new)
        copies = [torch.cat((a, b[None])) for a, b in zip(copies, new)]
        t, cl, _ = mgr.tables()
        held = (cl + bs - 1) // bs
        dev_t = tables.cpu().numpy()
        for s in range(n):
            assert np.array_equal(dev_t[s, :held[s]], t[s, :held[s]]), s
    c.check()
    assert shared > steps // 2
    assert history.cpu().tolist() == lists
    for s in range(n):
        mgr.release(s)
    assert pool.num_free() == 120


def test_refusals():
    z, s = torch.zeros(4, 50, device=DEV), torch.zeros(2, 2, device=DEV)
    with pytest.raises(InvalidInput):
        beam_select(z, s, 65)
    with pytest.raises(InvalidInput):
        beam_select(z, s, 0)
    with pytest.raises(TypeError):
        beam_select(z, s.double())
    with pytest.raises(TypeError):
        beam_select(z, s[:1])
    with pytest.raises(TypeError):
        beam_select(z.double(), s)
    with pytest.raises(ValueError):
        beam_select(z.t(), s)
    with pytest.raises(ValueError):
        beam_select(z.cpu(), s)
    with pytest.raises(InvalidInput):
        beam_select(z, s, ws=torch.empty(256, dtype=torch.uint8, device=DEV))
    with pytest.raises(InvalidInput):
        beam_select(torch.zeros(65, 50, device=DEV), torch.zeros(1, 65, device=DEV), 4)
    p = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    with pytest.raises(TypeError):
        beam_reorder(z, p.long())
    with pytest.raises(ValueError):
        beam_reorder(z[:3], p)
    with pytest.raises(ValueError):
        beam_reorder(z.t(), p, dim=1)
    with pytest.raises(ValueError):
        beam_reorder(z, p, dim=2)
    with pytest.raises(ValueError):
        beam_reorder(z.clone().requires_grad_(), p)
    with pytest.raises(InvalidInput):
        beam_reorder(p.view(4, 1), p)
