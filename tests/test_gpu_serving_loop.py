"""The operators together, as a serving loop uses them: a batch of requests is
prefilled (rotary append, chunked attention), decoded step by step (rotary
append of a fused projection, paged decode, logits, one drawn token per
request), compacted in mid-generation (tokens dropped out of the middle, keys
turned to their new positions, pages given back) and decoded on.

Every step's attention is compared with float64 softmax attention over rows
kept on the host: unrotated keys in the cache's dtype, rotated to the positions
that they have at that step.  Tolerance: keys are rounded to bf16 after each of
at most two rotations (2^-8 of a key's pair each), queries once: a score is off
by 3 2^-8 of |q| |k| / sqrt(D) at worst and by its root-mean-square over D terms
in fact; with |score| ~ 1 that moves an output by about 3 2^-8 / sqrt(D) of the
values' spread, and the decode's own bf16 output by 2^-8: 2e-2 + 1e-2 |out|
covers four times that."""
import numpy as np
import pytest

from kvutil import to_dev
from test_gpu_rotary import exact_turn
from test_gpu_sample import reference

pytestmark = pytest.mark.gpu


def test_prefill_decode_compact_decode():
    import torch
    from infer_train_amd import BF16, BlockPool, ContinuousBatcher, KvManager, SamplingParams
    from infer_train_amd.kv import PagedKvCache, Rotary

    hq, hkv, d, bs, nb, layers, vocab = 8, 2, 128, 16, 160, 2, 2003
    pool = BlockPool(nb, BF16)
    mgr = KvManager(pool, bs, 4, 40)
    batcher = ContinuousBatcher(4, mgr)
    cache = PagedKvCache(nb, bs, hkv, d, BF16, n_layers=layers)
    views = [cache.layer(i) for i in range(layers)]
    rotary = Rotary(d, scaling="parts", factor=4.0, original_ctx=64, low=1.0, high=32.0)
    gen = torch.Generator(device="cuda").manual_seed(5)
    rng = np.random.default_rng(5)
    prompts = [70, 33, 129]
    for i, n in enumerate(prompts):
        batcher.add_request(i, list(range(n)), 40, SamplingParams(temperature=0.8, top_k=40, top_p=0.95))
    batcher.schedule()
    tables = torch.full((4, 40), -1, dtype=torch.int32, device="cuda")
    rows = [[([], []) for _ in range(4)] for _ in range(layers)]  # per layer and sequence: k before rotation, v
    positions = [[] for _ in range(4)]

    def project(n):
        return torch.randn(n, hq + 2 * hkv, d, generator=gen, device="cuda").bfloat16()

    def remember(layer, seqs, k, v):
        for s, kk, vv in zip(seqs, k.double().cpu().numpy(), v.double().cpu().numpy()):
            rows[layer][s][0].append(kk)
            rows[layer][s][1].append(vv)

    def expect(layer, s, q, upto):
        """q [hq, d] unrotated at the last of the positions -> attention over the first `upto` rows."""
        k, _ = exact_turn(np.stack(rows[layer][s][0][:upto]), np.array(positions[s][:upto]), rotary.inv_freq, 1.0, "half")
        v = np.stack(rows[layer][s][1][:upto])
        qr, _ = exact_turn(q[None], np.array([positions[s][upto - 1]]), rotary.inv_freq, 1.0, "half")
        out = np.empty((hq, d))
        for h in range(hq):
            sc = k[:, h * hkv // hq] @ qr[0, h] / np.sqrt(d)
            p = np.exp(sc - sc.max())
            out[h] = p @ v[:, h * hkv // hq] / p.sum()
        return out

    def close(got, want, what):
        got = got.double().cpu().numpy()
        assert (np.abs(got - want) <= 2e-2 + 1e-2 * np.abs(want)).all(), (what, np.abs(got - want).max())

    def apply_plan(plan):
        if plan.evicted.size:
            cache.evict(to_dev(plan.evicted))
        seq, pos, slots = to_dev(plan.token_seq), to_dev(plan.token_pos), to_dev(plan.slots)
        cache.sync_tables(tables, seq, pos, slots)
        return pos, slots

    plan = batcher.plan_prefill([0, 1, 2])
    seqs = [batcher.seq_of[i] for i in range(3)]
    pos, slots = apply_plan(plan)
    for s, p in zip(plan.token_seq, plan.token_pos):
        positions[s].append(int(p))
    n = plan.slots.size
    cu = to_dev(np.concatenate([[0], np.cumsum(prompts)]).astype(np.int32))
    ctx = to_dev(plan.ctx_lens[seqs])
    for i, view in enumerate(views):
        x = project(n)
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        remember(i, plan.token_seq, k, v)
        qr = view.append_rotary(rotary, q, k, v, slots, pos)
        out = view.prefill(qr, cu, max(prompts), tables[seqs].contiguous(), ctx)
        for j, s in enumerate(seqs):
            at = sum(prompts[:j])
            for t in (0, prompts[j] // 2, prompts[j] - 1):
                close(out[at + t], expect(i, s, q[at + t].double().cpu().numpy(), t + 1), ("prefill", i, j, t))

    def decode_step():
        plan = batcher.plan_decode()
        order = [batcher.seq_of[r] for r in batcher.running]
        pos, slots = apply_plan(plan)
        for s, p in zip(plan.token_seq, plan.token_pos):
            positions[s].append(int(p))
        lens = plan.ctx_lens[order]
        for i, view in enumerate(views):
            x = project(len(order))
            q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
            remember(i, order, k, v)
            qr = view.append_rotary(rotary, q, k, v, slots, pos)
            out = view.decode(qr, tables[order].contiguous(), to_dev(lens), None, int(lens.max()), partition=64)
            for j, s in enumerate(order):
                assert len(positions[s]) == lens[j]
                close(out[j], expect(i, s, q[j].double().cpu().numpy(), int(lens[j])), ("decode", i, j))
        z = torch.randn(len(order), vocab, generator=gen, device="cuda") * 3
        u = torch.from_numpy(rng.random(len(order)).astype(np.float32)).cuda()
        got = batcher.sample(z, u)
        want = [reference(a, float(b), float(np.float32(0.8)), 40, float(np.float32(0.95)), 0.0)[0]
                for a, b in zip(z.double().cpu().numpy(), u.cpu().numpy())]
        assert got == want

    for _ in range(3):
        decode_step()
    # A fork keeps the tokens that its parent is about to drop.
    mgr.fork(seqs[2], 3)
    tables[3] = tables[seqs[2]]
    for layer in rows:
        layer[3] = (list(layer[seqs[2]][0]), list(layer[seqs[2]][1]))
    positions[3] = list(positions[seqs[2]])
    free = pool.num_free()
    for s, keep in ((seqs[0], list(range(4)) + list(range(40, len(positions[seqs[0]])))),
                    (seqs[2], list(range(20)) + sorted(rng.choice(np.arange(20, 120), 30, replace=False).tolist()) +
                     list(range(120, len(positions[seqs[2]])))), (seqs[1], list(range(len(positions[seqs[1]]) - 2)))):
        plan = mgr.compact(s, keep)
        if plan.src.size:
            cache.move(to_dev(plan.src), to_dev(plan.dst), rotary, to_dev(plan.delta))
            if plan.evicted.size:
                cache.evict(to_dev(plan.evicted))
            cache.sync_tables(tables, to_dev(plan.token_seq), to_dev(plan.token_pos), to_dev(plan.dst))
        for layer in rows:
            layer[s] = tuple([x[t] for t in keep] for x in layer[s])
        positions[s] = list(range(len(keep)))
    assert pool.num_free() != free
    for _ in range(2):
        decode_step()
    cache.check()
    for i, view in enumerate(views):  # the fork reads what it held before
        q = project(1)[:, :hq]
        qr = rotary.apply(q, to_dev(np.array([positions[3][-1]], np.int32)))
        n = len(positions[3])
        out = view.decode(qr, tables[3:4].contiguous(), to_dev(np.array([n], np.int32)), None, n, partition=64)
        close(out[0], expect(i, 3, q[0].double().cpu().numpy(), n), ("fork", i))
