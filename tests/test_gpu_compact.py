"""Compaction on the device beside forks and other sequences: pages hold what the
host's lists say, after moves, copies, evictions and appends in the documented
order.  Rows are float32 copies, compared bit for bit."""
import numpy as np
import pytest

from kvutil import to_dev

pytestmark = pytest.mark.gpu


class Rows:
    """A cache of small float32 rows, each filled with its token's number."""

    def __init__(self, pool_blocks, bs, n_seqs):
        from infer_train_amd import BlockPool, F32, KvManager
        from infer_train_amd.kv import PagedKvCache

        self.pool, self.bs = BlockPool(pool_blocks, F32), bs
        self.mgr = KvManager(self.pool, bs, n_seqs, pool_blocks)
        self.cache = PagedKvCache(pool_blocks, bs, 2, 8, F32, n_layers=2)
        self.views = [self.cache.layer(i) for i in range(2)]
        self.tokens, self.next = {s: [] for s in range(n_seqs)}, 1

    def run(self, plan):
        """A step's device work."""
        import torch

        if plan.cow_src.size:
            self.cache.copy_blocks(to_dev(plan.cow_src), to_dev(plan.cow_dst))
        if plan.evicted.size:
            self.cache.evict(to_dev(plan.evicted))
        ids = torch.arange(self.next, self.next + plan.slots.size, device="cuda", dtype=torch.float32)
        for i, view in enumerate(self.views):
            k = (ids + 10000 * i)[:, None, None].expand(-1, 2, 8).contiguous()
            view.append(k, -k, to_dev(plan.slots))
        for s in plan.token_seq.tolist():
            self.tokens[s].append(self.next)
            self.next += 1

    def compact(self, plan, keeps):
        if plan.src.size:
            self.cache.move(to_dev(plan.src), to_dev(plan.dst))
        if plan.evicted.size:
            self.cache.evict(to_dev(plan.evicted))
        for s, keep in keeps.items():
            self.tokens[s] = [self.tokens[s][i] for i in keep]

    def check(self):
        self.cache.check()
        tables, ctx, _ = self.mgr.tables()
        held = set(tables[tables >= 0].tolist())
        for i, view in enumerate(self.views):
            k, v = view.view("k").cpu().numpy(), view.view("v").cpu().numpy()
            for s, want in self.tokens.items():
                assert ctx[s] == len(want)
                for p, x in enumerate(want):
                    b, o = tables[s, p // self.bs], p % self.bs
                    assert (k[b, :, o] == x + 10000 * i).all() and (v[b, :, o] == -x - 10000 * i).all(), (i, s, p)
            for b in set(range(k.shape[0])) - held:  # returned pages are clear, a dropped tail's too
                assert not k[b].any() and not v[b].any(), (i, b)


@pytest.mark.parametrize("bs,ctx,tail", ((4, 15, 13), (16, 47, 17), (4, 16, 8), (1, 6, 2)))
def test_decode_after_a_dropped_tail_beside_a_fork(bs, ctx, tail):
    from infer_train_amd import ContinuousBatcher

    r = Rows(40, bs, 4)
    b = ContinuousBatcher(2, r.mgr)
    b.add_request(0, list(range(ctx)), 99)
    b.add_request(1, list(range(5)), 99)
    b.schedule()
    r.run(b.plan_prefill([0, 1]))
    seq = b.seq_of[0]
    r.mgr.fork(seq, 3)
    r.tokens[3] = list(r.tokens[seq])
    r.compact(r.mgr.compact(seq, range(tail)), {seq: range(tail)})
    r.check()
    for _ in range(bs + 2):
        r.run(b.plan_decode())
        r.check()
    r.run(r.mgr.append([3], bs + 1, cow=True))
    r.check()
    r.compact(r.mgr.compact(3, range(1)), {3: range(1)})  # unshared by now: whole blocks of a tail are cleared
    r.check()


def test_several_sequences_in_one_move():
    """Three sequences and a fork of one compacted together, in one move and one eviction."""
    r = Rows(40, 4, 5)
    r.run(r.mgr.append([0, 1, 2], [30, 25, 17]))
    r.mgr.fork(1, 3)
    r.tokens[3] = list(r.tokens[1])
    rng = np.random.default_rng(1)
    for _ in range(3):
        keeps = {s: np.flatnonzero(rng.random(len(r.tokens[s])) < 0.4).tolist() for s in range(4)}
        plan = r.mgr.compact_many(list(keeps), list(keeps.values()))
        assert plan.src.size
        r.compact(plan, keeps)
        r.check()
        r.run(r.mgr.append([0, 2], [13, 15], cow=True))
        r.check()


def test_tokens_are_drawn_for_the_requests_just_prefilled():
    """A request admitted while others decode: its first token comes from its own row, and joins it alone."""
    import torch
    from infer_train_amd import BlockPool, ContinuousBatcher, F32, KvManager, SamplingParams
    from test_gpu_sample import logits, reference

    b = ContinuousBatcher(3, KvManager(BlockPool(32, F32), 4, 3, 16))
    settings = {0: SamplingParams(0.7, 40, 0.9, 0.01), 1: SamplingParams(0.0), 2: SamplingParams(1.3, 0, 0.8)}
    seed = iter(range(100))

    def draw(ids):
        z, u = logits(next(seed), len(ids), 3001), np.random.default_rng(next(seed)).random(len(ids)).astype(np.float32)
        got = b.sample(torch.from_numpy(z).cuda(), to_dev(u), ids)
        for row, rid in enumerate(ids):
            s = settings[rid]
            want = reference(z[row], float(u[row]), float(np.float32(s.temperature)), s.top_k, float(np.float32(s.top_p)),
                             float(np.float32(s.min_p)))[0]
            assert got[row] == want == b.requests[rid].generated_tokens[-1]

    for new in ([0, 1], [2]):
        for rid in new:
            b.add_request(rid, list(range(6 + rid)), 9, settings[rid])
        b.schedule()
        b.plan_prefill(new)
        draw(new)
        b.plan_decode()
        draw(list(b.running))
    assert [len(b.requests[i].generated_tokens) for i in range(3)] == [3, 3, 2]
    assert b.manager.positions().tolist() == [6 + 2, 7 + 2, 8 + 1]
