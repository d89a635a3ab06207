"""Beams on the host: sequences reordered in the manager against a list model,
requests in the batcher, and the new entry points' refusals before any device."""
import ctypes as C

import numpy as np
import pytest

from infer_train_amd import BF16, BlockPool, ContinuousBatcher, InvalidInput, KvManager
from infer_train_amd import _lib as L


class Model:
    """Sequences as lists of (block, tokens): what the manager's tables say, by copying."""

    def __init__(self, pool, mgr):
        self.pool, self.mgr, self.tokens = pool, mgr, {}

    def check(self, pages):
        t, ctx, _ = self.mgr.tables()
        for s, tokens in self.tokens.items():
            assert ctx[s] == len(tokens)
            for p, tok in enumerate(tokens):
                assert pages[t[s, p // self.mgr.block_size], p % self.mgr.block_size] == tok, (s, p)
        held = {}
        for row in t:
            for b in row[row >= 0]:
                held[int(b)] = held.get(int(b), 0) + 1
        assert all(self.pool.ref_count(b) == n for b, n in held.items())
        assert self.pool.num_free() == self.pool.capacity() - len(held)


@pytest.mark.parametrize("window", [0, 24])
def test_reorder_random_searches(window):
    """Random selections, steps with copy-on-write, releases: every sequence's
    tokens are found through its table, references and free blocks add up, and
    returned blocks are those that nobody holds."""
    rng = np.random.default_rng(window)
    bs, n, cap = 8, 6, 200
    pool = BlockPool(cap, BF16)
    mgr = KvManager(pool, bs, n + 1, 16, window=window)
    pages = np.full((cap, bs), -1, np.int64)
    model, tok = Model(pool, mgr), 0

    def step(seqs, count):
        nonlocal tok
        plan = mgr.append(seqs, count, cow=True)
        for a, b in zip(plan.cow_src, plan.cow_dst):
            pages[b] = pages[a]
        for b in plan.evicted:
            pages[b] = -1
        for slot, s in zip(plan.slots, plan.token_seq):
            model.tokens[int(s)] = model.tokens[int(s)] + [tok]
            pages[slot // bs, slot % bs] = tok
            tok += 1

    model.tokens = {s: [] for s in range(n)}
    step([0], 13)
    for s in range(1, n):
        mgr.fork(0, s)
        model.tokens[s] = model.tokens[0]
    seqs = list(range(n))
    for turn in range(60):
        if min(len(t) for t in model.tokens.values()) > 100:
            break
        parents = rng.integers(-1, n, n)
        refs = {b: pool.ref_count(b) for b in range(cap)}
        t, _, _ = mgr.tables()
        freed = mgr.reorder(seqs, parents)
        assert len(set(freed.tolist())) == freed.size
        assert all(pool.ref_count(int(b)) == 0 < refs[int(b)] for b in freed)
        pages[freed] = -1
        of = [i if p < 0 else int(p) for i, p in enumerate(parents)]
        model.tokens = {s: model.tokens[p] for s, p in zip(seqs, of)}
        partial = any(len(model.tokens[s]) % bs for s in seqs) and len(set(of)) < n
        if mgr.needs_cow(seqs):
            assert partial
            before = mgr.tables()[0].copy()
            with pytest.raises(InvalidInput, match="copy-on-write"):
                mgr.append(seqs, 1)
            assert np.array_equal(before, mgr.tables()[0])
        if window == 0:
            model.check(pages)
        step(seqs, int(rng.integers(1, 4)))
        if window == 0:
            model.check(pages)
    for s in seqs:
        mgr.release(s)
    assert pool.num_free() == cap


def test_reorder_needs_cow_until_each_beam_has_its_block():
    pool = BlockPool(20, BF16)
    mgr = KvManager(pool, 8, 3, 4)
    mgr.append([0, 1, 2], [5, 8, 3])
    assert not mgr.needs_cow([0, 1, 2])
    freed = mgr.reorder([0, 1, 2], [0, 0, 0])
    assert freed.size == 2 and mgr.needs_cow([0]) and mgr.needs_cow([2])
    plan = mgr.append([1], 1, cow=True)
    assert plan.cow_src.size == 1 and mgr.needs_cow([0]) and not mgr.needs_cow([1])
    plan = mgr.append([0], 1, cow=True)
    assert plan.cow_src.size == 1 and not mgr.needs_cow([0, 1, 2])  # the last holder writes in place
    assert mgr.append([2], 1).cow_src.size == 0
    mgr.append([0, 1, 2], 2, cow=True)  # to the block's end
    mgr.reorder([0, 1, 2], [1, 1, 1])
    assert not mgr.needs_cow([0, 1, 2])  # whole blocks are shared as they are
    mgr.append([0, 1, 2], 1)
    # A reordered beam that then drops a tail is followed as any compacted sequence is.
    mgr.reorder([0, 1], [0, 0])
    mgr.compact(1, list(range(8)))
    assert not mgr.needs_cow([1]) and mgr.needs_cow([0]) is False


def test_reorder_refusals_change_nothing():
    pool = BlockPool(20, BF16)
    mgr = KvManager(pool, 8, 4, 4)
    mgr.append([0, 1, 2], [5, 9, 3])
    before = [x.copy() for x in mgr.tables()]
    with pytest.raises(ValueError):
        mgr.reorder([0, 1], [0])
    for seqs, parents in (([0, 1], [0, 2]), ([0, 0], [0, 1]), ([0, 4], [0, 0]), ([-1], [0])):
        with pytest.raises(InvalidInput):
            mgr.reorder(seqs, parents)
    at, of, nev = np.array([0, 1], np.int32), np.array([0, 0], np.int32), C.c_int32(7)
    ev = np.zeros(1, np.int32)
    assert L.lib.it_kv_manager_reorder(mgr._h, at.ctypes.data, of.ctypes.data, 2, ev.ctypes.data, 1, C.byref(nev)) == L.INVALID_INPUT
    assert L.lib.it_kv_manager_reorder(None, at.ctypes.data, of.ctypes.data, 2, ev.ctypes.data, 1, C.byref(nev)) == L.INVALID_INPUT
    assert L.lib.it_kv_manager_reorder(mgr._h, None, of.ctypes.data, 2, ev.ctypes.data, 1, C.byref(nev)) == L.INVALID_INPUT
    for a, b in zip(before, mgr.tables()):
        assert np.array_equal(a, b)
    assert mgr.reorder([], []).size == 0 and mgr.reorder([0, 1, 3], [-1, 1, 2]).size == 0
    assert np.array_equal(before[0], mgr.tables()[0])
    freed = mgr.reorder([0, 1, 3], [2, 2, 0])  # an empty sequence may be continued, and continue
    assert freed.size == 2 and mgr.positions().tolist() == [0, 0, 3, 5]


def test_batcher_reorders_requests():
    pool = BlockPool(40, BF16)
    mgr = KvManager(pool, 8, 4, 8)
    b = ContinuousBatcher(4, mgr)
    for r in range(3):
        b.add_request(10 + r, [1, 2, 3, 4, 5, 6, 7, 8, 9, r], 20)
    b.schedule()
    b.plan_prefill([10, 11, 12])
    for r in range(3):
        b.requests[10 + r].generated_tokens += [100 + r, 200 + r]
    b.plan_decode()
    b.plan_decode()
    mgr.compact(b.seq_of[11], [0, 2, 4, 6, 8, 9, 10, 11])
    with pytest.raises(ValueError):
        b.reorder([10, 99], [0, 0])
    with pytest.raises(ValueError):
        b.reorder([10, 11], [0, 2])
    with pytest.raises(ValueError):
        b.reorder([10, 11], [0])
    freed = b.reorder([10, 11, 12], [1, 1, 0])
    assert freed.size > 0
    assert b.requests[10].generated_tokens == b.requests[11].generated_tokens == [101, 201]
    assert b.requests[12].generated_tokens == [100, 200] and b.requests[12].prompt_tokens[-1] == 0
    assert b.context(10) == b.context(11) == [1, 3, 5, 7, 9, 1, 101, 201]
    assert b.context(12) == [1, 2, 3, 4, 5, 6, 7, 8, 9, 0, 100, 200]
    b.requests[10].generated_tokens.append(5)  # lists of their own
    assert b.requests[11].generated_tokens == [101, 201]
    plan = b.plan_decode()  # copy-on-write by itself where beams continue one block
    assert len(set(plan.slots.tolist())) == 3
    b.preempt(10)
    b.schedule()
    assert b.plan_resume([10]).slots.size == len(b.context(10))
    b.preempt(12)  # what has to be prefilled again goes with what the cache holds
    b.schedule()
    assert b.needs_prefill == {12}
    b.reorder([10, 11, 12], [2, 1, 2])
    assert b.needs_prefill == {10, 12} and mgr.positions()[b.seq_of[10]] == 0
    b.reorder([10, 11, 12], [1, 1, 0])
    assert b.needs_prefill == {12} and mgr.positions()[b.seq_of[10]] > 0
    assert b.plan_resume([12]).slots.size == len(b.context(12))
    for r in (10, 11, 12):
        b.finish(r)
    assert pool.num_free() == 40


def test_entry_points_refuse_before_any_device():
    lib, h = L.lib, C.c_void_p()
    for dims, code in (((0, 64), L.INVALID_INPUT), ((512, 0), L.INVALID_INPUT), ((100, 64), L.INVALID_INPUT), ((512, 12), L.INVALID_INPUT),
                       ((1032, 64), L.INVALID_INPUT), ((512, 264), L.INVALID_INPUT)):
        assert lib.it_kv_cache_new_latent(0, 1, 8, 16, *dims, L.BF16, C.byref(h)) == code, dims
    assert lib.it_kv_cache_new_latent(0, 1, 8, 16, 512, 64, L.Q8_0, C.byref(h)) == L.NOT_IMPLEMENTED
    assert lib.it_kv_cache_new_latent(0, 1, 8, 12, 512, 64, L.BF16, C.byref(h)) == L.NOT_IMPLEMENTED
    assert lib.it_kv_cache_new_latent(0, 0, 8, 16, 512, 64, L.BF16, C.byref(h)) == L.INVALID_INPUT
    assert lib.it_kv_cache_wrap_latent(0, 1, None, 8, 16, 512, 64, L.BF16, C.byref(h)) == L.INVALID_INPUT
    assert lib.it_kv_cache_wrap_latent(0, 1, 8, 8, 16, 512, 64, L.BF16, C.byref(h)) == L.INVALID_INPUT
    assert lib.it_kv_cache_latent_dim(None) == 0
    assert L.call.it_latent_append(None, None, None, L.BF16, 0, None, 0, 1e-6, None, 0, 0, 0, None, 0, 0, 0, None, None, None, 1,
                                   None) == L.INVALID_INPUT
    assert L.call.it_latent_decode(None, None, None, L.BF16, 0, 0, 0, 0, 1, 1, None, 1, None, None, 1, 1, 0.1, None, 0, None, L.BF16,
                                   None) == L.INVALID_INPUT
    assert L.call.it_latent_decode_workspace(None, 1, 1, 1, 1) == 0
    prefill = [None, None, None, None, L.BF16, 192, 192, 128, 128, 128, 128, 64, 1, 128, 64, 128, None, None, 1, 4, 4, 4, 4, 0.1, 1, None,
               L.BF16, None]
    assert L.call.it_latent_prefill(*prefill) == L.INVALID_INPUT and b"NULL" in lib.it_last_error()
    for at, bad, code in ((4, L.Q8_0, L.NOT_IMPLEMENTED), (12, 0, L.INVALID_INPUT), (13, 100, L.INVALID_INPUT), (14, 4, L.INVALID_INPUT),
                          (15, 1032, L.INVALID_INPUT), (13, 1024, L.INVALID_INPUT), (23, float("inf"), L.INVALID_INPUT), (5, -1, L.INVALID_INPUT),
                          (18, -1, L.INVALID_INPUT), (26, L.F16, L.NOT_IMPLEMENTED)):
        args = list(prefill)
        args[at] = bad
        assert L.call.it_latent_prefill(*args) == code, (at, bad)
    select = [None, L.F32, 100, 2, 4, 100, None, 8, None, None, None, None, 0, None]
    assert L.call.it_beam_select(*select) == L.INVALID_INPUT and b"NULL" in lib.it_last_error()
    for at, bad, code in ((1, L.Q8_0, L.NOT_IMPLEMENTED), (2, 99, L.INVALID_INPUT), (3, -1, L.INVALID_INPUT), (4, 0, L.INVALID_INPUT),
                          (4, 65, L.INVALID_INPUT), (3, 1 << 20, L.INVALID_INPUT), (5, (1 << 18) + 1, L.INVALID_INPUT), (7, 65, L.INVALID_INPUT)):
        args = list(select)
        args[at] = bad
        assert L.call.it_beam_select(*args) == code, (at, bad)
    assert L.call.it_beam_select_workspace(2, 65, 100, 8) == 0 < L.call.it_beam_select_workspace(2, 4, 100, 8)
    reorder = [None, 64, 64, 1, 0, 2, 4, None, None]
    assert L.call.it_beam_reorder(*reorder) == L.INVALID_INPUT
    for at, bad in ((1, -1), (2, 63), (5, -1), (6, 65), (6, 0)):
        args = list(reorder)
        args[at] = bad
        assert L.call.it_beam_reorder(*args) == L.INVALID_INPUT, (at, bad)
    args = [None, 64, 64, 2, 511, 2, 4, None, None]  # arrays that lie in one another
    assert L.call.it_beam_reorder(*args) == L.INVALID_INPUT
    assert L.call.it_beam_reorder(None, 0, 0, 1, 0, 0, 4, None, None) == L.OK
    for op in (L.OP_LATENT_APPEND, L.OP_LATENT_DECODE, L.OP_LATENT_PREFILL, L.OP_BEAM_SELECT):
        assert [lib.it_supports(op, d) for d in (L.F32, L.F16, L.BF16, L.Q8_0)] == [1, 1, 1, 0]
    assert lib.it_supports(L.OP_BEAM_REORDER, L.F32) == 1
