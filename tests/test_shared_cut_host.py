"""Sequences that share a block and are cut to the same length inside it: one
step that appends to several of them needs copy-on-write, whichever way they
came to share it."""
import numpy as np
import pytest

from infer_train_amd import BF16, BlockPool, ContinuousBatcher, InvalidInput, KvManager

BS = 8


def sharing(how, n=2, at=13):
    """n sequences that hold the same blocks, each `at` tokens long."""
    pool = BlockPool(160, BF16)
    mgr = KvManager(pool, BS, n + 1, 8)
    if how == "reorder":
        mgr.append(list(range(n)), [at] + [at - 2] * (n - 1))
        mgr.reorder(list(range(n)), [0] * n)
    else:
        mgr.append([0], at)
        for s in range(1, n):
            mgr.fork(0, s)
    return pool, mgr


def cut(mgr, seqs, keep, together):
    if together:
        mgr.compact_many(seqs, [range(keep)] * len(seqs))
    else:
        for s in seqs:
            mgr.compact(s, range(keep))


@pytest.mark.parametrize("how", ["reorder", "fork"])
@pytest.mark.parametrize("together", [True, False])
@pytest.mark.parametrize("keep", [11, 9, 5])  # of the last block, and of one before it
@pytest.mark.parametrize("n", [2, 4])
def test_equal_cuts_are_appended_with_copy_on_write(how, together, keep, n):
    pool, mgr = sharing(how, n)
    seqs = list(range(n))
    cut(mgr, seqs, keep, together)
    assert mgr.needs_cow(seqs)
    before = [x.copy() for x in mgr.tables()], pool.num_free()
    with pytest.raises(InvalidInput, match="copy-on-write"):
        mgr.append(seqs, 1)
    assert all(np.array_equal(a, b) for a, b in zip(before[0], mgr.tables())) and pool.num_free() == before[1]
    plan = mgr.append(seqs, 1, cow=True)
    assert len(set(plan.slots.tolist())) == n and plan.cow_src.size == n - 1  # the last holder writes in place
    assert not mgr.needs_cow(seqs) and len(set(mgr.append(seqs, 3).slots.tolist())) == 3 * n


@pytest.mark.parametrize("how", ["reorder", "fork"])
def test_equal_cuts_appended_one_after_another(how):
    """Alone, the first writes where no other reads; the other then needs a copy."""
    pool, mgr = sharing(how)
    cut(mgr, [0, 1], 11, True)
    if not mgr.needs_cow([0]):
        first = mgr.append([0], 1).slots.tolist()
        assert mgr.needs_cow([1]) and not mgr.needs_cow([0])
        with pytest.raises(InvalidInput, match="copy-on-write"):
            mgr.append([0, 1], 1)
        second = mgr.append([1], 1, cow=True).slots.tolist()
    else:
        first, second = (mgr.append([s], 1, cow=True).slots.tolist() for s in (0, 1))
    assert first != second and not mgr.needs_cow([0, 1])


def test_a_cut_back_to_a_snapshot_beside_it_in_one_step():
    """A fork that stands where a sequence is cut back to reads nothing there: alone the sequence goes on in place, in one
    step with the fork it does not."""
    pool, mgr = sharing("fork", at=9)
    mgr.append([0], 4)
    mgr.compact(0, range(9))
    assert not mgr.needs_cow([0]) and mgr.needs_cow([0, 1]) and mgr.needs_cow([1, 0])
    with pytest.raises(InvalidInput, match="copy-on-write"):
        mgr.append([0, 1], 1)
    assert len(mgr.append([0, 1], [1, 0]).slots) == 1  # the other is listed without a token


def test_unequal_cuts():
    pool, mgr = sharing("reorder")
    mgr.compact_many([0, 1], [range(9), range(11)])
    assert mgr.needs_cow([0]) and mgr.needs_cow([0, 1])
    plan = mgr.append([1, 0], 1, cow=True)
    assert len({int(s) // BS for s in plan.slots}) == 2


@pytest.mark.parametrize("together", [True, False])
def test_a_search_that_drops_its_drafts(together):
    """The batcher decides by itself: reorder, drafts rejected by all beams, the next token."""
    pool = BlockPool(40, BF16)
    mgr = KvManager(pool, BS, 2, 8)
    b = ContinuousBatcher(2, mgr)
    for r in (1, 2):
        b.add_request(r, list(range(13)), 20)
    b.schedule()
    b.plan_prefill([1, 2])
    b.reorder([1, 2], [0, 0])
    cut(mgr, [b.seq_of[1], b.seq_of[2]], 11, together)
    plan = b.plan_decode()
    assert len(set(plan.slots.tolist())) == 2 and plan.cow_src.size == 1


@pytest.mark.parametrize("seed", range(8))
def test_random_searches_with_cuts(seed):
    """Appends with copy-on-write only where it is asked for, reorderings, cuts and compactions of any of the sequences:
    each one's tokens are found through its table."""
    for sub in range(25):
        rng = np.random.default_rng([seed, sub])
        bs, n, tok = int(rng.choice([4, 8])), int(rng.integers(2, 6)), 0
        pool = BlockPool(400, BF16)
        mgr = KvManager(pool, bs, n, 32)
        pages, model = np.full((400, bs), -1, np.int64), {s: [] for s in range(n)}
        for _ in range(60):
            seqs = [int(x) for x in rng.permutation(n)[:rng.integers(1, n + 1)]]
            op = rng.integers(0, 6)
            if op < 3:
                counts = [int(x) for x in rng.integers(0, 4, len(seqs))]
                if max(len(model[s]) for s in seqs) + 4 > 32 * bs:
                    continue
                plan = mgr.append(seqs, counts, cow=mgr.needs_cow(seqs))
                for a, b in zip(plan.cow_src, plan.cow_dst):
                    pages[b] = pages[a]
                for slot, s in zip(plan.slots, plan.token_seq):
                    model[int(s)] = model[int(s)] + [tok]
                    pages[slot // bs, slot % bs] = tok
                    tok += 1
            elif op == 3:
                parents = [int(x) for x in rng.integers(-1, len(seqs), len(seqs))]
                pages[mgr.reorder(seqs, parents)] = -1
                was = {s: model[s] for s in seqs}
                model.update({s: was[seqs[p]] for s, p in zip(seqs, parents) if p >= 0})
            else:
                most = int(rng.integers(0, 40))
                keeps = [list(range(min(len(model[s]), most))) if rng.random() < 0.75 else
                         sorted(rng.permutation(len(model[s]))[:most].tolist()) for s in seqs]
                plan = mgr.compact_many(seqs, keeps)
                moved = pages[plan.src // bs, plan.src % bs].copy()
                pages[plan.dst // bs, plan.dst % bs] = moved
                pages[plan.evicted] = -1
                model.update({s: [model[s][j] for j in k] for s, k in zip(seqs, keeps)})
            tables, ctx, _ = mgr.tables()
            for s, tokens in model.items():
                p = np.arange(len(tokens))
                assert ctx[s] == len(tokens) and pages[tables[s, p // bs], p % bs].tolist() == tokens, (sub, s)
