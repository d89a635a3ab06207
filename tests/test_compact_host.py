"""CPU checks of compaction beside forks, other compactions and the batcher: no
row that somebody still reads is planned to be overwritten."""

import numpy as np
import pytest

from infer_train_amd import BF16, BlockPool, ContinuousBatcher, InvalidInput, KvManager
from infer_train_amd import _lib as L


def slots_of(mgr, seq, upto):
    """Slots of a sequence's positions 0 .. upto - 1."""
    row, bs = mgr.tables()[0][seq], mgr.block_size
    return [int(row[p // bs]) * bs + p % bs for p in range(upto)]


# ---- a tail dropped out of a block that a fork holds --------------------------
def forked(tail, ctx=15, bs=4):
    """Sequence 0 of a batcher with `ctx` tokens, forked to sequence 3, compacted to its first `tail`."""
    pool = BlockPool(24, BF16)
    mgr = KvManager(pool, bs, 4, 16)
    b = ContinuousBatcher(2, mgr)
    b.add_request(0, list(range(ctx)), 9)
    b.schedule()
    b.plan_prefill([0])
    seq = b.seq_of[0]
    mgr.fork(seq, 3)
    plan = mgr.compact(seq, list(range(tail)))
    assert plan.src.size == 0 == plan.evicted.size
    return b, mgr, pool, seq


@pytest.mark.parametrize("bs,ctx,tail", ((4, 15, 13), (4, 15, 10), (4, 16, 15), (16, 15, 1), (2, 9, 3), (4, 15, 12), (1, 7, 3)))
def test_append_after_a_dropped_tail_leaves_the_fork_alone(bs, ctx, tail):
    """Decode steps after the drop: no slot that the fork reads is written, and the sequence's own rows are found, in the
    fork's block or in its copy."""
    b, mgr, pool, seq = forked(tail, ctx, bs)
    fork, rows = slots_of(mgr, 3, ctx), slots_of(mgr, seq, tail)
    plan = b.plan_decode()
    assert not set(plan.slots.tolist()) & set(fork)
    if tail % bs:
        assert plan.cow_src.tolist() == [rows[-1] // bs] and plan.cow_dst.tolist() == [int(plan.slots[0]) // bs]
        copied = {s: int(plan.cow_dst[0]) * bs + s % bs for s in rows if s // bs == plan.cow_src[0]}
        assert slots_of(mgr, seq, tail) == [copied.get(s, s) for s in rows]
    else:
        assert plan.cow_src.size == 0
    assert slots_of(mgr, 3, ctx) == fork
    for _ in range(3):
        plan = b.plan_decode()
        assert plan.cow_src.size == 0 and not set(plan.slots.tolist()) & set(fork)


def test_append_without_copy_on_write_is_refused_before_any_change():
    b, mgr, pool, seq = forked(13)
    before = mgr.tables()[0].copy(), mgr.positions().copy(), pool.num_free()
    for seqs, n in (([seq], 1), ([1, seq], [2, 3])):
        with pytest.raises(InvalidInput):
            mgr.append(seqs, n)
        assert np.array_equal(mgr.tables()[0], before[0]) and np.array_equal(mgr.positions(), before[1]) and pool.num_free() == before[2]
    assert mgr.append([seq], 0).slots.size == 0
    assert mgr.append([3], 1).slots.tolist() == [slots_of(mgr, 3, 16)[-1]]  # the fork goes on in its block
    plan = mgr.append([seq], 1, cow=True)
    assert plan.cow_src.size == 1


def test_a_fork_that_drops_its_tail_leaves_its_parent_alone():
    pool = BlockPool(24, BF16)
    mgr = KvManager(pool, 4, 4, 16)
    mgr.append([0], 15)
    mgr.fork(0, 1)
    mgr.compact(1, range(13))
    mgr.fork(1, 2)  # stands where sequence 1 stands
    for s in (1, 2):
        assert mgr.needs_cow([s]) and mgr.needs_cow([0, s]) and not mgr.needs_cow([0, 3])
        with pytest.raises(InvalidInput):
            mgr.append([s], 1)
    parent = set(slots_of(mgr, 0, 15))
    for s in (1, 2):
        plan = mgr.append([s], 1, cow=True)
        assert plan.cow_src.size == 1 and not set(plan.slots.tolist()) & parent
    assert not mgr.needs_cow([0, 1, 2])


def test_append_in_place_where_nobody_reads_on():
    """A fork that ends before the drop (a snapshot of a prefix), or is gone, needs no copy: drafts are dropped and appended
    without one, as before the fork."""
    pool = BlockPool(24, BF16)
    mgr = KvManager(pool, 16, 4, 16)
    mgr.append([0], 9)
    mgr.fork(0, 1)
    mgr.append([0], 4)  # drafts
    assert mgr.compact(0, range(11)).src.size == 0
    assert not mgr.needs_cow([0])
    assert mgr.append([0], 2).slots.tolist() == slots_of(mgr, 0, 13)[11:]
    mgr.compact(0, range(8))  # now below the snapshot
    assert mgr.needs_cow([0])
    mgr.release(1)
    assert not mgr.needs_cow([0])
    assert mgr.append([0], 1).slots.tolist() == slots_of(mgr, 0, 9)[8:]
    # A holder outside the manager: nothing is known of what it reads.
    block = int(mgr.tables()[0][0, 0])
    pool.share(block)
    mgr.compact(0, range(5))
    assert mgr.needs_cow([0])
    with pytest.raises(InvalidInput):
        mgr.append([0], 1)
    mgr.release(0)
    assert not mgr.needs_cow([0, 1, 2, 3])
    for bad in ([4], [-1], [0, 9]):
        with pytest.raises(ValueError):
            mgr.needs_cow(bad)
    arr = np.zeros(1, np.int32)
    assert L.lib.it_kv_manager_needs_cow(None, arr.ctypes.data, 1) == -1 == L.lib.it_kv_manager_needs_cow(mgr._h, None, 1)
    assert L.lib.it_kv_manager_needs_cow(mgr._h, None, 0) == 0
