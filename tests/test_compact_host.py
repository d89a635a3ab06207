"""CPU checks of compaction beside forks, other compactions and the batcher: no
row that somebody still reads is planned to be overwritten."""

import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from infer_train_amd import BF16, BlockPool, ContinuousBatcher, InvalidInput, KvManager, NotImplementedOp
from infer_train_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


# ---- several sequences in one plan ---------------------------------------------
def test_a_plan_of_several_sequences_writes_nothing_that_it_reads():
    """Planned one after another, the second's fresh blocks are those the first gave back, which its move still reads and
    its eviction clears; planned together, destinations are apart from every source and returned block."""
    keep = range(0, 16, 2)
    pool = BlockPool(16, BF16)
    mgr = KvManager(pool, 4, 4, 16)
    mgr.append([0, 1], 16)
    plan = mgr.compact_many([0, 1], [keep, keep])
    blocks = lambda x: set((x // 4).tolist())  # noqa: E731
    assert not blocks(plan.dst) & (blocks(plan.src) | set(plan.evicted.tolist()))
    assert len(set(plan.dst.tolist())) == 16 == len(set(plan.src.tolist()))
    assert plan.token_seq.tolist() == [0] * 8 + [1] * 8 and plan.token_pos.tolist() == list(range(8)) * 2
    assert plan.delta.tolist() == [i - k for i, k in enumerate(keep)] * 2
    assert mgr.positions().tolist() == [8, 8, 0, 0] and pool.num_free() == 12 and len(plan.evicted) == 8


@pytest.mark.parametrize("bs,seed", ((1, 0), (4, 1), (16, 2), (16, 3)))
def test_compact_many_against_lists(bs, seed):
    """Random appends, forks, releases and compactions of several sequences, all of a plan's rows read before the first is
    written and its returned blocks cleared after: every kept token is where the table says."""
    rng = np.random.default_rng(seed)
    cap, n_seqs = 900 // bs + 16, 5
    pool = BlockPool(cap, BF16)
    mgr, cells, seqs, ident = KvManager(pool, bs, n_seqs, cap), {}, [[] for _ in range(5)], 0
    together = 0
    for _ in range(250):
        op, s = rng.integers(0, 8), int(rng.integers(0, n_seqs))
        if op <= 3:
            n = int(rng.integers(1, 40))
            if pool.num_free() < n // bs + 2:
                continue
            plan = mgr.append([s], n, cow=True)
            for a, b in zip(plan.cow_src, plan.cow_dst):
                for j in range(bs):
                    cells[int(b) * bs + j] = cells.get(int(a) * bs + j)
            for slot in plan.slots:
                cells[int(slot)] = ident
                seqs[s].append(ident)
                ident += 1
        elif op == 4:
            d = int(rng.integers(0, n_seqs))
            if d != s and not seqs[d]:
                mgr.fork(s, d)
                seqs[d] = list(seqs[s])
        elif op == 5 and rng.random() < 0.3:
            mgr.release(s)
            seqs[s] = []
        else:
            some = rng.permutation(n_seqs)[:int(rng.integers(0, n_seqs + 1))].tolist()
            keeps = [np.flatnonzero(rng.random(len(seqs[i])) < rng.choice([0.0, 0.3, 0.9, 1.0])) if rng.random() < 0.7
                     else np.arange(rng.integers(0, len(seqs[i]) + 1)) for i in some]
            if pool.num_free() < sum(-(-len(k) // bs) for k in keeps):
                continue
            held = {b for b in mgr.tables()[0].reshape(-1).tolist() if b >= 0}
            plan = mgr.compact_many(some, keeps)
            together += plan.src.size > 0 and len(some) > 1
            assert not set((plan.dst // bs).tolist()) & held and not set((plan.dst // bs).tolist()) & set(plan.evicted.tolist())
            assert len(set(plan.dst.tolist())) == plan.dst.size
            for b, x in [(int(b), cells[int(a)]) for a, b in zip(plan.src, plan.dst)]:
                cells[b] = x
            for b in plan.evicted.tolist():
                assert pool.ref_count(b) == 0 and b in held
                for j in range(bs):
                    cells[b * bs + j] = None
            for i, k in zip(some, keeps):
                seqs[i] = [seqs[i][t] for t in k]
        tables, ctx, _ = mgr.tables()
        users = {}
        for i, toks in enumerate(seqs):
            assert ctx[i] == len(toks)
            assert [cells[x] for x in slots_of(mgr, i, len(toks))] == toks, i
            for b in tables[i][tables[i] >= 0].tolist():
                users[b] = users.get(b, 0) + 1
        assert all(pool.ref_count(b) == users.get(b, 0) for b in range(cap)) and pool.num_free() == cap - len(users)
    assert together > 5


def test_forks_compacted_together_return_their_blocks():
    pool = BlockPool(12, BF16)
    mgr = KvManager(pool, 4, 3, 12)
    mgr.append([0], 12)
    mgr.fork(0, 1)
    shared = [int(b) for b in mgr.tables()[0][0][:3]]
    plan = mgr.compact_many([0, 1], [[1, 5], []])
    assert sorted(plan.evicted.tolist()) == sorted(shared) and plan.src.tolist() == [shared[0] * 4 + 1, shared[1] * 4 + 1]
    assert pool.num_free() == 11 and mgr.positions().tolist() == [2, 0, 0]


def test_compact_many_refusals_change_nothing():
    pool = BlockPool(9, BF16)
    mgr = KvManager(pool, 4, 3, 9)
    mgr.append([0, 1], [10, 12])  # six blocks, three free
    before = mgr.tables()[0].copy(), mgr.positions().copy(), pool.num_free()

    def unchanged():
        return np.array_equal(mgr.tables()[0], before[0]) and np.array_equal(mgr.positions(), before[1]) and pool.num_free() == before[2]

    for seqs, keeps in (([0, 0], [[1], [2]]), ([0, 3], [[1], []]), ([0, -1], [[1], []]), ([0, 1], [[1], [12]]), ([0, 1], [[1], [3, 3]]),
                        ([0, 1], [[1], [3, 2]]), ([0, 2], [[1], [0]]), ([0, 1], [range(1, 9), range(1, 9)])):  # the last: four fresh
        with pytest.raises(InvalidInput):
            mgr.compact_many(seqs, keeps)
        assert unchanged(), (seqs, keeps)
    for seqs, keeps, error in (([0, 1], [[1]], ValueError), ([0], [[-1]], ValueError), ([0], [[2 ** 31]], ValueError),
                               ([0], [[0.5]], TypeError), ([0], [np.ones(10, bool)], TypeError)):
        with pytest.raises(error):
            mgr.compact_many(seqs, keeps)
        assert unchanged()
    keep, cu, seqs = np.array([1, 2, 5, 6], np.int32), np.array([0, 2, 4], np.int32), np.array([0, 1], np.int32)
    down, late = np.array([0, 3, 2], np.int32), np.array([1, 2, 4], np.int32)
    src, dst, ev, n = np.empty(4, np.int64), np.empty(4, np.int64), np.empty(6, np.int32), C.c_int32()
    call = lambda **kw: L.lib.it_kv_manager_compact_many(*{**dict(  # noqa: E731
        m=mgr._h, seqs=seqs.ctypes.data, ns=2, keep=keep.ctypes.data, cu=cu.ctypes.data, src=src.ctypes.data, dst=dst.ctypes.data,
        delta=None, of=None, pos=None, cap=4, nm=C.byref(n), ev=ev.ctypes.data, evc=6, ne=C.byref(n)), **kw}.values())
    for kw in (dict(m=None), dict(seqs=None), dict(keep=None), dict(cu=None), dict(src=None), dict(dst=None), dict(cap=3), dict(nm=None),
               dict(ev=None), dict(evc=5), dict(ne=None), dict(ns=-1), dict(cu=down.ctypes.data), dict(cu=late.ctypes.data)):
        assert call(**kw) == L.INVALID_INPUT and unchanged(), kw
    assert call(ns=0, seqs=None, cu=None, keep=None, ev=None, evc=0) == L.OK and unchanged()
    assert mgr.compact_many([], []).src.size == 0 and unchanged()
    assert call() == L.OK and mgr.positions().tolist() == [2, 2, 0]  # token_seq, delta and pos are optional
    window = KvManager(BlockPool(8, BF16), 4, 2, 8, window=8)
    window.append([0], 6)
    with pytest.raises(NotImplementedOp):
        window.compact_many([0], [[0, 1]])


_DRIVER = r"""
#include <vector>
#include "it_kv.h"
int main() {
  unsigned r = 1;
  const auto rnd = [&](int n) { return int((r = r * 1664525u + 1013904223u) >> 8) % n; };
  it_block_pool* pool; it_kv_manager* m;
  if (it_block_pool_new(64, 30, &pool) || it_kv_manager_new(pool, 4, 4, 40, 0, &m)) return 1;
  std::vector<int32_t> ctx(4);
  for (int step = 0; step < 20000; ++step) {
    const int32_t s = rnd(4), n = rnd(9);
    it_kv_manager_tables(m, nullptr, 0, ctx.data(), nullptr);
    if (rnd(2) && it_block_pool_num_free(pool) > 4 && ctx[s] < 120) {
      std::vector<int64_t> slots(n + 1); std::vector<int32_t> ev(64), cs(n + 1), cd(n + 1); int32_t ne, nc;
      if (it_kv_manager_append_cow(m, &s, &n, 1, slots.data(), ev.data(), 64, &ne, cs.data(), cd.data(), n + 1, &nc)) return 2;
      if (it_kv_manager_needs_cow(m, &s, 1) < 0) return 5;
    } else {
      std::vector<int32_t> keep, cu{0}, seqs;
      for (int32_t i = s; i < 4 && i < s + 1 + n % 3; ++i) {
        const int drop = rnd(4), tail = rnd(2) ? rnd(ctx[i] + 1) : ctx[i];
        for (int32_t p = 0; p < tail; ++p) if (rnd(4) >= drop) keep.push_back(p);
        seqs.push_back(i); cu.push_back(int32_t(keep.size()));
      }
      const size_t k = keep.size();
      std::vector<int64_t> src(k), dst(k); std::vector<int32_t> d(k), of(k), pos(k), ev(64); int32_t nm, ne;
      const int rc = it_kv_manager_compact_many(m, seqs.data(), int32_t(seqs.size()), keep.data(), cu.data(), src.data(), dst.data(),
                                                d.data(), of.data(), pos.data(), int32_t(k), &nm, ev.data(), 64, &ne);
      if (rc && it_block_pool_num_free(pool) >= int64_t(k + 3 * seqs.size()) / 4) return 3;
      const int32_t t = (s + 1) % 4;
      if (!rc && rnd(3) == 0) { int32_t n2; if (it_kv_manager_release_seq(m, t, ev.data(), 64, &n2) || it_kv_manager_fork(m, s, t)) return 4; }
    }
  }
  it_kv_manager_destroy(m); it_block_pool_destroy(pool);
  return 0;
}
"""


def test_compact_many_under_sanitizers(tmp_path):
    src, exe = tmp_path / "compact.cpp", str(tmp_path / "compact")
    src.write_text(_DRIVER)
    host = os.path.join(ROOT, "infer_train_amd", "csrc", "it_host.cpp")
    b = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I",
                        os.path.join(ROOT, "include"), "-I", os.path.dirname(host), str(src), host, "-o", exe],
                       capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stderr[-2000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])


def test_a_seeded_row_that_names_a_block_twice_returns_it_once():
    pool = BlockPool(6, BF16)
    mgr = KvManager(pool, 4, 2, 6)
    block = pool.allocate()
    mgr.seed_seq(0, 8, 0, [block, block])
    plan = mgr.compact(0, [])
    assert plan.evicted.tolist() == [block] and pool.num_free() == 6 and pool.ref_count(block) == 0


# ---- a compacted request that is preempted --------------------------------------
def test_a_compacted_request_resumes_with_what_it_kept():
    """Twice compacted, decoded on in between, preempted and resumed: the tokens prefilled again are those that the cache held,
    in its order, and the one drawn last; a request beside it is prefilled whole."""
    pool = BlockPool(64, BF16)
    mgr = KvManager(pool, 4, 4, 32)
    b = ContinuousBatcher(2, mgr)
    for rid, n in ((5, 20), (6, 9)):
        b.add_request(rid, [100 * rid + i for i in range(n)], 50)
    b.schedule()
    b.plan_prefill([5, 6])
    cache, new = {r: list(b.requests[r].prompt_tokens) for r in (5, 6)}, {5: 9000, 6: 9500}

    def draw():
        for r in (5, 6):
            b.requests[r].generated_tokens.append(new[r])
            new[r] += 1

    def step():
        b.plan_decode()
        for r in (5, 6):
            cache[r].append(b.requests[r].generated_tokens[-1])
        draw()

    draw()
    for _ in range(3):
        step()
    for keep in ([0, 1, 2, 3] + list(range(10, 23)), [0, 2, 5, 6, 7, 8, 12, 13]):
        mgr.compact(b.seq_of[5], keep)
        cache[5] = [cache[5][i] for i in keep]
        step()
        step()
        assert len(cache[5]) == mgr.positions()[b.seq_of[5]]
        for r in (5, 6):
            assert b.context(r) == cache[r] + b.requests[r].generated_tokens[-1:]
    b.preempt(5)
    b.schedule()
    want = cache[5] + b.requests[5].generated_tokens[-1:]
    plan = b.plan_resume([5])
    assert plan.slots.size == len(want) == len(b.context(5)) and b.context(5) == want
    seq = b.seq_of[5]
    mgr.compact_many([b.seq_of[6], seq], [list(range(3)), list(range(1, 6))])
    assert b.context(5) == want[1:6] and b.context(6) == b.requests[6].prompt_tokens[:3] + b.requests[6].generated_tokens[-1:]
    b.finish(5)
    b.add_request(5, [1, 2], 4)
    assert b.context(5) == [1, 2]


@pytest.mark.parametrize("appended", (False, True))
def test_rejected_drafts_leave_the_context_whole(appended):
    """Drafts are in the cache before they are accepted; dropping the rejected ones takes nothing from the request, whether
    the accepted ones are already among its tokens or join them afterwards."""
    mgr = KvManager(BlockPool(32, BF16), 4, 2, 32)
    b = ContinuousBatcher(1, mgr)
    b.add_request(0, list(range(10)), 50)
    b.schedule()
    b.plan_prefill([0])
    seq, gen = b.seq_of[0], b.requests[0].generated_tokens
    for base in (0, 1):  # the second time behind a compaction of the middle
        gen.append(50)
        held = int(mgr.positions()[seq])
        mgr.append([seq], 5)  # 50 and four drafts, two of which are accepted
        if appended:
            gen.extend([51, 52])
        mgr.compact(seq, range(held + 3))
        if not appended:
            gen.extend([51, 52])
        whole = (list(range(10)) if base == 0 else [0, 1, 7, 8, 9, 50, 51, 52])
        assert b.context(0) == whole + [50, 51, 52] and mgr.positions()[seq] == len(b.context(0))
        mgr.compact(seq, [0, 1] + list(range(7, held + 3)))
        assert b.context(0) == [0, 1] + (whole + [50, 51, 52])[7:]


def test_compaction_of_sequences_that_are_no_request():
    mgr = KvManager(BlockPool(32, BF16), 4, 4, 32)
    gone = ContinuousBatcher(1, mgr)
    del gone
    b = ContinuousBatcher(1, mgr)
    b.add_request(0, [1, 2, 3, 4, 5, 6], 50)
    b.schedule()
    b.plan_prefill([0])
    mgr.fork(b.seq_of[0], 3)
    mgr.compact(3, [1, 4])
    assert b.context(0) == [1, 2, 3, 4, 5, 6]
    mgr.compact(b.seq_of[0], [])
    assert b.context(0) == []


# ---- drawing for some of the running requests ------------------------------------
def test_sample_takes_running_requests_alone(monkeypatch):
    """The rows' settings and the tokens go to the requests listed; the draw itself is stubbed (it needs a device)."""
    import torch
    from infer_train_amd import SamplingParams, sampling

    b = ContinuousBatcher(3)
    for rid in (4, 5, 6, 7):
        b.add_request(rid, [1], 9, SamplingParams(temperature=0.25 * rid, top_k=rid))
    assert b.schedule() == [4, 5, 6]
    seen = {}

    def draw(logits, u, **kw):
        seen.update({k: v.tolist() for k, v in kw.items()})
        return logits.argmax(1).int(), None

    monkeypatch.setattr(sampling, "sample", draw)
    z, u = torch.eye(3), torch.zeros(3)
    assert b.sample(z[[2, 0]], u[:2], [6, 4]) == [2, 0]
    assert seen["temperature"] == [1.5, 1.0] and seen["top_k"] == [6, 4]
    assert [b.requests[r].generated_tokens for r in (4, 5, 6)] == [[0], [], [2]]
    assert b.sample(z, u) == [0, 1, 2] and seen["top_k"] == [4, 5, 6]
    assert b.sample(z[:0], u[:0], []) == []
    for ids, rows in (([7], 1), ([99], 1), ([4, 4], 2), ([4, 5], 1), ([4], 2), ([], 1)):
        with pytest.raises(ValueError):
            b.sample(z[:rows], u[:rows], ids)
    assert [len(b.requests[r].generated_tokens) for r in (4, 5, 6, 7)] == [2, 1, 2, 0]
