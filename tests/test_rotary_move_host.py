"""CPU checks of the rotary, move and sampling entry points: frequencies, the
manager's compaction against a list model, and every refusal that is made
before the device is touched."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

from infer_train_amd import BF16, BlockPool, InvalidInput, KvManager, NotImplementedOp
from infer_train_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOME = 1 << 20  # an aligned address that no refused call reads


def desc(n_dims=64, layout=L.ROTARY_HALF, scaling=L.ROTARY_SCALE_NONE, original_ctx=0, base=10000.0, factor=1.0, low=1.0,
         high=32.0, magnitude=1.0, inv_freq=None):
    return L.RotaryDesc(n_dims, layout, scaling, original_ctx, base, factor, low, high, magnitude, inv_freq)


def frequencies(d):
    out = np.empty(d.n_dims // 2)
    L.check(L.lib.it_rotary_frequencies(C.byref(d), out.ctypes.data))
    return out


@pytest.mark.parametrize("n_dims", (2, 32, 128, 1024))
def test_frequencies(n_dims):
    p = np.arange(n_dims // 2)
    plain = 10000.0 ** (-2.0 * p / n_dims)
    # pow and one more product: a few units of 2^-53 each.
    close = lambda a, b: np.testing.assert_allclose(a, b, rtol=2.0 ** -48)  # noqa: E731
    close(frequencies(desc(n_dims)), plain)
    close(frequencies(desc(n_dims, scaling=L.ROTARY_SCALE_LINEAR, factor=8.0)), plain / 8)
    if n_dims > 2:
        got = frequencies(desc(n_dims, scaling=L.ROTARY_SCALE_BASE, factor=8.0))
        close(got[0], 1.0)
        close(got[-1], plain[-1] / 8)  # the slowest pair's wavelength is stretched by the factor
    parts = frequencies(desc(n_dims, scaling=L.ROTARY_SCALE_PARTS, factor=8.0, original_ctx=8192, low=1.0, high=32.0))
    for f, g in zip(plain, parts):
        turns = 8192 * f / (2 * math.pi)
        want = f if turns >= 32 else f / 8 if turns <= 1 else f * ((turns - 1) / 31) + f / 8 * (1 - (turns - 1) / 31)
        assert abs(g - want) <= 2.0 ** -48 * f
    own = np.linspace(0.5, 0.25, n_dims // 2)
    assert np.array_equal(frequencies(desc(n_dims, inv_freq=own.ctypes.data)), own)


def test_rotary_refusals():
    h, out = C.c_void_p(), np.empty(512)
    bad = [desc(0), desc(3), desc(-2), desc(1026), desc(base=0.0), desc(base=-1.0), desc(base=math.nan), desc(base=math.inf),
           desc(scaling=L.ROTARY_SCALE_LINEAR, factor=0.0), desc(scaling=L.ROTARY_SCALE_BASE, factor=math.inf),
           desc(scaling=L.ROTARY_SCALE_PARTS, factor=2.0), desc(scaling=L.ROTARY_SCALE_PARTS, factor=2.0, original_ctx=64, low=4.0, high=4.0),
           desc(scaling=L.ROTARY_SCALE_PARTS, factor=2.0, original_ctx=64, low=-1.0),
           desc(inv_freq=np.full(32, np.nan).ctypes.data), desc(inv_freq=np.full(32, 2.0 ** 21).ctypes.data)]
    for d in bad:
        assert L.lib.it_rotary_frequencies(C.byref(d), out.ctypes.data) == L.INVALID_INPUT, d.n_dims
        assert L.lib.it_rotary_new(0, C.byref(d), C.byref(h)) == L.INVALID_INPUT and not h.value
    for d in (desc(magnitude=0.0), desc(magnitude=-1.0), desc(magnitude=math.nan), desc(magnitude=1e60)):
        assert L.lib.it_rotary_new(0, C.byref(d), C.byref(h)) == L.INVALID_INPUT and not h.value
    for d in (desc(scaling=4), desc(scaling=-1)):
        assert L.lib.it_rotary_frequencies(C.byref(d), out.ctypes.data) == L.NOT_IMPLEMENTED
    assert L.lib.it_rotary_new(0, C.byref(desc(layout=2)), C.byref(h)) == L.NOT_IMPLEMENTED
    assert L.lib.it_rotary_new(0, None, C.byref(h)) == L.INVALID_INPUT
    assert L.lib.it_rotary_new(0, C.byref(desc()), None) == L.INVALID_INPUT
    assert L.lib.it_rotary_destroy(None) == L.OK
    assert L.lib.it_rotary_apply(None, SOME, L.F32, 64, SOME, 1, 1, 64, 0, SOME, 64, None) == L.INVALID_INPUT
    assert L.lib.it_kv_append_rotary(None, None, None, SOME, SOME, L.F32, 0, 64, 64, 0, SOME, SOME, 1, None, 0, None) == L.INVALID_INPUT
    assert L.lib.it_kv_move(None, SOME, SOME, 1, None, None, None) == L.INVALID_INPUT


def test_supports():
    floats, quant = (L.F32, L.F16, L.BF16), (L.Q8_0, L.Q4_0, L.Q4_1, L.Q5_0, L.Q5_1)
    for op in (L.OP_KV_APPEND_ROTARY, L.OP_KV_MOVE):
        assert all(L.lib.it_supports(op, dt) == 1 for dt in floats + quant) and L.lib.it_supports(op, 9) == 0
    for op in (L.OP_ROTARY, L.OP_SAMPLE):
        assert all(L.lib.it_supports(op, dt) == 1 for dt in floats) and not any(L.lib.it_supports(op, dt) for dt in quant)


def test_sample_refusals():
    need = L.lib.it_sample_workspace(2, 40000)
    assert need > 0 and L.lib.it_sample_workspace(0, 40000) == 0 == L.lib.it_sample_workspace(2, 32768)
    ok = dict(logits=SOME, dtype=L.F32, stride=40000, rows=2, vocab=40000, u=SOME, temps=None, ks=None, ps=None, ms=None, temp=1.0,
              k=0, p=1.0, m=0.0, tokens=SOME, probs=None, ws=SOME, ws_bytes=need, stream=None)
    call = lambda **kw: L.lib.it_sample(*{**ok, **kw}.values())  # noqa: E731
    for kw in (dict(rows=-1), dict(rows=65536), dict(vocab=0), dict(vocab=-5), dict(stride=39999), dict(temp=-1.0), dict(temp=math.nan),
               dict(temp=math.inf), dict(p=math.nan), dict(m=1.5), dict(m=math.nan), dict(logits=None), dict(u=None),
               dict(tokens=None), dict(logits=SOME + 2), dict(ws=None), dict(ws_bytes=need - 1), dict(ws=SOME + 16)):
        assert call(**kw) == L.INVALID_INPUT, kw
    for kw in (dict(dtype=L.Q8_0), dict(vocab=262145, stride=262145)):
        assert call(**kw) == L.NOT_IMPLEMENTED, kw
    assert call(rows=0, logits=None, ws=None) == L.OK


# ---- compaction -------------------------------------------------------------
class Model:
    """Blocks and token identities of sequences as plain lists; `cells` maps a slot to what is stored there."""

    def __init__(self, cap, bs):
        self.bs, self.cells = bs, {}
        self.seqs = {}

    def check(self, mgr, pool, n_seqs):
        tables, ctx, _ = mgr.tables()
        held = {}
        for s in range(n_seqs):
            toks = self.seqs.get(s, [])
            assert ctx[s] == len(toks)
            for i, tok in enumerate(toks):
                b = tables[s, i // self.bs]
                assert b >= 0 and self.cells[int(b) * self.bs + i % self.bs] == tok, (s, i)
            blocks = [int(b) for b in tables[s] if b >= 0]
            assert len(blocks) == -(-len(toks) // self.bs)
            for b in blocks:
                held[b] = held.get(b, 0) + 1
        for b in range(pool.capacity()):
            assert pool.ref_count(b) == held.get(b, 0)
        assert pool.num_free() == pool.capacity() - len(held)


@pytest.mark.parametrize("bs,seed", ((1, 0), (4, 1), (16, 2), (16, 3), (32, 4)))
def test_compact_against_lists(bs, seed):
    """Random appends, forks, compactions and releases: every kept token is found where the table says, block counts and
    references agree, moves go to blocks that nothing else holds, and what returns to the pool is listed."""
    rng = np.random.default_rng(seed)
    cap, n_seqs = 600 // bs + 12, 4
    pool = BlockPool(cap, BF16)
    mgr, m = KvManager(pool, bs, n_seqs, cap), Model(cap, bs)
    ident = 0
    for _ in range(300):
        op, s = rng.integers(0, 8), int(rng.integers(0, n_seqs))
        toks = m.seqs.setdefault(s, [])
        if op <= 3:
            n = int(rng.integers(1, 40))
            if pool.num_free() < n // bs + 2:
                continue
            plan = mgr.append([s], n, cow=True)
            for a, b in zip(plan.cow_src, plan.cow_dst):
                for j in range(bs):
                    m.cells[int(b) * bs + j] = m.cells.get(int(a) * bs + j)
            for slot in plan.slots:
                m.cells[int(slot)] = ident
                toks.append(ident)
                ident += 1
        elif op == 4:
            d = int(rng.integers(0, n_seqs))
            if d == s or m.seqs.get(d):
                continue
            mgr.fork(s, d)
            m.seqs[d] = list(toks)
        elif op == 5 and rng.random() < 0.3:
            mgr.release(s)
            m.seqs[s] = []
        else:
            n = len(toks)
            kind = rng.integers(0, 4)
            keep = (np.arange(int(rng.integers(0, n + 1))) if kind == 0 else np.flatnonzero(rng.random(n) < rng.random())
                    if kind == 1 else np.concatenate([np.arange(min(5, n)), np.arange(min(n, max(5, n // 2)), n)]) if kind == 2
                    else np.arange(n))
            if pool.num_free() < -(-len(keep) // bs):
                continue
            before = {b for t in (mgr.tables()[0],) for b in t[t >= 0].tolist()}
            free = pool.num_free()
            plan = mgr.compact(s, keep)
            if np.array_equal(keep, np.arange(len(keep))):
                assert plan.src.size == 0  # a dropped tail moves nothing
            assert len(set(plan.dst.tolist())) == plan.dst.size and not set((plan.dst // bs).tolist()) & before
            assert (plan.token_seq == s).all() and plan.delta.size == plan.token_pos.size == plan.src.size
            for a, b in zip(plan.src, plan.dst):
                m.cells[int(b)] = m.cells[int(a)]
            m.seqs[s] = [toks[i] for i in keep]
            for i, p in enumerate(plan.token_pos):
                assert keep[p] + plan.delta[i] == p and m.cells[int(plan.dst[i])] == m.seqs[s][p]
            fresh = len(set((plan.dst // bs).tolist()))
            assert pool.num_free() == free - fresh + plan.evicted.size
            for b in plan.evicted:
                assert pool.ref_count(int(b)) == 0
        m.check(mgr, pool, n_seqs)


def test_compact_refusals_change_nothing():
    pool = BlockPool(8, BF16)
    mgr = KvManager(pool, 4, 2, 8)
    mgr.append([0], 22)  # six blocks, two free
    before = (mgr.tables()[0].copy(), mgr.positions().copy(), pool.num_free())

    def unchanged():
        t, c, f = mgr.tables()[0], mgr.positions(), pool.num_free()
        return np.array_equal(t, before[0]) and np.array_equal(c, before[1]) and f == before[2]

    for keep in ([-1], [2 ** 40], np.array([0, -5])):
        with pytest.raises(ValueError):
            mgr.compact(0, keep)
    for keep in ([0.0, 1.0], np.ones(22, bool)):
        with pytest.raises(TypeError):
            mgr.compact(0, keep)
    assert unchanged()
    for seq, keep in ((0, [1, 1]), (0, [2, 1]), (0, [22]), (0, [0, 5, 40]), (1, [0]), (2, []), (-1, []),
                      (0, list(range(1, 22)))):  # the last: six fresh blocks
        with pytest.raises(InvalidInput):
            mgr.compact(seq, keep)
        assert unchanged(), (seq, keep)
    arr, n = np.arange(1, 7, dtype=np.int32), C.c_int32()
    src, dst, ev = np.empty(6, np.int64), np.empty(6, np.int64), np.empty(8, np.int32)
    call = lambda **kw: L.lib.it_kv_manager_compact(*{**dict(  # noqa: E731
        m=mgr._h, seq=0, keep=arr.ctypes.data, n=6, src=src.ctypes.data, dst=dst.ctypes.data, delta=None, pos=None, cap=6,
        nm=C.byref(n), ev=ev.ctypes.data, evc=8, ne=C.byref(n)), **kw}.values())
    for kw in (dict(m=None), dict(keep=None), dict(src=None), dict(dst=None), dict(cap=5), dict(nm=None), dict(ev=None),
               dict(evc=5), dict(ne=None), dict(n=-1)):
        assert call(**kw) == L.INVALID_INPUT and unchanged(), kw
    assert call() == L.OK  # delta and pos are optional
    window = KvManager(BlockPool(8, BF16), 4, 1, 8, window=8)
    window.append([0], 6)
    with pytest.raises(NotImplementedOp):
        window.compact(0, [0, 1])


def test_compact_of_a_seeded_sequence_starts_at_zero():
    """Blocks that begin above logical block 0 (a sequence taken over from elsewhere): kept tokens are renumbered from 0."""
    pool = BlockPool(12, BF16)
    blocks = [pool.allocate() for _ in range(3)]
    mgr = KvManager(pool, 4, 1, 12)
    mgr.seed_seq(0, 18, 2, blocks)  # positions 8..17
    with pytest.raises(InvalidInput):
        mgr.compact(0, [7, 8])
    plan = mgr.compact(0, [9, 17])
    assert plan.src.tolist() == [blocks[0] * 4 + 1, blocks[2] * 4 + 1] and plan.delta.tolist() == [-9, -16]
    assert sorted(plan.evicted.tolist()) == sorted(blocks) and mgr.positions()[0] == 2


_DRIVER = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "it_kv.h"
int main() {
  unsigned r = 1;
  const auto rnd = [&](int n) { return int((r = r * 1664525u + 1013904223u) >> 8) % n; };
  it_block_pool* pool; it_kv_manager* m;
  if (it_block_pool_new(64, 30, &pool) || it_kv_manager_new(pool, 4, 3, 40, 0, &m)) return 1;
  std::vector<int32_t> ctx(3);
  for (int step = 0; step < 20000; ++step) {
    const int32_t s = rnd(3), n = rnd(9);
    it_kv_manager_tables(m, nullptr, 0, ctx.data(), nullptr);
    if (rnd(2) && it_block_pool_num_free(pool) > 4 && ctx[s] < 120) {
      std::vector<int64_t> slots(n + 1); std::vector<int32_t> ev(64), cs(n + 1), cd(n + 1); int32_t ne, nc;
      if (it_kv_manager_append_cow(m, &s, &n, 1, slots.data(), ev.data(), 64, &ne, cs.data(), cd.data(), n + 1, &nc)) return 2;
    } else {
      std::vector<int32_t> keep;
      const int drop = rnd(4);
      for (int32_t p = 0; p < ctx[s]; ++p) if (rnd(4) >= drop) keep.push_back(p);
      const size_t k = keep.size();
      std::vector<int64_t> src(k), dst(k); std::vector<int32_t> d(k), pos(k), ev(40); int32_t nm, ne;
      const int rc = it_kv_manager_compact(m, s, keep.data(), int32_t(k), src.data(), dst.data(), d.data(), pos.data(), int32_t(k), &nm, ev.data(), 40, &ne);
      if (rc && it_block_pool_num_free(pool) >= int64_t(k + 3) / 4) return 3;
      const int32_t t = (s + 1) % 3;
      if (!rc && rnd(3) == 0) { int32_t n2; if (it_kv_manager_release_seq(m, t, ev.data(), 40, &n2) || it_kv_manager_fork(m, s, t)) return 4; }
    }
  }
  it_kv_manager_destroy(m); it_block_pool_destroy(pool);
  return 0;
}
"""


def test_compact_under_sanitizers(tmp_path):
    src, exe = tmp_path / "compact.cpp", str(tmp_path / "compact")
    src.write_text(_DRIVER)
    host = os.path.join(ROOT, "infer_train_amd", "csrc", "it_host.cpp")
    b = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I",
                        os.path.join(ROOT, "include"), "-I", os.path.dirname(host), str(src), host, "-o", exe],
                       capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stderr[-2000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])


def test_batcher_sample_checks_rows():
    import torch
    from infer_train_amd import ContinuousBatcher, SamplingParams

    b = ContinuousBatcher(4)
    b.add_request(7, [1, 2], 5, SamplingParams(temperature=0.0))
    b.add_request(8, [1], 5)
    assert b.requests[8].sampling == SamplingParams()
    b.schedule()
    with pytest.raises(ValueError):
        b.sample(torch.zeros(1, 10), torch.zeros(1))
    with pytest.raises(ValueError):
        b.sample(torch.zeros(2, 10), torch.zeros(2))  # host tensors
    assert b.requests[7].generated_tokens == []
    assert ContinuousBatcher(1).sample(torch.zeros(0, 10), torch.zeros(0)) == []
