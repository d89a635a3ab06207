"""Host-side batch state: the reference's FIFO `ContinuousBatcher`
(src/batcher/continuous.rs:8-74) plus the per-step slot mapping, block
tables and sliding-window eviction it lacks (native: it_kv_manager_*)."""
from __future__ import annotations

import ctypes as C
import weakref
from collections import deque
from dataclasses import dataclass, field
from enum import Enum
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np

from ._lib import StepPlanC, check, lib
from .memory import BlockPool

__all__ = ["KvManager", "ContinuousBatcher", "RequestState", "RequestContext", "StepPlan", "CompactPlan",
           "SamplingParams"]


_EMPTY = np.zeros(0, np.int32)
_EMPTY.flags.writeable = False


@dataclass
class StepPlan:
    """What one append step hands to the device: the slot of every new token
    with its sequence and position (it_kv_sync_tables' inputs), the blocks
    the step returned to the pool (refcount 0: the pages to clear with
    kv_evict), the copy-on-write page pairs (to copy with kv_copy_blocks
    before the append), and every sequence slot's context length and window
    start after the step."""

    slots: np.ndarray
    evicted: np.ndarray
    cow_src: np.ndarray = field(default_factory=lambda: np.zeros(0, np.int32))
    cow_dst: np.ndarray = field(default_factory=lambda: np.zeros(0, np.int32))
    token_seq: np.ndarray = field(default_factory=lambda: np.zeros(0, np.int32))
    token_pos: np.ndarray = field(default_factory=lambda: np.zeros(0, np.int32))
    ctx_lens: Optional[np.ndarray] = None
    start_pos: Optional[np.ndarray] = None


@dataclass
class CompactPlan:
    """What dropping tokens out of sequences hands to the device, in this
    order: kv_move (src, dst, and delta for rotated keys), kv_evict of the
    blocks that returned to the pool, kv_sync_tables with (token_seq,
    token_pos, dst).  All of it is queued before what any later plan of the
    manager hands over: that may use the returned blocks.  Two plans are never
    joined; KvManager.compact_many makes one for several sequences."""

    src: np.ndarray
    dst: np.ndarray
    delta: np.ndarray
    token_seq: np.ndarray
    token_pos: np.ndarray
    evicted: np.ndarray


class KvManager:
    """Slot mapping and block tables over a BlockPool (native:
    it_kv_manager_step).

    slot(pos) = table[pos // bs] * bs + pos % bs; a block is allocated when
    pos % bs == 0.  With `window` W > 0, before the token at position p every
    held block whose last position is < p - W + 1 drops this sequence's
    reference (oldest first); the blocks whose refcount reaches 0 are the
    step's `evicted` list.  Sequences of one step are processed in the order
    listed.
    """

    def __init__(self, pool: BlockPool, block_size: int, max_seqs: int, max_blocks_per_seq: int, window: int = 0):
        self.pool = pool  # keep the borrowed pool alive
        self.block_size = block_size
        self.max_seqs = max_seqs
        self.max_blocks = max_blocks_per_seq
        self.window = window
        h = C.c_void_p()
        check(lib.it_kv_manager_new(pool.handle, block_size, max_seqs, max_blocks_per_seq, window, C.byref(h)))
        self._h = h
        self._compacted = False  # a sequence was compacted or reordered: appends may need copy-on-write
        self._watchers: List[weakref.WeakMethod] = []  # called with what a compaction kept
        self._destroy = lib.it_kv_manager_destroy  # bound now: module globals may be gone at exit
        # Reused buffers of it_kv_manager_step (grown on demand), with their
        # addresses cached (ndarray.ctypes.data costs about a microsecond);
        # the plan returned to the caller holds copies.
        self._plan = StepPlanC()
        self._plan_ref = C.byref(self._plan)
        self._step_fn = lib.it_kv_manager_step
        self._tok_cap = 0
        self._seq_cap = 0
        # Blocks returned to the pool in one step: at most the pool's capacity.
        self._ev = np.empty(pool.capacity() + 1, np.int32)
        self._plan.evicted = self._ev.ctypes.data
        self._plan.evicted_cap = self._ev.size
        self._lens = np.empty((2, max_seqs), np.int32)  # ctx_lens, start_pos
        self._plan.ctx_lens, self._plan.start_pos = self._lens[0].ctypes.data, self._lens[1].ctypes.data
        self._grow_tokens(64)
        self._grow_seqs(64)

    def _grow_tokens(self, total: int) -> None:
        cap = max(total, 2 * self._tok_cap)
        self._slots = np.empty(cap, np.int64)
        self._tsp = np.empty((2, cap), np.int32)  # token_seq, token_pos
        self._cs = np.empty(cap, np.int32)
        self._cd = np.empty(cap, np.int32)
        pl = self._plan
        pl.slots, pl.token_seq, pl.token_pos = self._slots.ctypes.data, self._tsp[0].ctypes.data, self._tsp[1].ctypes.data
        pl.tokens_cap = cap
        pl.cow_cap = cap  # at most one copy per token
        self._cs_addr, self._cd_addr = self._cs.ctypes.data, self._cd.ctypes.data
        self._tok_cap = cap

    def _grow_seqs(self, n: int) -> None:
        cap = max(n, 2 * self._seq_cap)
        self._seqbuf = np.empty(cap, np.int32)
        self._ntbuf = np.empty(cap, np.int32)
        self._seq_addr, self._nt_addr = self._seqbuf.ctypes.data, self._ntbuf.ctypes.data
        self._seq_cap = cap

    def seed_seq(self, seq: int, pos: int, first_block: int, blocks: Sequence[int]) -> None:
        arr = np.ascontiguousarray(np.asarray(blocks, dtype=np.int32))
        check(lib.it_kv_manager_seed_seq(self._h, seq, int(pos), int(first_block), arr.ctypes.data, arr.size))

    def append(self, seqs: Sequence[int], n_tokens: Sequence[int] | int = 1, cow: bool = False) -> StepPlan:
        """One step: n_tokens[i] tokens to seqs[i] (in list order)."""
        n = len(seqs)
        if n > self._seq_cap:
            self._grow_seqs(n)
        self._seqbuf[:n] = seqs
        nt = self._ntbuf[:n]
        if np.isscalar(n_tokens):
            nt.fill(n_tokens)
            total = int(n_tokens) * n
        else:
            nt[:] = n_tokens
            total = int(nt.sum())
        if total > self._tok_cap:
            self._grow_tokens(total)
        pl = self._plan
        pl.cow_src = self._cs_addr if cow else None
        pl.cow_dst = self._cd_addr if cow else None
        rc = self._step_fn(self._h, self._seq_addr, self._nt_addr, n, self._plan_ref)
        if rc:
            check(rc)
        k, ne, nc = pl.n_tokens, pl.n_evicted, pl.n_cow
        tsp, lens = self._tsp[:, :k].copy(), self._lens.copy()
        return StepPlan(self._slots[:k].copy(), self._ev[:ne].copy() if ne else _EMPTY,
                        self._cs[:nc].copy() if nc else _EMPTY, self._cd[:nc].copy() if nc else _EMPTY,
                        tsp[0], tsp[1], lens[0], lens[1])

    def compact(self, seq: int, keep: Sequence[int]) -> CompactPlan:
        """Keep only the tokens at these positions (ascending) of `seq`:
        keep[i] becomes position i (it_kv_manager_compact).  Leading blocks
        whose tokens all keep their positions stay, what is kept of the others
        moves to fresh ones.  Dropping a tail moves nothing; if a fork still
        reads dropped tokens in the last block, the next append to `seq` has to
        be with cow=True (needs_cow), and is refused without.  The plan's device
        work is queued before that of any later plan; compact_many plans several
        sequences for one move."""
        return self.compact_many([seq], [keep])

    def compact_many(self, seqs: Sequence[int], keeps: Sequence[Sequence[int]]) -> CompactPlan:
        """compact() of several sequences as one plan, whose rows go in one
        move: no row of it is written before all of them are read
        (it_kv_manager_compact_many).  All are compacted, or none."""
        if len(seqs) != len(keeps):
            raise ValueError("a list of positions per sequence")
        rows = [self._positions(k) for k in keeps]
        cu = np.zeros(len(rows) + 1, np.int64)
        np.cumsum([r.size for r in rows], out=cu[1:])
        n = int(cu[-1])
        if n > np.iinfo(np.int32).max:
            raise ValueError("keep: more than 2^31 - 1 positions")
        cu = cu.astype(np.int32)
        at = np.ascontiguousarray(seqs, dtype=np.int32)
        pos = np.concatenate(rows) if rows else _EMPTY
        src, dst = np.empty(n, np.int64), np.empty(n, np.int64)
        delta, of, new = np.empty(n, np.int32), np.empty(n, np.int32), np.empty(n, np.int32)
        ev = np.empty(min(self.max_blocks * max(at.size, 1), self.pool.capacity()), np.int32)
        nm, nev = C.c_int32(0), C.c_int32(0)
        held = self.positions() if self._watchers else None
        check(lib.it_kv_manager_compact_many(self._h, at.ctypes.data, at.size, pos.ctypes.data, cu.ctypes.data, src.ctypes.data,
                                             dst.ctypes.data, delta.ctypes.data, of.ctypes.data, new.ctypes.data, n, C.byref(nm),
                                             ev.ctypes.data, ev.size, C.byref(nev)))
        m = nm.value
        self._compacted = True
        for watcher in self._watchers:
            kept = watcher()
            for seq, row in zip(at.tolist(), rows) if kept is not None else ():
                kept(seq, row.tolist(), int(held[seq]))
        return CompactPlan(src[:m], dst[:m], delta[:m], of[:m], new[:m], ev[:nev.value].copy())

    @staticmethod
    def _positions(keep: Sequence[int]) -> np.ndarray:
        kept = np.asarray(keep)
        if kept.size and kept.dtype.kind not in "iu":
            raise TypeError("keep must hold positions (integers)")
        if kept.size and (kept.min() < 0 or kept.max() > np.iinfo(np.int32).max):
            raise ValueError("keep: positions outside the sequence")
        return np.ascontiguousarray(kept, dtype=np.int32).reshape(-1)

    def reorder(self, seqs: Sequence[int], parents: Sequence[int]) -> np.ndarray:
        """Beams reordered: sequence seqs[i] continues what seqs[parents[i]]
        held (it_kv_manager_reorder; a parent below 0: it stays).  Nothing is
        copied: the next append has to be cow=True where beams continue the same
        partial block (needs_cow), and is refused without.  Returns the blocks
        that went back to the pool, the pages to clear; the rows of a device
        block table are put in the same order (beam.beam_reorder)."""
        if len(seqs) != len(parents):
            raise ValueError("a parent per sequence")
        at, of = np.ascontiguousarray(seqs, dtype=np.int32), np.ascontiguousarray(parents, dtype=np.int32)
        ev = np.empty(min(self.max_blocks * max(at.size, 1), self.pool.capacity()), np.int32)
        nev = C.c_int32(0)
        check(lib.it_kv_manager_reorder(self._h, at.ctypes.data, of.ctypes.data, at.size, ev.ctypes.data, ev.size, C.byref(nev)))
        self._compacted = True
        return ev[:nev.value].copy()

    def needs_cow(self, seqs: Sequence[int]) -> bool:
        """Whether one append to these sequences needs copy-on-write, because a
        compaction set one back to where a fork holds a token in the same block
        or another of them would write one, or a reordering left several to
        continue it (it_kv_manager_needs_cow)."""
        if not self._compacted:
            return False
        at = np.ascontiguousarray(seqs, dtype=np.int32)
        rc = lib.it_kv_manager_needs_cow(self._h, at.ctypes.data, at.size)
        if rc < 0:
            raise ValueError("sequence slots outside the manager")
        return rc == 1

    def positions(self) -> np.ndarray:
        """Next position (= context length) of every sequence slot."""
        cl = np.empty(self.max_seqs, dtype=np.int32)
        check(lib.it_kv_manager_tables(self._h, None, 0, cl.ctypes.data, None))
        return cl

    def release(self, seq: int) -> np.ndarray:
        """Drop every block of `seq`; returns the blocks that went back to
        the pool (refcount 0), the pages to clear."""
        cap = self.max_blocks
        ev = np.empty(cap, dtype=np.int32)
        nev = C.c_int32(0)
        check(lib.it_kv_manager_release_seq(self._h, seq, ev.ctypes.data, cap, C.byref(nev)))
        return ev[:nev.value].copy()

    def fork(self, src: int, dst: int) -> None:
        check(lib.it_kv_manager_fork(self._h, src, dst))

    def tables(self, max_blocks: Optional[int] = None) -> Tuple[np.ndarray, np.ndarray, np.ndarray]:
        mb = self.max_blocks if max_blocks is None else max_blocks
        t = np.empty((self.max_seqs, mb), dtype=np.int32)
        cl = np.empty(self.max_seqs, dtype=np.int32)
        sp = np.empty(self.max_seqs, dtype=np.int32)
        check(lib.it_kv_manager_tables(self._h, t.ctypes.data, mb, cl.ctypes.data, sp.ctypes.data))
        return t, cl, sp

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            self._destroy(h)
            self._h = None


@dataclass(frozen=True)
class SamplingParams:
    """How a request's tokens are drawn (sampling.sample); the defaults draw
    from the whole distribution.  temperature 0 takes the most likely token;
    top_k 0, top_p 1 and min_p 0 are off."""

    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0


class RequestState(Enum):  # continuous.rs:8-15
    Running = "Running"
    Waiting = "Waiting"
    Preempted = "Preempted"
    Finished = "Finished"


@dataclass
class RequestContext:  # continuous.rs:17-25
    request_id: int
    state: RequestState
    prompt_tokens: List[int]
    generated_tokens: List[int]
    max_tokens: int
    sampling: SamplingParams = SamplingParams()


class ContinuousBatcher:
    """FIFO admission (continuous.rs:28-74) wired to a KvManager.

    `schedule()` moves waiting requests to running up to max_batch_size, in
    arrival order (continuous.rs:62-73).  Each running request is bound to a
    manager sequence slot; `plan_prefill` / `plan_decode` produce the step's
    slot mapping through the manager, and `finish` releases the blocks.

    Preemption (the reference declares RequestState::Preempted,
    continuous.rs:13, but never enters it): `preempt` moves a running
    request to Preempted, either releasing its blocks and sequence slot (the
    request is prefilled again, prompt and generated tokens, when it resumes)
    or keeping them (it resumes where it stopped).  `preempt_for(n)` frees
    pool blocks by preempting, releasing, the most recently admitted running
    requests first until n blocks are free.  `schedule()` resumes preempted
    requests, in the order they were preempted, before it admits waiting
    ones.  Every choice depends only on the call sequence, so block ids stay
    deterministic.

    A request whose sequence was compacted (KvManager.compact) is prefilled
    again with what it had kept, at the positions that it had moved to
    (`context`).  Its generated_tokens are expected to hold the accepted tokens
    alone when drafts are dropped, or to lack the drafts altogether.
    """

    def __init__(self, max_batch_size: int, manager: Optional[KvManager] = None):
        self.requests: Dict[int, RequestContext] = {}
        self.running: List[int] = []
        self.waiting: deque = deque()
        self.max_batch_size = max_batch_size
        self.manager = manager
        self.seq_of: Dict[int, int] = {}
        self._free_seqs: List[int] = list(range(manager.max_seqs - 1, -1, -1)) if manager else []
        self.preempted: deque = deque()  # preemption order
        self.needs_prefill: set = set()  # released by preemption: prefill again on resume
        # Of compacted requests: which of their tokens (prompt, then generated) the cache
        # holds, in order, and the first of those that follow them.
        self._kept: Dict[int, Tuple[List[int], int]] = {}
        if manager is not None:
            manager._watchers.append(weakref.WeakMethod(self._note_compaction))

    def add_request(self, request_id: int, prompt: Sequence[int], max_tokens: int,
                    sampling: SamplingParams = SamplingParams()) -> None:  # :45-60
        self.requests[request_id] = RequestContext(request_id, RequestState.Waiting, list(prompt), [], max_tokens, sampling)
        self._kept.pop(request_id, None)
        self.waiting.append(request_id)

    def _note_compaction(self, seq: int, keep: List[int], held: int) -> None:
        rid = next((r for r, s in self.seq_of.items() if s == seq), None)
        if rid is None:  # not a request's sequence
            return
        ctx = self.requests[rid]
        n = len(ctx.prompt_tokens) + len(ctx.generated_tokens)
        base, follow = self._kept.get(rid, ([], 0))
        token = lambda p: base[p] if p < len(base) else follow + p - len(base)  # noqa: E731
        kept = [token(p) for p in keep]
        # Positions past the tokens known are drafts; those kept become the next tokens.
        follow = max(min(token(max(held, len(base))), n), kept[-1] + 1 if kept else 0)
        kept += base[held:]
        if kept == list(range(follow)):
            self._kept.pop(rid, None)
        else:
            self._kept[rid] = kept, follow

    def context(self, request_id: int) -> List[int]:
        """The tokens of a request's context, in the order of their positions:
        its prompt and generated tokens, without those that compactions
        dropped.  What plan_resume prefills."""
        ctx = self.requests[request_id]
        tokens = ctx.prompt_tokens + ctx.generated_tokens
        kept, follow = self._kept.get(request_id, ([], 0))
        return [tokens[i] for i in kept if i < len(tokens)] + tokens[follow:]

    def schedule(self) -> List[int]:  # :62-73
        while len(self.running) < self.max_batch_size:
            if self.preempted:  # resumed first, in preemption order
                rid = self.preempted.popleft()
            elif self.waiting:
                rid = self.waiting.popleft()
            else:
                break
            ctx = self.requests.get(rid)
            if ctx is not None:
                ctx.state = RequestState.Running
                self.running.append(rid)
                if self.manager is not None and rid not in self.seq_of:
                    if not self._free_seqs:
                        raise RuntimeError("no free sequence slot in the KV manager")
                    self.seq_of[rid] = self._free_seqs.pop()
        return list(self.running)

    def preempt(self, request_id: int, keep_blocks: bool = False) -> np.ndarray:
        """Running -> Preempted.  keep_blocks False: the request's blocks are
        released (BlockPool::free, lowest logical block first) with its
        sequence slot, and it is prefilled again on resume; True: blocks and
        slot stay held.  Returns the blocks that went back to the pool
        (refcount 0: the pages to clear; a block a forked request still
        holds is not among them), empty when kept."""
        ctx = self.requests[request_id]
        if ctx.state != RequestState.Running:
            raise ValueError(f"request {request_id} is {ctx.state.value}, not Running")
        ctx.state = RequestState.Preempted
        self.running.remove(request_id)
        self.preempted.append(request_id)
        freed = np.zeros(0, np.int32)
        if not keep_blocks and self.manager is not None and request_id in self.seq_of:
            seq = self.seq_of.pop(request_id)
            freed = self.manager.release(seq)
            self._free_seqs.append(seq)
            self.needs_prefill.add(request_id)
        return freed

    def preempt_for(self, n_blocks: int) -> List[int]:
        """Preempt (releasing) the most recently admitted running requests
        until the pool holds n_blocks free blocks; returns them in the order
        they were preempted.  Raises if even preempting every running request
        does not free enough."""
        pool = self.manager.pool
        out: List[int] = []
        while pool.num_free() < n_blocks:
            if not self.running:
                raise RuntimeError(f"cannot free {n_blocks} blocks: {pool.num_free()} free with nothing running")
            rid = self.running[-1]
            self.preempt(rid, keep_blocks=False)
            out.append(rid)
        return out

    def plan_resume(self, request_ids: Sequence[int]) -> StepPlan:
        """Prefill again the requests a releasing preemption emptied: their
        prompt plus the tokens generated before the preemption, without what
        compactions had dropped (context)."""
        seqs = [self.seq_of[r] for r in request_ids]
        lens = [len(self.context(r)) for r in request_ids]
        for r in request_ids:
            self.needs_prefill.discard(r)
        return self.manager.append(seqs, lens)

    def plan_prefill(self, request_ids: Sequence[int]) -> StepPlan:
        seqs = [self.seq_of[r] for r in request_ids]
        lens = [len(self.requests[r].prompt_tokens) for r in request_ids]
        return self.manager.append(seqs, lens)

    def plan_decode(self) -> StepPlan:
        """One token for every running request.  After a compaction that
        dropped a tail which a fork still reads, or a reordering after which
        beams continue the same block, the plan holds copy-on-write pairs (cow_src, cow_dst), whose pages are copied before the append."""
        seqs = [self.seq_of[r] for r in self.running]
        return self.manager.append(seqs, 1, cow=self.manager.needs_cow(seqs))

    def sample(self, logits, u, request_ids: Optional[Sequence[int]] = None) -> List[int]:
        """Draw the next tokens of running requests, each with its own settings,
        from logits [n, vocab] and uniform numbers u [n] (device tensors, as
        sampling.sample takes them): a row for each of request_ids (the ones
        just prefilled or resumed, say), or for all that run, in plan_decode's
        order.  They join the requests' generated_tokens, and the caller
        finishes those that reached max_tokens.  A row with nothing above -inf
        raises before any request changes."""
        import torch

        from .sampling import sample

        ids = self.running if request_ids is None else list(request_ids)
        n = len(ids)
        if request_ids is not None and (len(set(ids)) != n or not set(ids) <= set(self.running)):
            raise ValueError("request_ids must be running requests, each listed once")
        if logits.dim() != 2 or logits.shape[0] != n:
            raise ValueError(f"logits must be [{n}, vocab], a row per request")
        if n == 0:
            return []
        host = np.empty((4, n), np.float32)  # one copy to the device
        for i, rid in enumerate(ids):
            p = self.requests[rid].sampling
            host[0, i], host[2, i], host[3, i] = p.temperature, p.top_p, p.min_p
            host[1].view(np.int32)[i] = p.top_k
        dev = torch.from_numpy(host).to(logits.device)
        drawn, _ = sample(logits, u, temperature=dev[0], top_k=dev[1].view(torch.int32), top_p=dev[2], min_p=dev[3])
        tokens = drawn.tolist()
        if min(tokens) < 0:
            raise ValueError(f"request {ids[tokens.index(-1)]}: no token above -inf")
        for rid, token in zip(ids, tokens):
            self.requests[rid].generated_tokens.append(token)
        return tokens

    def reorder(self, request_ids: Sequence[int], parents: Sequence[int]) -> np.ndarray:
        """Running requests that are one search's beams put in the selected
        order: request_ids[i] continues what request_ids[parents[i]] held, its
        prompt, generated tokens and cached blocks (a parent below 0: it stays).
        The caller then appends each one's selected token.  Returns the blocks
        that went back to the pool, the pages to clear."""
        ids = list(request_ids)
        if len(set(ids)) != len(ids) or not set(ids) <= set(self.running):
            raise ValueError("request_ids must be running requests, each listed once")
        of = [i if p < 0 else p for i, p in enumerate(int(p) for p in parents)]
        if len(of) != len(ids) or max(of, default=0) >= max(len(ids), 1):
            raise ValueError("a parent per request, each an index into request_ids")
        freed = np.zeros(0, np.int32)
        if self.manager is not None:
            freed = self.manager.reorder([self.seq_of[r] for r in ids], of)
        was = [(self.requests[r].prompt_tokens, self.requests[r].generated_tokens, self._kept.get(r), r in self.needs_prefill) for r in ids]
        for rid, p in zip(ids, of):
            prompt, generated, kept, empty = was[p]
            (self.needs_prefill.add if empty else self.needs_prefill.discard)(rid)
            self.requests[rid].prompt_tokens, self.requests[rid].generated_tokens = list(prompt), list(generated)
            if kept is None:
                self._kept.pop(rid, None)
            else:
                self._kept[rid] = (list(kept[0]), kept[1])
        return freed

    def finish(self, request_id: int) -> np.ndarray:
        """Running or Preempted -> Finished; the request's blocks (if it
        still holds them) and sequence slot are released.  Returns the
        blocks that went back to the pool (refcount 0)."""
        ctx = self.requests[request_id]
        if ctx.state == RequestState.Running:
            self.running.remove(request_id)
        elif ctx.state == RequestState.Preempted:
            self.preempted.remove(request_id)
        else:
            raise ValueError(f"request {request_id} is {ctx.state.value}")
        ctx.state = RequestState.Finished
        self.needs_prefill.discard(request_id)
        self._kept.pop(request_id, None)
        freed = np.zeros(0, np.int32)
        if self.manager is not None and request_id in self.seq_of:
            seq = self.seq_of.pop(request_id)
            freed = self.manager.release(seq)
            self._free_seqs.append(seq)
        return freed
