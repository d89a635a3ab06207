"""The operators around the paged cache's attention: rotary positions on the
way into the cache, moving rows inside it, and the draw of the next token.

Kinds of case:

  append  a step's projections rotated and stored: q, k and v of `tokens` new
          tokens (k and v into their pages, k rotated), q rotated for the
          attention that follows;
  rotate  the rotation of one tensor, forwards or transposed (its gradient);
  move    a cache compacted: rows kept out of a sequence's middle moved to
          other slots in every layer, keys re-rotated to their new positions;
  sample  one token per row of logits: temperature, min-p, top-k, top-p and a
          given uniform number.

Sizes belong to the case, the values, positions, block order and parameters
per row to the seed of `prepare`.  Where `own` is false the operators run in
their plain form, in float32 (angles and probability masses in float64).
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_DEV = "cuda:0"
_BASE = 10000.0


def listed():
    return [
        # One user's next token: 28 query heads over 4 KV heads, where latency is all there is.
        {"name": "append_one_bf16", "kind": "append", "heads": 28, "kv_heads": 4, "dim": 128, "rot": 128, "layout": "half",
         "scaling": "none", "factor": 1.0, "src": "bf16", "cache": "bf16", "block": 16, "tokens": 1, "seqs": 1,
         "max_pos": 4096, "pad": 0, "fused": True},
        # A decode step of 128 sequences, some of them far into a context extended 16 times.
        {"name": "append_batch_bf16", "kind": "append", "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "layout": "half", "scaling": "parts", "factor": 16.0, "src": "bf16", "cache": "bf16", "block": 16, "tokens": 128,
         "seqs": 128, "max_pos": 131072, "pad": 0, "fused": True},
        # A batch of prompt chunks from float32 projections, in interleaved pairs, positions interpolated.
        {"name": "append_chunk_f32", "kind": "append", "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "layout": "interleaved", "scaling": "linear", "factor": 4.0, "src": "f32", "cache": "bf16", "block": 16,
         "tokens": 4096, "seqs": 8, "max_pos": 32768, "pad": 0, "fused": False},
        # A third of each head rotated, an odd number of tokens, the batch padded.
        {"name": "append_part_f16", "kind": "append", "heads": 9, "kv_heads": 3, "dim": 96, "rot": 32, "layout": "half",
         "scaling": "none", "factor": 1.0, "src": "f16", "cache": "f16", "block": 32, "tokens": 1543, "seqs": 5,
         "max_pos": 8192, "pad": 57, "fused": False},
        # The gradient of a training step's rotation.
        {"name": "rotate_grad_f32", "kind": "rotate", "heads": 32, "dim": 128, "rot": 128, "layout": "half",
         "scaling": "none", "factor": 1.0, "src": "f32", "tokens": 4096, "seqs": 2, "max_pos": 4096, "transpose": True},
        # One sequence compacted in one layer: its first tokens, the heavy ones and the recent ones stay.
        {"name": "move_one_bf16", "kind": "move", "layers": 1, "kv_heads": 4, "dim": 128, "rot": 128, "layout": "half",
         "cache": "bf16", "block": 16, "seqs": 1, "ctx": 1024, "keep": 0.25, "rotate": True},
        # Four sequences halved in all 28 layers of a model.
        {"name": "move_model_bf16", "kind": "move", "layers": 28, "kv_heads": 4, "dim": 128, "rot": 128, "layout": "half",
         "cache": "bf16", "block": 16, "seqs": 4, "ctx": 2048, "keep": 0.5, "rotate": True},
        # Rows copied as they are (keys stored without positions), float32, an odd count.
        {"name": "move_copy_f32", "kind": "move", "layers": 3, "kv_heads": 4, "dim": 256, "rot": 256,
         "layout": "interleaved", "cache": "f32", "block": 32, "seqs": 3, "ctx": 1999, "keep": 0.37, "rotate": False},
        # One user's next token with the usual settings.
        {"name": "sample_one_f32", "kind": "sample", "rows": 1, "vocab": 32000, "src": "f32", "mode": "usual", "masked": False},
        # A served batch: every request has its own settings, some are greedy, an odd vocabulary.
        {"name": "sample_mixed_bf16", "kind": "sample", "rows": 64, "vocab": 100003, "src": "bf16", "mode": "mixed",
         "masked": True},
        # Sampling the whole distribution, half the vocabulary masked in some rows (a grammar).
        {"name": "sample_full_f16", "kind": "sample", "rows": 16, "vocab": 32768, "src": "f16", "mode": "full", "masked": True},
        # The largest: 256 rows of a large vocabulary cut by mass alone.
        {"name": "sample_mass_f32", "kind": "sample", "rows": 256, "vocab": 131072, "src": "f32", "mode": "mass",
         "masked": False},
    ]


# (query heads, KV heads, head dim) of the repository's configurations and tests, and generic ones.
_HEADS = ((12, 2, 128), (28, 4, 128), (32, 8, 128), (16, 2, 128), (24, 4, 256), (8, 8, 64), (10, 2, 128), (9, 3, 96),
          (64, 8, 128), (5, 1, 80))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(("append", "append", "rotate", "move", "move", "sample", "sample", "sample"))
    if kind == "sample":
        rows = _log(rng, 1, 256)
        return {"kind": kind, "rows": rows, "vocab": min(_log(rng, 64, 262144), (256 * 131072) // rows),
                "src": rng.choice(("f32", "bf16", "f16")), "mode": rng.choice(("usual", "mixed", "full", "mass")),
                "masked": rng.random() < 0.5}
    heads, kv, dim = rng.choice(_HEADS)
    c = {"kind": kind, "kv_heads": kv, "dim": dim, "rot": rng.choice((dim, dim, dim // 2, 32)),
         "layout": rng.choice(("half", "half", "interleaved"))}
    if kind == "move":
        c.update(cache=rng.choice(("bf16", "bf16", "f16", "f32")), block=rng.choice((8, 16, 32)), layers=_log(rng, 1, 32),
                 seqs=_log(rng, 1, 16), keep=round(rng.uniform(0.05, 0.95), 3), rotate=rng.random() < 0.75)
        token = c["layers"] * kv * dim * _SIZE[c["cache"]]
        c["ctx"] = _log(rng, 16, max(17, min(32768, 4 * 2048 * 28 * 4 * 128 * 2 // (token * c["seqs"]))))
        return c
    scaling = rng.choice(("none", "none", "linear", "base", "parts"))
    c.update(heads=heads, scaling=scaling, factor=1.0 if scaling == "none" else rng.choice((2.0, 8.0, 40.0)),
             src=rng.choice(("bf16", "bf16", "f16", "f32")), max_pos=_log(rng, 8192, 1 << 20))
    row = (heads + 2 * kv if kind == "append" else heads) * dim * _SIZE[c["src"]]
    cap = 4096 * (48 if kind == "append" else 32) * 128 * 4 // row
    c["tokens"] = _log(rng, 1, min(8191, cap))
    c["seqs"] = min(c["tokens"], _log(rng, 1, 256))
    if kind == "rotate":
        c["transpose"] = rng.random() < 0.5
        return c
    c.update(cache=rng.choice((c["src"], c["src"], "f32")) if c["src"] != "f32" else rng.choice(("f32", "bf16", "f16")),
             block=rng.choice((8, 16, 32)), pad=c["tokens"] // rng.choice((7, 1 << 20)), fused=rng.random() < 0.5)
    return c


def _frequencies(c):
    """Angle per position of each pair, float64, and the rotation's magnitude."""
    i = torch.arange(c["rot"] // 2, dtype=torch.float64)
    base, s = _BASE, c.get("factor", 1.0)
    scaling = c.get("scaling", "none")
    if scaling == "base":
        base *= s ** (c["rot"] / max(c["rot"] - 2, 1))
    f = base ** (-2.0 * i / c["rot"])
    if scaling == "linear":
        f = f / s
    if scaling == "parts":  # 8192 positions trained; 1 to 32 turns in them are blended
        turns = 8192.0 * f / (2 * math.pi)
        g = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        return f * (g + (1.0 - g) / s), 0.1 * math.log(s) + 1.0
    return f, 1.0


def _rotary(c):
    import infer_train_amd.kv as kv

    m = _frequencies(c)[1]
    return kv.Rotary(c["rot"], layout=c["layout"], freq_base=_BASE, scaling=c.get("scaling", "none"),
                     factor=c.get("factor", 1.0), original_ctx=8192, low=1.0, high=32.0, magnitude=m)


def _id(name):
    import infer_train_amd as it

    return {"f32": it.F32, "f16": it.F16, "bf16": it.BF16}[name]


def _pools(c, blocks, layers, gen):
    """K and V pools holding random rows, [layers, blocks, heads, block, dim]; the plain form's with one
    more block at the end, which takes the padding tokens' rows."""
    shape = (layers, blocks, c["kv_heads"], c["block"], c["dim"])
    if own:
        from infer_train_amd.kv import PagedKvCache

        cache = PagedKvCache(blocks, c["block"], c["kv_heads"], c["dim"], _id(c["cache"]), n_layers=layers)
        pools = [p.view(_TORCH[c["cache"]]).view(shape) for p in (cache.k_pool, cache.v_pool)]
    else:
        cache = None
        pools = [torch.zeros((layers, blocks + 1) + shape[2:], dtype=_TORCH[c["cache"]], device=_DEV) for _ in "kv"]
    for p in pools:
        p[:, :blocks].copy_(torch.randn(shape, generator=gen, device=_DEV, dtype=torch.float32))
    return cache, pools


def _runs(c, rng):
    """Positions of `tokens` tokens in `seqs` runs, and each run's length."""
    n, s = c["tokens"], min(c["seqs"], c["tokens"])
    cuts = sorted(rng.sample(range(1, n), s - 1)) if s > 1 else []
    lens = [b - a for a, b in zip([0] + cuts, cuts + [n])]
    return [(rng.randrange(0, max(1, c["max_pos"] - m)), m) for m in lens]


def _append_inputs(c, seed):
    rng = random.Random(seed)
    runs, bs = _runs(c, rng), c["block"]
    pos = np.concatenate([np.arange(p, p + m) for p, m in runs])
    logical, at = [], 0
    for p, m in runs:  # a fresh block for each block of positions that a run touches
        logical.append(np.arange(p, p + m) // bs - p // bs + at)
        at += (p + m - 1) // bs - p // bs + 1
    blocks = c["tokens"] // bs + 2 * c["seqs"] + 2  # of any runs
    order = np.random.default_rng(seed).permutation(blocks)
    slots = order[np.concatenate(logical)] * bs + pos % bs
    if c.get("pad"):
        slots[len(slots) - c["pad"]:] = -1
    return pos.astype(np.int32), slots.astype(np.int64), blocks


def _move_inputs(c, seed):
    """Source and destination slots and position changes of the rows that a compaction moves."""
    rng = np.random.default_rng(seed)
    bs, ctx = c["block"], c["ctx"]
    held = -(-ctx // bs)
    blocks = c["seqs"] * 2 * held
    order = rng.permutation(blocks)
    src, dst, delta = [], [], []
    for s in range(c["seqs"]):
        n = max(1, int(ctx * c["keep"]))
        old_blocks = order[s * held:(s + 1) * held]
        new_blocks = order[(c["seqs"] + s) * held:(c["seqs"] + s + 1) * held]
        sinks, recent = min(4, n), max(0, n // 2 - 4)
        middle = np.sort(rng.choice(np.arange(sinks, ctx - recent), n - sinks - recent, replace=False))
        old = np.concatenate([np.arange(sinks), middle, np.arange(ctx - recent, ctx)])
        new = np.arange(n)
        first = int(np.argmax(old != new)) // bs * bs if (old != new).any() else n  # whole blocks that stay as they are
        old, new = old[first:], new[first:]
        src.append(old_blocks[old // bs] * bs + old % bs)
        dst.append(new_blocks[new // bs] * bs + new % bs)
        delta.append(new - old)
    cat = lambda a: np.concatenate(a)  # noqa: E731
    return cat(src).astype(np.int64), cat(dst).astype(np.int64), cat(delta).astype(np.int32), blocks


def _sample_params(c, seed):
    """temperature, top_k, top_p, min_p of every row."""
    rng, rows = np.random.default_rng(seed), c["rows"]
    t = rng.uniform(0.5, 1.3, rows)
    k, p, m = np.zeros(rows, np.int32), np.ones(rows), np.zeros(rows)
    if c["mode"] == "usual":
        t, k, p = np.full(rows, 0.8), np.full(rows, 50, np.int32), np.full(rows, 0.95)
    elif c["mode"] == "mass":
        t, p = np.full(rows, 1.0), rng.uniform(0.8, 0.99, rows)
    elif c["mode"] == "mixed":
        t = np.where(rng.random(rows) < 0.15, 0.0, t)
        k = np.where(rng.random(rows) < 0.5, rng.choice([1, 20, 40, 200, 1000], rows), 0).astype(np.int32)
        p = np.where(rng.random(rows) < 0.5, rng.uniform(0.5, 0.99, rows), 1.0)
        m = np.where(rng.random(rows) < 0.4, rng.uniform(0.01, 0.2, rows), 0.0)
    return t.astype(np.float32), k, p.astype(np.float32), m.astype(np.float32)


def _logits(c, gen):
    """A bulk of unlikely tokens, a few percent above it; in masked cases every fourth row keeps about
    half its tokens, and the row after it has others at the type's lowest value."""
    shape = (c["rows"], c["vocab"])
    z = torch.randn(shape, generator=gen, device=_DEV) * 2
    z += 10 * torch.rand(shape, generator=gen, device=_DEV) ** 24
    z = z.to(_TORCH[c["src"]])
    if c["masked"]:
        out = torch.rand(shape, generator=gen, device=_DEV) < 0.5
        z[::4] = z[::4].masked_fill(out[::4], float("-inf"))
        z[1::4] = z[1::4].masked_fill(out[1::4], torch.finfo(z.dtype).min)
    return z


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)
    dt = _TORCH[c["src"]] if "src" in c else None
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(_DEV)  # noqa: E731
    normal = lambda *shape: torch.randn(shape, generator=gen, device=_DEV)  # noqa: E731
    s = {"case": c}
    if c["kind"] == "sample":
        t, k, p, m = _sample_params(c, seed)
        s.update(logits=_logits(c, gen), u=torch.rand(c["rows"], generator=gen, device=_DEV), temperature=dev(t), top_k=dev(k),
                 top_p=dev(p), min_p=dev(m))
        return s
    if own:
        s["rotary"] = _rotary(c)
    else:
        f, s["magnitude"] = _frequencies(c)
        s["freq"] = f.to(_DEV)
    if c["kind"] == "move":
        src, dst, delta, blocks = _move_inputs(c, seed)
        s["cache"], s["pools"] = _pools(c, blocks, c["layers"], gen)
        s.update(src=dev(src), dst=dev(dst), delta=dev(delta), blocks=blocks)
        return s
    if c["kind"] == "rotate":
        pos = np.concatenate([np.arange(p, p + m) for p, m in _runs(c, random.Random(seed))]).astype(np.int32)
        s.update(x=normal(c["tokens"], c["heads"], c["dim"]).to(dt), pos=dev(pos))
        return s
    pos, slots, blocks = _append_inputs(c, seed)
    s["cache"], s["pools"] = _pools(c, blocks, 1, gen)
    n, hq, hkv, d = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    qkv = normal(n, hq + 2 * hkv, d).to(dt)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    if not c["fused"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    s.update(q=q, k=k, v=v, pos=dev(pos), slots=dev(slots), blocks=blocks)
    return s


def _turn(x, pos, freq, magnitude, layout, transpose=False):
    """x [n, ..., d] float32 rotated by its token's position."""
    angle = pos.double()[:, None] * freq
    shape = (pos.numel(),) + (1,) * (x.dim() - 2) + (freq.numel(),)
    cos = (angle.cos() * magnitude).float().view(shape)
    sin = (angle.sin() * (-magnitude if transpose else magnitude)).float().view(shape)
    rot = 2 * freq.numel()
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_sample(s):
    z = s["logits"].float()
    v = z.shape[1]
    z = torch.where(torch.isnan(z), float("-inf"), z)
    z, order = torch.sort(z, dim=1, descending=True, stable=True)
    rank = torch.arange(v, device=z.device)
    d = z.double() - z[:, :1].double()
    t = s["temperature"].double()[:, None]
    w = torch.where(t > 0, torch.exp(d / t), (rank == 0).double())
    w = torch.where(z == z[:, :1], torch.where((t > 0) | (rank == 0), 1.0, 0.0).double(), w)
    w = torch.where(torch.isinf(z) & (z < 0), 0.0, w)
    w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    k = s["top_k"][:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    c = w.cumsum(1)
    before = torch.cat((torch.zeros_like(c[:, :1]), c[:, :-1]), 1)
    kept = (w > 0) & ((before < s["top_p"].double()[:, None] * c[:, -1:]) | (rank == 0))
    count = kept.sum(1, keepdim=True)
    total = c.gather(1, (count - 1).clamp(min=0))
    at = (c <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    at = torch.minimum(at, (count - 1).clamp(min=0))
    token = torch.where(count > 0, order.gather(1, at), -1)
    prob = torch.where(count > 0, w.gather(1, at) / total, 0.0)
    return token[:, 0].int(), prob[:, 0].float()


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "sample":
        if not own:
            return _plain_sample(s)
        from infer_train_amd.sampling import sample

        return sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    if c["kind"] == "rotate":
        if own:
            return s["rotary"].apply(s["x"], s["pos"], transpose=c["transpose"])
        return _turn(s["x"].float(), s["pos"], s["freq"], s["magnitude"], c["layout"], c["transpose"]).to(s["x"].dtype)
    kp, vp = s["pools"]
    if c["kind"] == "move":
        if own:
            s["cache"].move(s["src"], s["dst"], s["rotary"] if c["rotate"] else None, s["delta"] if c["rotate"] else None)
            return kp, vp
        bs = c["block"]
        sb, so, db, do = s["src"] // bs, s["src"] % bs, s["dst"] // bs, s["dst"] % bs
        k, v = kp[:, sb, :, so], vp[:, sb, :, so]  # [rows, layers, heads, dim]
        if c["rotate"]:
            k = _turn(k.float(), s["delta"], s["freq"], 1.0, c["layout"]).to(kp.dtype)
        kp[:, db, :, do] = k
        vp[:, db, :, do] = v
        return kp[:, :s["blocks"]], vp[:, :s["blocks"]]
    if own:
        out = s["cache"].append_rotary(s["rotary"], s["q"], s["k"], s["v"], s["slots"], s["pos"])
        return out, kp, vp
    turn = lambda x: _turn(x.float(), s["pos"], s["freq"], s["magnitude"], c["layout"])  # noqa: E731
    slots = torch.where(s["slots"] < 0, s["blocks"] * c["block"], s["slots"])
    b, o = slots // c["block"], slots % c["block"]
    kp[0][b, :, o] = turn(s["k"]).to(kp.dtype)
    vp[0][b, :, o] = s["v"].to(vp.dtype)
    return turn(s["q"]).to(s["q"].dtype), kp[:, :s["blocks"]], vp[:, :s["blocks"]]


def work(case):
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * _SIZE[c["src"]] + c["rows"] * (5 * 4 + 8), "flops": 4 * n}
    if c["kind"] == "rotate":
        n = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * _SIZE[c["src"]] + 4 * c["tokens"], "flops": 3 * c["tokens"] * c["heads"] * c["rot"]}
    if c["kind"] == "move":
        rows = len(_move_inputs(c, 1)[0])
        n = rows * c["layers"] * c["kv_heads"]
        return {"bytes": 4 * n * c["dim"] * _SIZE[c["cache"]] + 20 * rows, "flops": (3 * n * c["rot"]) * c["rotate"]}
    n, live = c["tokens"], c["tokens"] - c["pad"]
    q, kv = c["heads"] * c["dim"], 2 * c["kv_heads"] * c["dim"]
    return {"bytes": 2 * n * q * _SIZE[c["src"]] + live * kv * (_SIZE[c["src"]] + _SIZE[c["cache"]]) + 12 * n,
            "flops": 3 * n * (c["heads"] + c["kv_heads"]) * c["rot"]}


def _exact_turn(x, pos, f, m, layout, transpose=False):
    """x float64 [..., heads, dim] with pos of its leading shape: a complex product per pair."""
    f, rot = f.to(x.device), 2 * f.numel()
    e = torch.polar(torch.full((), float(m), dtype=torch.float64, device=x.device),
                    pos.to(x.device, torch.float64)[..., None] * f)[..., None, :]
    if transpose:
        e = e.conj()
    y = x.clone()
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    z = torch.complex(x[..., first], x[..., second]) * e
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_sample(s):
    z = s["logits"].double().cpu().numpy()
    u, t, k, p, m = (s[n].double().cpu().numpy() for n in ("u", "temperature", "top_k", "top_p", "min_p"))
    tokens, probs = np.full(len(z), -1, np.int32), np.zeros(len(z))
    for r, row in enumerate(z):
        row = np.where(np.isnan(row), -np.inf, row)
        live = np.flatnonzero(row > -np.inf)
        if live.size == 0:
            continue
        live = live[np.argsort(-row[live], kind="stable")]
        if t[r] <= 0:
            tokens[r], probs[r] = live[0], 1.0
            continue
        w = np.exp((row[live] - row[live[0]]) / t[r])
        n = int(np.count_nonzero(w >= m[r]))
        n = max(1, min(n, int(k[r])) if k[r] > 0 else n)
        c = np.cumsum(w[:n])
        n = max(1, int(np.searchsorted(c, p[r] * c[-1], side="left")) + 1) if p[r] < 1 else n
        n = min(n, c.size)
        i = min(int(np.searchsorted(c[:n], u[r] * c[n - 1], side="right")), n - 1)
        tokens[r], probs[r] = live[i], w[i] / c[n - 1]
    return torch.from_numpy(tokens), torch.from_numpy(probs)


def exact(case, seed):
    global own
    c, was = dict(case), own
    own = False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if c["kind"] == "sample":
        return _exact_sample(s)
    f, m = _frequencies(c)
    if c["kind"] == "rotate":
        return _exact_turn(s["x"].double(), s["pos"], f, m, c["layout"], c["transpose"])
    out = [p[:, :s["blocks"]].double() for p in s["pools"]]
    flat = [p.transpose(2, 3).reshape(p.shape[0], -1, p.shape[2], p.shape[4]) for p in out]  # [layers, slots, heads, dim]
    if c["kind"] == "move":
        for i, p in enumerate(flat):
            rows = p[:, s["src"]]
            if i == 0 and c["rotate"]:
                rows = torch.stack([_exact_turn(layer, s["delta"], f, 1.0, c["layout"]) for layer in rows])
            p[:, s["dst"]] = rows
        q = None
    else:
        live = s["slots"] >= 0
        q = _exact_turn(s["q"].double(), s["pos"], f, m, c["layout"])
        flat[0][0, s["slots"][live]] = _exact_turn(s["k"].double(), s["pos"], f, m, c["layout"])[live]
        flat[1][0, s["slots"][live]] = s["v"].double()[live]
    pools = tuple(p.view(p.shape[0], s["blocks"], c["block"], c["kv_heads"], c["dim"]).transpose(2, 3) for p in flat)
    return pools if q is None else (q,) + pools
