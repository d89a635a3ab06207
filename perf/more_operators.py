"""Latent attention over a paged cache, and beam search.

Kinds of case:

  store    a step's latent rows into the cache: the latent part normalised, the
           rope key rotated, the rope part of each query head rotated;
  decode   absorbed latent attention: all query heads over one shared latent row
           a token, values the row's latent part, one or a few new tokens a
           sequence;
  prefill  expanded latent attention: a chunk's heads over keys and values that
           were projected up from the latents, one rope key shared by all heads;
  select   beam search's step: the best continuations over a group's beams and
           the vocabulary, by cumulative log-probability;
  reorder  per-beam states (block tables, token histories, recurrent states) put
           in the order of the beams that were selected.

Sizes and lengths belong to the case, values, positions and block order to the
seed of `prepare`.  Where `own` is false the operators run in their plain form,
in float32 (angles and log-probabilities in float64).
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4}
_DEV = "cuda:0"
_BASE = 10000.0
_EPS = 1e-6


def listed():
    return [
        # One user's next token: a latency-bound append of a single row and 28 query heads.
        {"name": "store_one_bf16", "kind": "store", "tokens": 1, "heads": 28, "latent": 512, "rope": 64, "src": "bf16",
         "cache": "bf16", "block": 16, "norm": True, "max_pos": 4096, "pad": 0, "rows": False},
        # Prompt chunks: rows also handed back for the projection up, the batch padded.
        {"name": "store_chunk_f16", "kind": "store", "tokens": 4001, "heads": 32, "latent": 512, "rope": 64, "src": "f16",
         "cache": "f16", "block": 16, "norm": True, "max_pos": 32768, "pad": 57, "rows": True},
        # One user over a short context.
        {"name": "decode_one_bf16", "kind": "decode", "seqs": 1, "heads": 28, "latent": 512, "rope": 64, "cache": "bf16",
         "block": 16, "q_len": 1, "lo": 1023, "hi": 1023, "empty": False},
        # A served batch of ragged contexts, 32 query heads on this device.
        {"name": "decode_batch_bf16", "kind": "decode", "seqs": 32, "heads": 32, "latent": 512, "rope": 64, "cache": "bf16",
         "block": 16, "q_len": 1, "lo": 256, "hi": 8192, "empty": True},
        # All heads of a large model on one device, long contexts.
        {"name": "decode_heads_bf16", "kind": "decode", "seqs": 16, "heads": 128, "latent": 512, "rope": 64, "cache": "bf16",
         "block": 32, "q_len": 1, "lo": 8192, "hi": 16384, "empty": False},
        # Drafted tokens checked, four a sequence, a narrower latent in float16.
        {"name": "decode_draft_f16", "kind": "decode", "seqs": 24, "heads": 12, "latent": 256, "rope": 32, "cache": "f16",
         "block": 16, "q_len": 4, "lo": 100, "hi": 4096, "empty": False},
        # A few short prompts of odd lengths, one of a single token.
        {"name": "prefill_short_f16", "kind": "prefill", "seqs": 3, "heads": 12, "nope": 64, "rope": 32, "v": 64, "src": "f16",
         "q_lo": 1, "q_hi": 250, "prefix": 0},
        # Chunks of 512 tokens after cached prefixes, 32 heads.
        {"name": "prefill_chunk_bf16", "kind": "prefill", "seqs": 8, "heads": 32, "nope": 128, "rope": 64, "v": 128,
         "src": "bf16", "q_lo": 512, "q_hi": 512, "prefix": 2048},
        # One request's beams after a token.
        {"name": "select_one_f32", "kind": "select", "groups": 1, "beams": 4, "vocab": 32000, "out": 8, "src": "f32",
         "masked": False},
        # A batch of requests with eight beams each, an odd vocabulary, grammars masking part of it.
        {"name": "select_batch_bf16", "kind": "select", "groups": 32, "beams": 8, "vocab": 100003, "out": 16, "src": "bf16",
         "masked": True},
        # The block tables of 32 requests of four beams.
        {"name": "reorder_tables_i32", "kind": "reorder", "layers": 1, "groups": 32, "beams": 4, "width": 2048, "src": "i32"},
        # Recurrent states of every layer, eight beams a request.
        {"name": "reorder_states_f32", "kind": "reorder", "layers": 28, "groups": 8, "beams": 8, "width": 65536, "src": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(("store", "decode", "decode", "decode", "prefill", "prefill", "select", "select", "reorder"))
    if kind == "select":
        beams, vocab = rng.choice((1, 2, 3, 4, 5, 8, 16)), _log(rng, 100, 200000)
        groups = _log(rng, 1, max(1, min(64, 32 * 8 * 100003 // (beams * vocab))))
        return {"kind": kind, "groups": groups, "beams": beams, "vocab": vocab, "out": beams * rng.choice((1, 2)),
                "src": rng.choice(("f32", "bf16", "f16")), "masked": rng.random() < 0.5}
    if kind == "reorder":
        layers, groups, beams = _log(rng, 1, 32), _log(rng, 1, 64), rng.choice((2, 3, 4, 5, 8, 16))
        return {"kind": kind, "layers": layers, "groups": groups, "beams": beams,
                "width": _log(rng, 16, max(17, 28 * 64 * 65536 // (layers * groups * beams))),
                "src": rng.choice(("i32", "f32", "bf16"))}
    heads = rng.choice((4, 8, 12, 16, 28, 32, 64, 128, 5, 9))
    src = rng.choice(("bf16", "bf16", "f16"))
    if kind == "prefill":
        nope, rope, v = rng.choice(((128, 64, 128), (128, 64, 128), (64, 32, 64), (128, 32, 64)))
        cap = 8 * 32 * 512 * 2304  # rows x keys x heads of the listed chunk
        hi = _log(rng, 1, 2048)
        prefix = rng.choice((0, 0, _log(rng, 1, 4096)))
        seqs = _log(rng, 1, max(1, min(24, cap // (heads * hi * (hi + prefix)))))
        return {"kind": kind, "seqs": seqs, "heads": min(heads, 32), "nope": nope, "rope": rope, "v": v, "src": src,
                "q_lo": rng.choice((1, max(1, hi // 2))), "q_hi": hi, "prefix": prefix}
    latent, rope = rng.choice(((512, 64), (512, 64), (256, 64), (256, 32)))
    c = {"kind": kind, "heads": heads, "latent": latent, "rope": rope, "block": rng.choice((8, 16, 32, 64))}
    if kind == "store":
        n = _log(rng, 1, max(1, min(8191, 4001 * 32 // heads)))
        return {**c, "tokens": n, "src": rng.choice((src, src, "f32")), "cache": src, "norm": rng.random() < 0.8,
                "max_pos": _log(rng, 8192, 1 << 20), "pad": n // rng.choice((7, 1 << 20)), "rows": rng.random() < 0.5}
    q_len = rng.choice((1, 1, 1, 2, 3, 5))
    hi = _log(rng, 8, 32768)
    seqs = _log(rng, 1, max(1, min(128, 16 * 128 * 12288 // (max(heads * q_len, 32) * hi))))
    return {**c, "cache": src, "seqs": seqs, "q_len": q_len, "lo": rng.choice((q_len, max(q_len, hi // 2))), "hi": max(hi, q_len),
            "empty": rng.random() < 0.3}


def _id(name):
    import infer_train_amd as it

    return {"f32": it.F32, "f16": it.F16, "bf16": it.BF16}[name]


def _frequencies(rope):
    i = torch.arange(rope // 2, dtype=torch.float64)
    return _BASE ** (-2.0 * i / rope)


def _contexts(c):
    """Context length of every sequence, the new tokens counted."""
    rng = random.Random(c["seqs"] * 1000003 + c["hi"])
    lens = [rng.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]
    if c["empty"]:  # a slot of the batch that holds no request
        lens[len(lens) // 2] = 0
    return lens


def _chunks(c):
    """Query rows and keys of every sequence."""
    rng = random.Random(c["seqs"] * 1000003 + c["q_hi"])
    q = [rng.randint(c["q_lo"], c["q_hi"]) for _ in range(c["seqs"])]
    if c["q_lo"] == 1:
        q[-1] = 1
    return q, [n + (rng.randint(c["prefix"] // 2, c["prefix"]) if c["prefix"] else 0) for n in q]


def _cu(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=_DEV)


def _cache(c, blocks):
    from infer_train_amd.latent import LatentKvCache

    cache = LatentKvCache(blocks, c["block"], c["latent"], c["rope"], _id(c["cache"]))
    return cache, cache.view()


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(_DEV)  # noqa: E731
    normal = lambda *shape: torch.randn(shape, generator=gen, device=_DEV)  # noqa: E731
    s = {"case": c}
    if c["kind"] == "select":
        rows, dt = c["groups"] * c["beams"], _TORCH[c["src"]]
        z = normal(rows, c["vocab"]) * 2
        z += 10 * torch.rand(z.shape, generator=gen, device=_DEV) ** 24
        z = z.to(dt)
        if c["masked"]:  # a grammar takes half the tokens out, by -inf or by the type's lowest value
            out = torch.rand(z.shape, generator=gen, device=_DEV) < 0.5
            z[::4] = z[::4].masked_fill(out[::4], float("-inf"))
            z[1::4] = z[1::4].masked_fill(out[1::4], torch.finfo(dt).min)
        scores = -20 * torch.rand((c["groups"], c["beams"]), generator=gen, device=_DEV)
        if c["masked"] and c["beams"] > 1:
            scores[::3, -1] = float("-inf")  # a beam that is not in use
        s.update(logits=z, scores=scores)
        return s
    if c["kind"] == "reorder":
        shape = (c["layers"], c["groups"] * c["beams"], c["width"])
        s["x"] = (dev(rng.integers(0, 1 << 20, shape, dtype=np.int32)) if c["src"] == "i32" else normal(*shape).to(_TORCH[c["src"]]))
        s["parents"] = dev(rng.integers(0, c["beams"], (c["groups"], c["beams"])).astype(np.int32))
        return s
    if c["kind"] == "prefill":
        q, k = _chunks(c)
        dt, h = _TORCH[c["src"]], c["heads"]
        kv = normal(sum(k), h, c["nope"] + c["v"]).to(dt)  # one projection's keys and values
        rows = normal(sum(k), 512 + c["rope"]).to(dt)      # the latent rows, rope key last
        s.update(q=normal(sum(q), h, c["nope"] + c["rope"]).to(dt), k=kv[..., :c["nope"]], v=kv[..., c["nope"]:],
                 k_rope=rows[:, 512:], cu_q=_cu(q), cu_k=_cu(k), scale=1.0 / math.sqrt(c["nope"] + c["rope"]))
        return s
    dt, row, bs = _TORCH[c["cache"]], c["latent"] + c["rope"], c["block"]
    if c["kind"] == "store":
        n, src = c["tokens"], _TORCH[c["src"]]
        blocks = -(-n // bs) + 3
        start = int(rng.integers(0, max(1, c["max_pos"] - n)))
        slots = rng.permutation(blocks)[(np.arange(n) + start % bs) // bs] * bs + (np.arange(n) + start) % bs
        if c["pad"]:
            slots[n - c["pad"]:] = -1
        q = normal(n, c["heads"], 128 + c["rope"]).to(src)
        s.update(kv=normal(n, row).to(src) * 3, q=q, q_rope=q[..., 128:], slots=dev(slots.astype(np.int64)),
                 pos=dev(np.arange(start, start + n, dtype=np.int32)),
                 weight=(1 + 0.2 * normal(c["latent"])).to(src) if c["norm"] else None)
        if own:
            import infer_train_amd.kv as kv

            s["cache"], s["pool"] = _cache(c, blocks)
            s["rotary"] = kv.Rotary(c["rope"], layout="interleaved", freq_base=_BASE)
        else:
            s["pool"] = torch.zeros(blocks + 1, bs, row, dtype=dt, device=_DEV)  # the last block takes the padding's rows
            s["freq"] = _frequencies(c["rope"]).to(_DEV)
        s["pool"][:blocks].copy_(normal(blocks, bs, row))
        s["blocks"] = blocks
        return s
    lens, t = _contexts(c), c["q_len"]
    held = [-(-n // bs) for n in lens]
    blocks = sum(held) + 2
    order, at = rng.permutation(blocks), 0
    tables = np.full((len(lens), max(held) + 1), -1, np.int32)
    for i, m in enumerate(held):
        tables[i, :m], at = order[at:at + m], at + m
    if own:
        s["cache"], s["pool"] = _cache(c, blocks)
    else:
        s["pool"] = torch.zeros(blocks, bs, row, dtype=dt, device=_DEV)
    for i in range(0, blocks, 4096):
        s["pool"][i:i + 4096].copy_(normal(min(4096, blocks - i), bs, row))
    q = normal(len(lens) * t, c["heads"], row).to(dt)
    s.update(q=q, tables=dev(tables), lens=dev(np.array(lens, np.int32)), longest=max(lens), scale=1.0 / math.sqrt(128 + c["rope"]))
    if own:
        s["ws"] = s["cache"].decode_workspace(len(lens), c["heads"], max(lens), q_len=t)
    return s


def _turn(x, pos, freq):
    """x [n, ..., 2 pairs] float32, interleaved pairs rotated by the token's position."""
    angle = (pos.double()[:, None] * freq).view((pos.numel(),) + (1,) * (x.dim() - 2) + (freq.numel(),))
    cos, sin = angle.cos().float(), angle.sin().float()
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _softmax(s):
    """Probabilities of the last axis; rows without a key are 0."""
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).min) if s.shape[-1] else s.sum(-1, keepdim=True)
    e = torch.exp(s - m)
    return e / e.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_store(s, c):
    kv = s["kv"].float()
    latent, rope = kv[:, :c["latent"]], kv[:, c["latent"]:]
    if s["weight"] is not None:
        latent = latent * torch.rsqrt((latent * latent).mean(-1, keepdim=True) + _EPS) * s["weight"].float()
    row = torch.cat((latent, _turn(rope, s["pos"], s["freq"])), -1).to(s["pool"].dtype)
    slots = torch.where(s["slots"] < 0, s["blocks"] * c["block"], s["slots"])
    s["pool"].view(-1, row.shape[1])[slots] = row
    q = _turn(s["q_rope"].float(), s["pos"], s["freq"]).to(s["q"].dtype)
    return (q, s["pool"][:s["blocks"]]) + ((row,) if c["rows"] else ())


def _plain_decode(s, c):
    t, bs, lat = c["q_len"], c["block"], c["latent"]
    out = torch.zeros(s["q"].shape[0], c["heads"], lat, device=_DEV)
    for i, n in enumerate(_contexts(c)):
        if n == 0:
            continue
        rows = s["pool"][s["tables"][i, :-(-n // bs)].long()].reshape(-1, lat + c["rope"])[:n].float()
        q = s["q"][i * t:(i + 1) * t].float()
        score = (q.reshape(-1, rows.shape[1]) @ rows.t() * s["scale"]).view(t, c["heads"], n)
        if t > 1:
            hidden = torch.arange(n, device=_DEV)[None] > n - t + torch.arange(t, device=_DEV)[:, None]
            score = score.masked_fill(hidden[:, None], float("-inf"))
        out[i * t:(i + 1) * t] = (_softmax(score).view(-1, n) @ rows[:, :lat]).view(t, c["heads"], lat)
    return out.to(s["q"].dtype)


def _plain_prefill(s, c):
    out = torch.empty(s["q"].shape[0], c["heads"], c["v"], device=_DEV)
    qs, ks = _chunks(c)
    at_q = at_k = 0
    for nq, nk in zip(qs, ks):
        q = s["q"][at_q:at_q + nq].float().transpose(0, 1).contiguous()
        k = torch.cat((s["k"][at_k:at_k + nk].float(), s["k_rope"][at_k:at_k + nk].float()[:, None].expand(-1, c["heads"], -1)), -1)
        v = s["v"][at_k:at_k + nk].float().transpose(0, 1).contiguous()
        score = torch.matmul(q, k.permute(1, 2, 0).contiguous()) * s["scale"]
        hidden = torch.arange(nk, device=_DEV)[None] > nk - nq + torch.arange(nq, device=_DEV)[:, None]
        out[at_q:at_q + nq] = torch.matmul(_softmax(score.masked_fill(hidden, float("-inf"))), v).transpose(0, 1)
        at_q, at_k = at_q + nq, at_k + nk
    return out.to(s["q"].dtype)


def _plain_select(s, c):
    g, b, v = c["groups"], c["beams"], c["vocab"]
    z = s["logits"].double().view(g, b, v)
    top = z.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float64).min)
    lse = top + torch.log(torch.exp(z - top).sum(-1, keepdim=True))
    value = (s["scores"].double()[..., None] - lse) + z
    value = torch.where((z == -math.inf) | (s["scores"][..., None] == -math.inf), -math.inf, value).view(g, b * v)
    best, at = torch.sort(value, dim=1, descending=True, stable=True)
    n = min(c["out"], b * v)
    best, at = best[:, :n], at[:, :n]
    dead = best == -math.inf
    return best.float(), torch.where(dead, -1, at // v).int(), torch.where(dead, -1, at % v).int()


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "reorder":
        if own:
            from infer_train_amd.beam import beam_reorder

            return beam_reorder(s["x"], s["parents"], dim=1)
        rows = (s["parents"] + torch.arange(c["groups"], device=_DEV)[:, None] * c["beams"]).flatten()
        s["x"].copy_(s["x"][:, rows])
        return s["x"]
    if kind == "select":
        if not own:
            return _plain_select(s, c)
        from infer_train_amd.beam import beam_select

        return beam_select(s["logits"], s["scores"], c["out"])
    if kind == "prefill":
        if not own:
            return _plain_prefill(s, c)
        from infer_train_amd.latent import latent_prefill

        qs, ks = _chunks(c)
        return latent_prefill(s["q"], s["k"], s["v"], s["k_rope"], s["cu_q"], s["cu_k"], max(qs), max(ks), s["scale"])
    if kind == "decode":
        if not own:
            return _plain_decode(s, c)
        lat = c["latent"]
        return s["cache"].decode(s["q"][..., :lat], s["q"][..., lat:], s["tables"], s["lens"], s["longest"], s["scale"],
                                 q_len=c["q_len"], ws=s["ws"])
    if not own:
        return _plain_store(s, c)
    rows = torch.empty(c["tokens"], c["latent"] + c["rope"], dtype=s["pool"].dtype, device=_DEV) if c["rows"] else None
    q = s["cache"].append(s["kv"], s["slots"], s["rotary"], s["pos"], weight=s["weight"], eps=_EPS, q_rope=s["q_rope"],
                          rows_out=rows)
    return (q, s["pool"]) + ((rows,) if c["rows"] else ())


def work(case):
    c = case
    if c["kind"] == "reorder":
        n = c["layers"] * c["groups"] * c["beams"] * c["width"]
        return {"bytes": 2 * n * _SIZE[c["src"]] + 4 * c["groups"] * c["beams"], "flops": 0}
    if c["kind"] == "select":
        n = c["groups"] * c["beams"] * c["vocab"]
        return {"bytes": n * _SIZE[c["src"]] + c["groups"] * (4 * c["beams"] + 12 * c["out"]), "flops": 4 * n}
    if c["kind"] == "prefill":
        q, k = _chunks(c)
        pairs = sum(nq * nk - nq * (nq - 1) // 2 for nq, nk in zip(q, k))
        h, qk = c["heads"], c["nope"] + c["rope"]
        return {"bytes": _SIZE[c["src"]] * (sum(q) * h * (qk + c["v"]) + sum(k) * (h * (c["nope"] + c["v"]) + c["rope"])),
                "flops": 2 * pairs * h * (qk + c["v"])}
    row = c["latent"] + c["rope"]
    if c["kind"] == "store":
        n, live = c["tokens"], c["tokens"] - c["pad"]
        src, dst = _SIZE[c["src"]], _SIZE[c["cache"]]
        return {"bytes": n * row * (src + dst * c["rows"]) + live * row * dst + 2 * n * c["heads"] * c["rope"] * src + 12 * n,
                "flops": n * (4 * c["latent"] * c["norm"] + 3 * (c["heads"] + 1) * c["rope"])}
    lens, t = _contexts(c), c["q_len"]
    return {"bytes": 2 * (sum(lens) * row + c["seqs"] * t * c["heads"] * (row + c["latent"])),
            "flops": 2 * sum(t * n - t * (t - 1) // 2 for n in lens if n) * c["heads"] * (row + c["latent"])}


def _exact_rotation(x, pos, rope):
    """x float64 [n, ..., rope] as complex numbers times exp(i position f)."""
    angle = pos.double().view((-1,) + (1,) * (x.dim() - 1)) * _frequencies(rope).to(x.device)
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * torch.polar(torch.ones_like(angle), angle)
    return torch.view_as_real(z).flatten(-2)


def _exact_attention(q, k, v, scale, causal_rows):
    """One head: q [m, d], k [n, d], v [n, e] float64; causal_rows: row i sees the keys before n - m + 1 + i."""
    m, n = q.shape[0], k.shape[0]
    z = (q * scale) @ k.t().contiguous()
    if causal_rows:
        z = z.tril(n - m) + torch.full_like(z, -math.inf).triu(n - m + 1)
    return torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) @ v


def exact(case, seed):
    global own
    c, was = dict(case), own
    own = False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if c["kind"] == "reorder":
        x = s["x"].view(c["layers"], c["groups"], c["beams"], c["width"])
        index = s["parents"].long()[None, :, :, None].expand(x.shape)
        return torch.gather(x, 2, index).view(s["x"].shape)
    if c["kind"] == "select":
        z, beam_scores = s["logits"].double().cpu().numpy(), s["scores"].double().cpu().numpy()
        z = z.reshape(c["groups"], c["beams"], -1)
        n = min(c["out"], c["beams"] * c["vocab"])
        score, parent, token = (np.full((c["groups"], n), x) for x in (-np.inf, -1, -1))
        for g in range(c["groups"]):
            best = []
            for b in range(c["beams"]):
                row = z[g, b]
                live = np.flatnonzero(row > -np.inf)
                if live.size == 0 or beam_scores[g, b] == -np.inf:
                    continue
                log_sum = row.max() + math.log(math.fsum(np.exp(row[live] - row.max()).tolist()))
                for i in live[np.argsort(-row[live], kind="stable")[:n]]:
                    best.append((-(beam_scores[g, b] - log_sum + row[i]), b, int(i)))
            for j, (value, b, i) in enumerate(sorted(best)[:n]):
                score[g, j], parent[g, j], token[g, j] = -value, b, i
        return torch.from_numpy(score), torch.from_numpy(parent.astype(np.int32)), torch.from_numpy(token.astype(np.int32))
    if c["kind"] == "prefill":
        out, at_q, at_k = [], 0, 0
        for nq, nk in zip(*_chunks(c)):
            heads = []
            for h in range(c["heads"]):
                q = s["q"][at_q:at_q + nq, h].double()
                k = torch.cat((s["k"][at_k:at_k + nk, h], s["k_rope"][at_k:at_k + nk]), 1).double()
                heads.append(_exact_attention(q, k, s["v"][at_k:at_k + nk, h].double(), s["scale"], True))
            out.append(torch.stack(heads, 1))
            at_q, at_k = at_q + nq, at_k + nk
        return torch.cat(out)
    if c["kind"] == "decode":
        t, flat, out = c["q_len"], s["pool"].flatten(0, 1), []
        for i, n in enumerate(_contexts(c)):
            at = torch.arange(n, device=_DEV)
            rows = flat[s["tables"][i][at // c["block"]].long() * c["block"] + at % c["block"]].double()
            for j in range(t):
                seen = rows[:n - t + 1 + j] if n else rows
                q = s["q"][i * t + j].double()
                out.append(_exact_attention(q, seen, seen[:, :c["latent"]], s["scale"], False) if n else
                           torch.zeros(c["heads"], c["latent"], dtype=torch.float64, device=_DEV))
        return torch.stack(out)
    kv, lat = s["kv"].double(), c["latent"]
    x = kv[:, :lat]
    if s["weight"] is not None:
        x = x / torch.sqrt(x.square().sum(1, keepdim=True) / lat + _EPS) * s["weight"].double()
    row = torch.cat((x, _exact_rotation(kv[:, lat:], s["pos"], c["rope"])), 1)
    pool = s["pool"][:s["blocks"]].double()
    live = s["slots"] >= 0
    pool.view(-1, row.shape[1])[s["slots"][live]] = row[live]
    return (_exact_rotation(s["q_rope"].double(), s["pos"], c["rope"]), pool) + ((row,) if c["rows"] else ())
