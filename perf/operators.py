"""What the streaming operators cost: rotary positions of several axes, attention to states of another
length, and the 8-bit key / value cache with the attention that reads it.

A program that streams frames (or decodes tokens) through transformer blocks rotates the new queries and
keys by their (time, height, width) positions, appends the new keys and values to the cache of the earlier
ones, lets the new queries attend to the cache, and lets decoder queries attend to the states of an encoder.
The four kinds of case are these four calls:

* ``rope``: ``rope_axes`` on the query and key heads of some tokens.
* ``cross``: ``cross_attention``, queries and keys of different lengths, optionally a key mask per sequence.
* ``append``: ``Int8KVCache.append``: quantise new keys and values into blocks of 64 tokens, one scale for each
  block and head; then ``values`` of every block that the call wrote.
* ``cached``: ``Int8KVCache.attention``: new queries over the cache, optionally causal.

``run`` computes each with elementary torch operations where ``own`` is false, and with the package's kernels
where it is true; ``exact`` is the operators' definition in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TOKENS = 1374        # tokens of one frame
BLOCK = 64           # tokens of a cache block
SCORES = 1 << 28     # scores that the plain forms hold at a time

F16, BF16 = "float16", "bfloat16"


def listed():
    return [
        # one new token of each of 16 sequences, far positions: launch latency
        dict(name="rope_step", kind="rope", tokens=16, heads=24, dim=128, dtype=BF16, layout="half", sections="32 48 48",
             far=100000),
        # the q and k heads of one frame
        dict(name="rope_frame", kind="rope", tokens=TOKENS, heads=32, dim=64, dtype=F16, layout="block", sections="16 24 24",
             far=40),
        # the q and k heads of 32 frames at once: bandwidth
        dict(name="rope_32_frames", kind="rope", tokens=32 * TOKENS, heads=32, dim=64, dtype=F16, layout="block",
             sections="16 24 24", far=40),
        # one query token of each of 8 sequences against one frame's states: latency
        dict(name="cross_step", kind="cross", batch=8, queries=1, keys=TOKENS, heads=16, kv_heads=16, dim=64, dtype=F16,
             masked=False),
        # a padded batch with a key mask, shared key heads, odd lengths, wide heads
        dict(name="cross_ragged", kind="cross", batch=4, queries=333, keys=1501, heads=16, kv_heads=4, dim=128, dtype=BF16,
             masked=True),
        # the tokens of one frame against the states of eight
        dict(name="cross_8_frames", kind="cross", batch=1, queries=TOKENS, keys=8 * TOKENS, heads=16, kv_heads=16, dim=64,
             dtype=F16, masked=False),
        # one new token of each of 32 sequences, somewhere inside a block
        dict(name="append_step", kind="append", batch=32, new=1, past=500, kv_heads=8, dim=128, dtype=BF16, ragged=False),
        # one frame behind two others, its first block half full
        dict(name="append_frame", kind="append", batch=1, new=TOKENS, past=2 * TOKENS, kv_heads=16, dim=64, dtype=F16,
             ragged=False),
        # prompts of a padded batch into an empty cache
        dict(name="append_prompts", kind="append", batch=8, new=2900, past=0, kv_heads=8, dim=128, dtype=F16, ragged=True),
        # a decode step of 16 sequences of up to 8000 tokens: the cache's bytes
        dict(name="cached_step", kind="cached", batch=16, queries=1, past=8000, heads=32, kv_heads=8, dim=128, dtype=BF16,
             causal=True),
        # a chunk of a prompt behind what is cached
        dict(name="cached_chunk", kind="cached", batch=2, queries=517, past=5500, heads=16, kv_heads=4, dim=128, dtype=F16,
             causal=True),
        # one new frame against 32 cached ones, itself among them: the largest
        dict(name="cached_32_frames", kind="cached", batch=1, queries=TOKENS, past=31 * TOKENS, heads=16, kv_heads=16, dim=64,
             dtype=F16, causal=False),
    ]


def _sections(case):
    """Dims that rotate by each axis."""
    return tuple(int(n) for n in case["sections"].split())


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv = rng.choice((1, 2, 4, 5, 8, 12, 16))
    return kv * rng.choice((1, 1, 2, 3, 4, 8) if kv <= 5 else (1, 1, 2, 4) if kv <= 8 else (1, 2)), kv


def draw(rng):
    kind = rng.choice(("rope", "cross", "cross", "append", "append", "cached", "cached", "cached"))
    dtype = rng.choice((F16, F16, BF16))
    dim = rng.choice((64, 128))
    if kind == "rope":
        heads = rng.choice((1, 3, 8, 18, 24, 32))
        layout = rng.choice(("block", "half"))
        sections = rng.choice({64: ("16 24 24", "32 32", "64", "10 26 28", "12 20 20"),
                               128: ("32 48 48", "64 64", "16 56 56", "22 50 56", "128")}[dim])
        return dict(kind=kind, tokens=_log(rng, 1, 32 * TOKENS * 2048 // (heads * dim)), heads=heads, dim=dim, layout=layout,
                    dtype=rng.choice((F16, BF16, "float32")) if heads <= 8 else dtype, sections=sections,
                    far=rng.choice((40, 5000, 1000000)))
    heads, kv = _heads(rng)
    if kind == "append":
        new = 1 if rng.random() < 0.3 else _log(rng, 1, 8 * TOKENS)
        batch = rng.randint(1, max(1, min(48, 16 * TOKENS * 1024 // (new * kv * dim))))
        return dict(kind=kind, batch=batch, new=new, past=rng.choice((0, _log(rng, 1, 3000))), kv_heads=kv, dim=dim, dtype=dtype,
                    ragged=batch > 1 and rng.random() < 0.6)
    queries = 1 if rng.random() < 0.35 else _log(rng, 1, 2 * TOKENS)
    keys = _log(rng, 1 if kind == "cross" else max(1, queries), 32 * TOKENS)
    # at most a third of the largest listed case's products, and of the largest cache
    most = min(TOKENS * 32 * TOKENS * 16 * 64 // (3 * queries * keys * heads * dim), 16 * 8000 * 8 * 128 // (keys * kv * dim))
    if most < 1:
        keys = max(1, min(32 * TOKENS * 64 // (queries * dim), 16 * 8000 * 8 * 128 // (2 * kv * dim)))
        heads = kv = min(kv, 5)
        queries = min(queries, keys)
    batch = rng.randint(1, max(1, min(32, most)))
    if kind == "cross":
        return dict(kind=kind, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv, dim=dim, dtype=dtype,
                    masked=rng.random() < 0.5)
    return dict(kind=kind, batch=batch, queries=queries, past=max(0, keys - queries), heads=heads, kv_heads=kv, dim=dim,
                dtype=dtype, causal=rng.random() < 0.6)


# ------------------------------------------------------- inputs from a seed
def _lens(case, gen, most, least=1):
    """Tokens of each sequence, the longest ``most``."""
    n = case["batch"]
    lens = (least + (most - least) * torch.rand(n, generator=gen)).round().int()
    lens[int(torch.randint(n, (1,), generator=gen))] = most
    return lens


def _states(gen, dev, shape, dtype, spread=0.25):
    """Keys or values: unit normal, the channels of a head of different sizes."""
    chan = torch.exp(spread * torch.randn(shape[-2:], generator=gen, device=dev))
    return (torch.randn(shape, generator=gen, device=dev) * chan).to(dtype)


def _scale(amax):
    """The smallest number of four significant bits that is at least amax / 127 (0 for 0)."""
    m, e = torch.frexp(amax.double() / 127)
    power = ((e.long() + 1023) << 52).view(torch.float64)      # 2 ** e, exactly: pow and exp2 round
    return torch.ceil(m * 16) / 16 * power


def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    dtype = getattr(torch, case["dtype"])
    gen = torch.Generator(device=dev).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    d, kind = case["dim"], case["kind"]
    st = dict(case=case)
    if kind == "rope":
        t = case["tokens"]
        st["x"] = _states(gen, dev, (t, case["heads"], d), dtype)
        st["positions"] = torch.randint(0, case["far"], (t, len(_sections(case))), generator=gen, device=dev, dtype=torch.int32)
        return st
    b, hk = case["batch"], case["kv_heads"]
    if kind == "cross":
        st["q"] = torch.randn(b, case["queries"], case["heads"], d, generator=gen, device=dev).to(dtype)
        st["k"] = _states(gen, dev, (b, case["keys"], hk, d), dtype)
        st["v"] = _states(gen, dev, (b, case["keys"], hk, d), dtype)
        st["mask"] = None
        if case["masked"]:
            # each sequence padded behind its length, single tokens left out before it
            lens = _lens(case, cpu, case["keys"]).to(dev)
            keep = torch.rand(b, case["keys"], generator=gen, device=dev) > 0.05
            st["mask"] = keep & (torch.arange(case["keys"], device=dev) < lens[:, None])
        return st
    if kind == "append":
        new, past = case["new"], case["past"]
        start = _lens(case, cpu, past, min(past, 1)) if past else torch.zeros(b, dtype=torch.int32)
        counts = _lens(case, cpu, new) if case["ragged"] else torch.full((b,), new, dtype=torch.int32)
        st["k"] = _states(gen, dev, (b, new, hk, d), dtype, 0.5)
        st["v"] = _states(gen, dev, (b, new, hk, d), dtype)
        # what the cache holds of earlier tokens, from the block that the first new token falls into on
        first = start // BLOCK * BLOCK
        st["window"] = int(((start - first) + counts).max() + BLOCK - 1) // BLOCK * BLOCK
        st["start"], st["counts"], st["first"] = start.to(dev), counts.to(dev) if case["ragged"] else None, first.to(dev)
        old = (torch.arange(BLOCK) < (start - first)[:, None]).to(dev)
        for name, spread in (("k", 0.5), ("v", 0.25)):
            x = _states(gen, dev, (b, BLOCK, hk, d), dtype, spread).double() * old[..., None, None]
            s = _scale(x.abs().amax((1, 3)))                                            # (B, Hk)
            st[name + "_scale"] = s.float()
            st[name + "_code"] = torch.round(x / torch.where(s > 0, s, 1)[:, None, :, None]).to(torch.int8)
        st["capacity"] = past + new + BLOCK
        return st
    n, total = case["queries"], case["past"] + case["queries"]
    lens = _lens(case, cpu, total, n)
    blocks = -(-total // BLOCK)
    st["q"] = torch.randn(b, n, case["heads"], d, generator=gen, device=dev).to(dtype)
    st["lens"] = lens.to(dev)
    live = (torch.arange(blocks * BLOCK, device=dev) < st["lens"][:, None])[..., None, None]
    for name, spread in (("k", 0.25), ("v", 0.25)):
        # sequence by sequence: the codes of a long cache, made in one piece, would take many times its size
        codes, scales = [], []
        for i in range(b):
            x = (_states(gen, dev, (blocks * BLOCK, hk, d), dtype, spread) * live[i]).view(blocks, BLOCK, hk, d)
            s = _scale(x.abs().amax((1, 3)))                                            # (blocks, Hk)
            codes.append(torch.round(x.double() / torch.where(s > 0, s, 1)[:, None, :, None]).to(torch.int8))
            scales.append(s.float())
        st[name + "_code"] = torch.stack(codes).view(b, blocks * BLOCK, hk, d)
        st[name + "_scale"] = torch.stack(scales)                                       # (B, blocks, Hk)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if not own:
        return st
    if case["kind"] == "rope":
        from qvggt_amd import awq_inference_engine as engine
        st["plan"] = engine.rope_axes_plan(case["dim"], _sections(case), base=100.0, layout=case["layout"],
                                           device=st["x"].device)
    elif case["kind"] == "append":
        from qvggt_amd.kv_cache import Int8KVCache
        cache = Int8KVCache(case["batch"], case["kv_heads"], case["dim"], st["capacity"], device=st["k"].device)
        codes, scales = {}, {}
        for name in ("k", "v"):      # the block that the first new token falls into
            codes[name] = torch.zeros(case["batch"], cache.capacity, case["kv_heads"], case["dim"], dtype=torch.int8,
                                      device=st["k"].device)
            scales[name] = torch.zeros(case["batch"], cache.capacity // BLOCK, case["kv_heads"], device=st["k"].device)
            for i, at in enumerate(st["first"].tolist()):
                codes[name][i, at:at + BLOCK] = st[name + "_code"][i]
                scales[name][i, at // BLOCK] = st[name + "_scale"][i]
        cache.load_codes(codes["k"], scales["k"], codes["v"], scales["v"], st["start"])
        st["cache"] = cache
    elif case["kind"] == "cached":
        from qvggt_amd.kv_cache import Int8KVCache
        cache = Int8KVCache(case["batch"], case["kv_heads"], case["dim"], st["k_code"].shape[1], device=st["q"].device)
        cache.load_codes(st["k_code"], st["k_scale"], st["v_code"], st["v_scale"], st["lens"])
        st["cache"] = cache
    return st


# ---------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from qvggt_amd import awq_inference_engine as engine
        if kind == "rope":
            return engine.rope_axes(st["x"], st["positions"], st["plan"])
        if kind == "cross":
            return engine.cross_attention(st["q"], st["k"], st["v"], key_mask=st["mask"])
        cache = st["cache"]
        if kind == "append":
            cache.append(st["k"], st["v"], counts=st["counts"], start=st["start"])
            return (*cache.values(st["window"], first=st["first"]), cache.lens)
        return cache.attention(st["q"], causal=case["causal"])
    if kind == "rope":
        return _plain_rope(st, case)
    if kind == "cross":
        return _plain_cross(st, case)
    if kind == "append":
        return _plain_append(st, case)
    return _plain_cached(st, case)


def _pairs(case):
    """For each rotated pair its two dims, its axis and its angle per position."""
    sec = _sections(case)
    rot = sum(sec)
    out, at = [], 0
    for axis, n in enumerate(sec):
        for i in range(n // 2):
            if case["layout"] == "block":
                out.append((at + i, at + n // 2 + i, axis, 100.0 ** (-2.0 * i / n)))
            else:
                j = at // 2 + i
                out.append((j, rot // 2 + j, axis, 100.0 ** (-2.0 * j / rot)))
        at += n
    return out


def _plain_rope(st, case):
    x, pos = st["x"], st["positions"]
    lo, hi, axis, theta = zip(*_pairs(case))
    ang = pos.double()[:, list(axis)] * torch.tensor(theta, dtype=torch.float64, device=x.device)
    c, s = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
    lo, hi = list(lo), list(hi)
    a, b = x[..., lo].float(), x[..., hi].float()
    y = x.clone()
    y[..., lo] = (a * c - b * s).to(x.dtype)
    y[..., hi] = (b * c + a * s).to(x.dtype)
    return y


def _softmax_rows(s, keep):
    """Softmax over the last dim of the scores where ``keep``; rows with nothing kept are zero."""
    if keep is not None:
        s = s.masked_fill(~keep, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m.isinf(), 0, m))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _attend(q, k, v, keep_of, scale):
    """q (B, Lq, H, D); k and v (B, Lk, Hk, D); keep_of(b, first, last): the mask of query rows first..last or None."""
    out = torch.empty_like(q)
    n, group = q.shape[1], q.shape[2] // k.shape[2]
    for b in range(q.shape[0]):
        kb = k[b].permute(1, 2, 0).float().contiguous()     # (Hk, D, Lk)
        vb = v[b].transpose(0, 1).float().contiguous()      # (Hk, Lk, D)
        rows = max(1, SCORES // (q.shape[2] * k.shape[1]))
        for r in range(0, n, rows):
            e = min(n, r + rows)
            qb = q[b, r:e].float().view(e - r, k.shape[2], group, -1).permute(1, 2, 0, 3)
            qb = qb.reshape(k.shape[2], group * (e - r), -1)
            s = (torch.matmul(qb, kb) * scale).view(k.shape[2], group, e - r, -1)
            p = _softmax_rows(s, keep_of(b, r, e)).view(k.shape[2], group * (e - r), -1)
            o = torch.matmul(p, vb).view(k.shape[2], group, e - r, -1).permute(2, 0, 1, 3)
            out[b, r:e] = o.reshape(e - r, q.shape[2], -1).to(q.dtype)
    return out


def _plain_cross(st, case):
    mask = st["mask"]
    return _attend(st["q"], st["k"], st["v"], lambda b, r, e: None if mask is None else mask[b], case["dim"] ** -0.5)


def _plain_append(st, case):
    start, first, w = st["start"], st["first"], st["window"]
    new = st["k"].shape[1]
    counts = st["counts"] if st["counts"] is not None else torch.full_like(start, new)
    pos = first[:, None] + torch.arange(w, device=start.device)
    is_old = (pos < start[:, None])[..., None, None]
    is_new = ((pos >= start[:, None]) & (pos < (start + counts)[:, None]))[..., None, None]
    at = (pos - start[:, None]).clamp(0, new - 1).long()
    outs = []
    for name in ("k", "v"):
        x = st[name]
        b, _, hk, d = x.shape
        got = torch.gather(x, 1, at[..., None, None].expand(b, w, hk, d))
        got = torch.where(is_new, got.float(), 0)
        was = (st[name + "_code"].float() * st[name + "_scale"][:, None, :, None])       # (B, 64, Hk, D)
        s = _scale(got.view(b, w // BLOCK, BLOCK, hk, d).abs().amax((2, 4)))             # (B, blocks, Hk)
        s[:, 0] = torch.maximum(s[:, 0], st[name + "_scale"].double())
        got[:, :BLOCK] = torch.where(is_old[:, :BLOCK], was, got[:, :BLOCK])
        by = torch.where(s > 0, s, 1).repeat_interleave(BLOCK, 1)[..., None]
        outs.append((torch.round(got.double() / by) * by).float())
    return (*outs, start + counts)


def _plain_cached(st, case):
    total = st["k_code"].shape[1]
    n = case["queries"]
    k, v = ((st[x + "_code"].float().view(case["batch"], -1, BLOCK, case["kv_heads"], case["dim"])
             * st[x + "_scale"][:, :, None, :, None]).view(st[x + "_code"].shape) for x in ("k", "v"))
    key = torch.arange(total, device=k.device)

    def keep(b, r, e):
        if not case["causal"]:
            return key < st["lens"][b]
        return key <= (st["lens"][b] - n + torch.arange(r, e, device=k.device))[:, None]

    return _attend(st["q"], k, v, keep, case["dim"] ** -0.5)


# ------------------------------------------------ what a pass cannot do without
def _size(case):
    return {"float16": 2, "bfloat16": 2, "float32": 4}[case["dtype"]]


def work(case):
    kind, d, es = case["kind"], case["dim"], _size(case)
    if kind == "rope":
        n = case["tokens"] * case["heads"] * d
        return {"bytes": 2 * n * es + 4 * case["tokens"] * len(_sections(case)), "flops": 3 * n}
    b, hk = case["batch"], case["kv_heads"]
    if kind == "cross":
        rows, keys = b * case["queries"] * case["heads"], case["keys"]
        share = 0.5 if case["masked"] and b > 1 else 1.0      # sequences end anywhere
        return {"bytes": (2 * rows * d + 2 * b * keys * share * hk * d) * es + (b * keys if case["masked"] else 0),
                "flops": 4 * rows * keys * share * d}
    if kind == "append":
        n = 2 * b * case["new"] * (0.5 if case["ragged"] else 1.0) * hk * d
        # new values read, codes written; then codes read and values written
        return {"bytes": n * (es + 1) + n * 5, "flops": 4 * n}
    rows, keys = b * case["queries"] * case["heads"], case["past"] + case["queries"]
    mean = keys if b == 1 else (keys + case["queries"]) / 2
    seen = mean - (case["queries"] - 1) / 2 if case["causal"] else mean
    return {"bytes": 2 * rows * d * es + 2 * b * mean * hk * d + 8 * b * mean / BLOCK * hk, "flops": 4 * rows * seen * d}


# ------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    st = _inputs(case, seed)
    kind = case["kind"]
    if kind == "rope":
        x = st["x"].double()
        y = x.clone()
        for lo, hi, axis, theta in _pairs(case):
            a = (st["positions"][:, axis].double() * theta)[:, None]
            y[:, :, lo] = x[:, :, lo] * a.cos() - x[:, :, hi] * a.sin()
            y[:, :, hi] = x[:, :, hi] * a.cos() + x[:, :, lo] * a.sin()
        return y
    if kind == "append":
        return _exact_append(st, case)
    k, v = st.get("k"), st.get("v")
    if kind == "cached":
        k, v = ((st[x + "_code"].double() * st[x + "_scale"].double().repeat_interleave(BLOCK, 1)[..., None]) for x in "kv")
    q = st["q"].double()
    out = torch.zeros_like(q)
    n, group, scale = case["queries"], case["heads"] // case["kv_heads"], 1 / math.sqrt(case["dim"])
    for b in range(case["batch"]):
        length = int(st["lens"][b]) if kind == "cached" else case["keys"]
        seen = st["mask"][b].nonzero()[:, 0] if kind == "cross" and case["masked"] else torch.arange(length, device=q.device)
        if len(seen) == 0:
            continue
        for h in range(case["heads"]):
            keys, vals = k[b, seen, h // group].double(), v[b, seen, h // group].double()
            s = torch.mm(q[b, :, h], keys.t()) * scale
            if kind == "cached" and case["causal"]:
                ahead = seen[None, :] - (length - n + torch.arange(n, device=q.device))[:, None] > 0
                s[ahead] = float("-inf")
            out[b, :, h] = torch.mm(torch.softmax(s, -1), vals)
    return out


def _exact_append(st, case):
    w, dev = st["window"], st["k"].device
    starts, firsts = st["start"].tolist(), st["first"].tolist()
    counts = st["counts"].tolist() if st["counts"] is not None else [case["new"]] * case["batch"]
    outs = []
    for name in ("k", "v"):
        out = torch.zeros(case["batch"], w, case["kv_heads"], case["dim"], dtype=torch.float64, device=dev)
        for b, (start, first, count) in enumerate(zip(starts, firsts, counts)):
            for at in range(first, start + count, BLOCK):
                lo, hi = max(at, start), min(at + BLOCK, start + count)
                fresh = st[name][b, lo - start:hi - start].double()                      # (tokens, Hk, D)
                s = np.zeros(case["kv_heads"])
                for h, need in enumerate((fresh.abs().amax((0, 2)) / 127).tolist()):
                    if need > 0:
                        step = math.ldexp(1.0, math.frexp(need)[1] - 4)                  # need is 8 to 16 steps
                        s[h] = math.ceil(need / step) * step
                s = torch.from_numpy(s).to(dev)
                if at < start:
                    s0 = st[name + "_scale"][b].double()
                    s = torch.maximum(s, s0)
                    held = st[name + "_code"][b, :start - at].double() * s0[:, None]
                    fresh = torch.cat([held, fresh])
                unit = torch.where(s > 0, s, 1)[:, None]
                out[b, at - first:hi - first] = torch.round(fresh / unit) * unit
        outs.append(out)
    return (*outs, st["start"] + torch.tensor(counts, dtype=torch.int32, device=dev))
