"""What attention with shaped scores and rotary positions of several axes are measured on.

Two operators of a layer's attention, each in its plain form (elementary torch operations in 32 bits;
``own`` false) and as calls of the library (``own`` true):

``attend``  softmax attention over cached K/V whose scores are capped, ``cap * tanh(s / cap)``, or lose
            ``slope[head] * |position - key|``, and whose rows see a range of keys of their own: a prefix
            mask (the tokens of an image and what comes before it see each other), a document mask
            (tokens of packed documents see their own document), a window, or the causal range.
``rope``    the rows a layer's projections hand over, rotated at positions of several axes (time, height,
            width), Q returned, K and V stored into the cache and read back as its pages hold them.

A batch is ``rows`` sequences that append one token, with contexts spread over ``ctx_lo .. ctx_hi``, then
``chunks`` sequences that append ``chunk_lo .. chunk_hi`` prompt tokens after ``prior`` cached ones.
``lens`` seeds lengths, prefixes, documents and image sizes: they belong to the case, values to the seed.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_BASE = {"kind": "attend", "kv": "f16", "heads": 32, "kv_heads": 8, "hd": 128, "hdv": 128, "rows": 0, "ctx_lo": 1,
         "ctx_hi": 1, "chunks": 0, "chunk_lo": 0, "chunk_hi": 0, "prior": 0, "window": 0, "cap": 0.0, "bias": False,
         "mask": "causal", "block": 16, "lens": 0, "rot": 0, "axes": 3, "interleaved": False, "neox": True,
         "qk_norm": False, "theta": 10000.0}


def _case(name, **kw):
    return {"name": name, **_BASE, **kw}


def listed():
    return [
        # one token of a short turn on full-precision pages, scores biased by distance: all latency
        _case("one_row_bias_f32", kv="f32", heads=8, kv_heads=8, hd=64, hdv=64, rows=1, ctx_lo=256, ctx_hi=256, bias=True),
        # a decode batch of mixed context lengths through a layer with capped scores
        _case("decode_cap_f16", rows=32, ctx_lo=512, ctx_hi=4096, cap=50.0, lens=2),
        # few very long contexts on quantised pages, scores biased by distance
        _case("decode_long_bias_q8", kv="q8_0", heads=64, rows=8, ctx_lo=32768, ctx_hi=32768, bias=True),
        # decode rows of packed contexts: each sees its last document only
        _case("decode_documents_bf16", kv="bf16", heads=40, rows=48, ctx_lo=700, ctx_hi=8192, mask="documents", lens=3),
        # four whole prompts that begin with an image: its tokens see each other
        _case("prompts_prefix_bf16", kv="bf16", chunks=4, chunk_lo=2048, chunk_hi=2048, mask="prefix", lens=4),
        # one packed prompt of many documents
        _case("documents_f16", heads=16, kv_heads=4, hd=64, hdv=64, chunks=1, chunk_lo=8192, chunk_hi=8192, mask="documents", lens=5),
        # wide heads, capped scores and a sliding window: prompts beside decode rows
        _case("cap_window_wide_bf16", kv="bf16", heads=16, kv_heads=4, hd=256, hdv=256, rows=4, ctx_lo=700, ctx_hi=3000,
              chunks=2, chunk_lo=600, chunk_hi=1100, window=1024, cap=50.0, lens=9),
        # a head width off the matrix instructions' multiples, every head its own K/V, distance bias
        _case("step_bias_hd80_f16", heads=32, kv_heads=32, hd=80, hdv=80, rows=8, ctx_lo=200, ctx_hi=3000, chunks=1,
              chunk_lo=120, chunk_hi=120, prior=300, bias=True, lens=11),
        # ragged prompts with an image first, capped scores, on quantised pages
        _case("prompts_cap_prefix_q8", kv="q8_0", chunks=3, chunk_lo=401, chunk_hi=2047, cap=30.0, mask="prefix", lens=7),
        # one decoded token of an image prompt: the smallest store
        _case("axes_one_f16", kind="rope", rows=1, ctx_lo=2987, ctx_hi=2987, theta=1000000.0),
        # four prompts of text and images, with the norms of Q and K
        _case("axes_images_bf16", kind="rope", kv="bf16", chunks=4, chunk_lo=2048, chunk_hi=2048, qk_norm=True, theta=1000000.0, lens=12),
        # chunks of a video whose axes take turns over the pairs, on narrower heads rotated in part
        _case("axes_video_f16", kind="rope", heads=16, kv_heads=4, hd=64, hdv=64, chunks=3, chunk_lo=401, chunk_hi=2047, prior=777,
              interleaved=True, rot=48, neox=False, lens=13),
    ]


# (heads, kv_heads, hd, hdv) by use: grouped heads of the usual widths, every head its own K/V, wide heads, a
# value width of its own, a width off the matrix instructions' multiples
_GEOMS = [(32, 8, 128, 128), (40, 8, 128, 128), (64, 8, 128, 128), (16, 4, 64, 64), (8, 8, 64, 64), (32, 32, 64, 64),
          (16, 4, 256, 256), (32, 8, 192, 128), (12, 4, 96, 96), (32, 32, 80, 80)]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    while True:
        c = dict(_BASE)
        c["kind"] = rng.choice(["attend", "attend", "attend", "rope"])
        c["heads"], c["kv_heads"], c["hd"], c["hdv"] = rng.choice(_GEOMS)
        c["kv"] = rng.choice(["f16", "bf16", "q8_0", "f32"] if c["kind"] == "attend" else ["f16", "bf16", "f32"])
        if c["kv"] == "q8_0" and (c["hd"] % 32 or c["hdv"] % 32):
            c["kv"] = "f16"
        c["block"], c["lens"] = rng.choice([16, 32]), rng.randrange(1 << 30)
        shape = rng.choice(["decode", "decode", "prompt", "mixed"])
        if shape != "prompt":
            c["rows"], c["ctx_lo"] = _log(rng, 1, 48), _log(rng, 1, 8192)
            c["ctx_hi"] = min(32768, c["ctx_lo"] * rng.choice([1, 2, 4, 8]))
        if shape != "decode":
            c["chunks"], c["chunk_lo"] = rng.randint(1, 4), _log(rng, 2, 2048)
            c["chunk_hi"] = min(2048, c["chunk_lo"] * rng.choice([1, 1, 2, 4]))
            c["prior"] = rng.choice([0, 0, _log(rng, 1, 4096)])
        if c["kind"] == "attend":
            c["cap"] = rng.choice([0.0, 0.0, 20.0, 30.0, 50.0])
            c["bias"] = rng.random() < 0.35
            c["mask"] = rng.choice(["causal", "prefix", "documents"])
            c["window"] = rng.choice([0, 0, 0, 1024]) if c["mask"] == "causal" else 0
        else:
            c["hdv"] = c["hd"]   # the fused store takes one width
            c["axes"], c["interleaved"] = rng.choice([2, 3, 3, 4]), rng.random() < 0.5
            c["neox"], c["qk_norm"] = rng.random() < 0.6, rng.random() < 0.6
            c["rot"] = rng.choice([0, 0, c["hd"] // 2])
            c["theta"] = rng.choice([10000.0, 500000.0, 1000000.0])
        w = work(c)
        small = c["kv"] == "f32" or c["hd"] % 32 != 0
        if w["bytes"] <= (250e6 if small else 560e6) and w["flops"] <= (6e9 if small else 60e9) and _scores(c) <= 2e9:
            return c


# ---- the batch of a case ---------------------------------------------------------------------------


def _batch(c):
    """[(cached tokens, new tokens)] of the decode rows, and of the prompt chunks."""
    rng = random.Random(c["lens"])
    rows = [(_log(rng, c["ctx_lo"], c["ctx_hi"]) - 1, 1) for _ in range(c["rows"])]
    return rows, [(c["prior"], _log(rng, c["chunk_lo"], c["chunk_hi"])) for _ in range(c["chunks"])]


def _ranges(c):
    """Per sequence of the batch, its new rows' [(position, first key, key after the last)]."""
    rng = random.Random(c["lens"] + 1)
    out = []
    for prior, new in sum(_batch(c), []):
        total = prior + new
        prefix = rng.randint(1, total) if c["mask"] == "prefix" else 0
        starts = [0]
        while c["mask"] == "documents" and starts[-1] < total:
            starts.append(starts[-1] + _log(rng, 40, 2000))
        rows, d = [], 0
        for pos in range(prior, total):
            while d + 1 < len(starts) and starts[d + 1] <= pos:
                d += 1
            lo = max(starts[d], pos + 1 - c["window"] if c["window"] else 0)
            rows.append((pos, lo, max(pos + 1, prefix if pos < prefix else 0)))
        out.append(rows)
    return out


def _scores(c):
    """Scores of the plain form's padded batches."""
    return sum(c["heads"] * len(g) * max(n for _, n in g) * max(p + n for p, n in g) for g in _batch(c) if g)


def _elem_bytes(c):
    return {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "q8_0": 34.0 / 32.0}[c["kv"]]


def work(case):
    c = case
    kv_row, q_row = c["kv_heads"] * (c["hd"] + c["hdv"]), c["heads"] * (c["hd"] + c["hdv"])
    if c["kind"] == "rope":   # q, k, v and the positions in, q out, K and V rows in the pages' type
        n = sum(m for g in _batch(c) for _, m in g)
        half = (c["rot"] or c["hd"]) // 2
        return {"bytes": n * (4.0 * (q_row + kv_row + c["axes"]) + kv_row * _elem_bytes(c)),
                "flops": n * (c["heads"] + c["kv_heads"]) * (6.0 * half + (4.0 * c["hd"] if c["qk_norm"] else 0.0))}
    n_bytes = pairs = 0.0
    for rows in _ranges(c):
        n_bytes += _span(rows) * kv_row * _elem_bytes(c) + len(rows) * q_row * 4.0
        pairs += sum(hi - lo for _, lo, hi in rows)
    return {"bytes": n_bytes, "flops": 2.0 * (c["hd"] + c["hdv"]) * pairs * c["heads"]}


def _span(rows):
    """Keys that some row sees (the ranges of a sequence's rows move forward)."""
    n = end = 0
    for _, lo, hi in rows:
        n += max(0, hi - max(lo, end))
        end = max(end, hi)
    return n


# ---- inputs ----------------------------------------------------------------------------------------


def _rand(seed, tag, shape):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + tag * 7919 + 1) & 0x7FFFFFFFFFFF)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _held(x, kv):
    """x [..., width] as a cache holds it: its type's values, or q8_0 codes and scales of 32 values."""
    if kv != "q8_0":
        return (x.to({"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[kv]),)
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = b.abs().amax(dim=-1, keepdim=True) / 127.0
    codes = torch.round(b * torch.where(d != 0, 1.0 / d, torch.zeros_like(d)))
    return codes.to(torch.int8), d.half()


def _values(held):
    """The f32 values of what _held gives."""
    if len(held) == 1:
        return held[0].float()
    return (held[0].float() * held[1].float()).flatten(-2)


def _slopes(c):
    """Distance slopes: a geometric series over the heads, from 1/2 down to 1/256."""
    return torch.tensor([2.0 ** (-1.0 - 7.0 * h / max(c["heads"] - 1, 1)) for h in range(c["heads"])], device="cuda")


def _sections(c):
    """Pairs of each axis: about a quarter for the first and the rest shared by the others, or by turns."""
    half = (c["rot"] or c["hd"]) // 2
    rest = [half // c["axes"] if c["interleaved"] else (half - half // 4) // (c["axes"] - 1)] * (c["axes"] - 1)
    return [half - sum(rest)] + rest


def _axis_of(c):
    """The axis of each pair: sections one after the other, or pair i of axis i % axes while that has some left."""
    n, sec = c["axes"], _sections(c)
    if not c["interleaved"]:
        return [a for a in range(n) for _ in range(sec[a])]
    return [i % n if i % n and i < n * sec[i % n] else 0 for i in range(sum(sec))]


def _positions(c):
    """[axes][rows] positions as prompts of text and images have them: every axis alike in text, a grid in an image."""
    rng = random.Random(c["lens"] + 2)
    n, out = c["axes"], [[] for _ in range(c["axes"])]
    for prior, new in sum(_batch(c), []):
        at, done = prior, 0
        while done < new:
            text = min(new - done, rng.randint(1, 60))
            for a in range(n):
                out[a] += range(at, at + text)
            at, done = at + text, done + text
            t, h, w = rng.choice([1, 1, 4]), rng.randint(2, 24), rng.randint(2, 24)
            for i in range(min(new - done, t * h * w)):
                grid = (i // (h * w), i // w % h, i % w, i // (h * w))
                for a in range(n):
                    out[a].append(at + grid[a])
            done += min(new - done, t * h * w)
            at += max(t, h, w)
    return out


def _kv_of(c, seed, s, tokens):
    """K and V of sequence s as drawn (f32): what the cache holds are their roundings."""
    return _rand(seed, 2 * s, (tokens, c["kv_heads"], c["hd"])), _rand(seed, 2 * s + 1, (tokens, c["kv_heads"], c["hdv"]))


def _step_in(c, seed, n):
    """The step's rows: q, and for the store k, v."""
    shapes = (c["heads"], c["hd"]), (c["kv_heads"], c["hd"]), (c["kv_heads"], c["hdv"])
    return [_rand(seed, 100000 + i, (n, *s)) for i, s in enumerate(shapes)]


def _norms(c, seed):
    w = 1.0 + 0.1 * _rand(seed, 200000, (2, c["hd"]))
    return (w[0].contiguous(), w[1].contiguous()) if c["qk_norm"] else (None, None)


_EPS = 1e-6


# ---- the measured passes ---------------------------------------------------------------------------


def prepare(case, seed):
    """The step's inputs, and the cached tokens: in the library's cache (its handle, pages and packed
    segments live as long as the sequences), or for the plain form as padded tensors of the pages' values."""
    c, groups = case, _batch(case)
    n = sum(m for g in groups for _, m in g)
    q, k, v = _step_in(c, seed, n)
    st = {"case": c, "q": q, "scale": 1.0 / math.sqrt(c["hd"])}
    if c["kind"] == "rope":
        st |= {"k": k, "v": v, "norms": _norms(c, seed), "positions": torch.tensor(_positions(c), dtype=torch.int32, device="cuda")}
    else:
        st["slopes"] = _slopes(c) if c["bias"] else None
    if own:
        _prepare_cache(st, c, seed, sum(groups, []))
    elif c["kind"] == "attend":
        st["groups"] = []
        ranges, s0, row0 = _ranges(c), 0, 0
        for g in groups:
            if not g:
                continue
            t, length = max(m for _, m in g), max(p + m for p, m in g)
            k = torch.zeros(len(g), length, c["kv_heads"], c["hd"], device="cuda")
            v = torch.zeros(len(g), length, c["kv_heads"], c["hdv"], device="cuda")
            at = torch.zeros(len(g), t, 4, dtype=torch.int32)   # row, position, first key, key after the last
            real = torch.zeros(len(g), t, dtype=torch.bool)
            for i, (p, m) in enumerate(g):
                k[i, :p + m], v[i, :p + m] = _kv_of(c, seed, s0 + i, p + m)
                at[i, :m, 0] = torch.arange(row0, row0 + m)
                at[i, :m, 1:] = torch.tensor(ranges[s0 + i])
                real[i, :m] = True
                row0 += m
            s0 += len(g)
            st["groups"].append({"k": _held(k, c["kv"]), "v": _held(v, c["kv"]), "at": at.cuda(), "real": real.cuda()})
    torch.cuda.synchronize()
    return st


def _prepare_cache(st, c, seed, batch):
    from llmario_amd.kv import HipKvCache, Layer, RowRanges, Segments
    hc = HipKvCache([Layer(c["heads"], c["kv_heads"], c["hd"], c["hdv"])], max_ctx=max(p + m for p, m in batch), n_seqs=len(batch),
                    kv_type=c["kv"], block_tokens=c["block"], pool_tokens=sum(p + m for p, m in batch) + c["block"] * len(batch))
    order = list(range(hc.layout()["pool_blocks"]))   # block ids as a long-running cache has them
    random.Random(seed).shuffle(order)
    at, row0, segs = 0, 0, []
    for s, (p, m) in enumerate(batch):
        need = -(-(p + m) // c["block"])
        hc.adopt_blocks(s, order[at:at + need])
        at += need
        if c["kind"] == "attend":
            k, v = _kv_of(c, seed, s, p + m)
            hc.store(0, [(s, 0, p + m, 0)], _values(_held(k, c["kv"])), _values(_held(v, c["kv"])))
        hc.set_len(s, p)
        segs.append((s, row0, m, p))
        row0 += m
    st |= {"cache": hc, "segs": Segments(segs), "out": torch.empty(row0, c["heads"], c["hdv"], device="cuda")}
    if c["kind"] == "attend" and c["mask"] != "causal":
        flat = [r for rows in _ranges(c) for r in rows]
        st["ranges"] = RowRanges([r[1] for r in flat], [r[2] for r in flat])
    if c["kind"] == "rope":
        t = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[c["kv"]]
        st["q_out"] = torch.empty_like(st["q"])
        st["rows"] = [torch.empty(row0, c["kv_heads"], c["hd"], dtype=t, device="cuda") for _ in range(2)]


def run(state):
    c = state["case"]
    if c["kind"] == "attend":
        return _attend_own(state, c) if own else torch.cat([_attend_plain(state, c, g) for g in state["groups"]])
    return _rope_own(state, c) if own else _rope_plain(state, c)


def _attend_own(st, c):
    st["cache"].attend_scored(0, st["segs"], st["q"], st["out"], st["scale"], window=c["window"], cap=c["cap"], slopes=st["slopes"],
                              ranges=st.get("ranges"))
    return st["out"]


def _rope_own(st, c):
    hc, (k_rows, v_rows), (q_norm, k_norm) = st["cache"], st["rows"], st["norms"]
    hc.qk_rope_store_axes(0, st["segs"], st["q"], st["k"], st["v"], st["q_out"], st["positions"], _sections(c), interleaved=c["interleaved"],
                          rot_dim=c["rot"], theta=c["theta"], neox=c["neox"], q_norm=q_norm, k_norm=k_norm, eps=_EPS)
    hc.gather_encoded(0, st["segs"], k_rows, v_rows)
    return [st["q_out"], k_rows, v_rows]


def _attend_plain(st, c, g):
    """One padded batch: g's K / V [seqs, keys, kv_heads, width], its rows' (row, position, lo, hi)."""
    k, v = _values(g["k"]), _values(g["v"])
    (n, t), length, kvh, group = g["real"].shape, k.shape[1], c["kv_heads"], c["heads"] // c["kv_heads"]
    row, pos, lo, hi = (x.reshape(n, 1, t, 1) for x in g["at"].unbind(-1))
    q = st["q"][row.flatten()].reshape(n, t, kvh, group, c["hd"]).permute(0, 2, 3, 1, 4).reshape(n, kvh, group * t, c["hd"])
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).reshape(n, c["heads"], t, length) * st["scale"]
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    key = torch.arange(length, device="cuda", dtype=torch.int32)
    if c["bias"]:
        s = s - st["slopes"].reshape(1, -1, 1, 1) * (pos - key).abs()
    s = torch.where((key >= lo) & (key < hi), s, -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.reshape(n, kvh, group * t, length), v.permute(0, 2, 1, 3).contiguous()).reshape(n, c["heads"], t, c["hdv"])
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 2, 1, 3)[g["real"]]


def _rope_plain(st, c):
    """RMS norm, rotation with angles in 64 bits, and the pages' rounding."""
    rot = c["rot"] or c["hd"]
    pair = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    pos = st["positions"][torch.tensor(_axis_of(c), device="cuda")].t().double()   # [rows, pairs]
    ang = pos * torch.pow(torch.tensor(c["theta"], dtype=torch.float64, device="cuda"), -2.0 * pair / rot)
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
    q, k = _rotated(c, st["q"], st["norms"][0], cos, sin), _rotated(c, st["k"], st["norms"][1], cos, sin)
    return [q, *_held(k, c["kv"]), *_held(st["v"], c["kv"])]


def _rotated(c, x, w, cos, sin):
    rot = c["rot"] or c["hd"]
    if w is not None:
        x = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + _EPS) * w
    if c["neox"]:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], dim=-1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2), x[..., rot:]], dim=-1)


# ---- the same in 64 bits ---------------------------------------------------------------------------


def exact(case, seed):
    c, batch = case, sum(_batch(case), [])
    n = sum(m for _, m in batch)
    q, k, v = _step_in(c, seed, n)
    if c["kind"] == "rope":
        wq, wk = _norms(c, seed)
        return [_rope64(c, q, wq), _rope64(c, k, wk), v.double()]
    slopes = _slopes(c).double()
    group, outs, row0 = c["heads"] // c["kv_heads"], [], 0
    for s, rows in enumerate(_ranges(c)):
        p, m = batch[s]
        ks, vs = (_values(_held(x, c["kv"])).double() for x in _kv_of(c, seed, s, p + m))
        at = torch.tensor(rows, device="cuda")
        out = torch.zeros(m, c["heads"], c["hdv"], dtype=torch.float64, device="cuda")
        for h in range(c["heads"]):
            kt, vh = ks[:, h // group].t().contiguous(), vs[:, h // group].contiguous()
            for t in range(0, m, 2048):
                pos, lo, hi = (at[t:t + 2048, i:i + 1] for i in range(3))
                x = torch.mm(q[row0 + t:row0 + min(m, t + 2048), h].double(), kt) / math.sqrt(c["hd"])
                if c["cap"]:
                    e = torch.expm1(2.0 * x.abs() / c["cap"])
                    x = torch.sign(x) * c["cap"] * (e / (e + 2.0))
                key = torch.arange(p + m, device="cuda")[None, :]
                if c["bias"]:
                    x -= slopes[h] * torch.maximum(pos - key, key - pos)
                see = ~((key < lo) | (key >= hi))
                x.masked_fill_(~see, -math.inf)
                out[t:t + 2048, h] = torch.mm(torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0), vh)
        outs.append(out)
        row0 += m
    return torch.cat(outs)


def _rope64(c, x, w):
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(torch.sum(x ** 2, dim=-1, keepdim=True) / c["hd"] + _EPS) * w.double()
    rot, axis, pos = c["rot"] or c["hd"], _axis_of(c), torch.tensor(_positions(c), dtype=torch.float64, device="cuda")
    y = x.clone()
    for i in range(rot // 2):
        angle = pos[axis[i]] * math.exp(-math.log(c["theta"]) * 2 * i / rot)
        z = torch.polar(torch.ones_like(angle), angle)[:, None]
        a, b = (i, i + rot // 2) if c["neox"] else (2 * i, 2 * i + 1)
        z = z * torch.complex(x[..., a], x[..., b])
        y[..., a], y[..., b] = z.real, z.imag
    return y
