"""lmh_attend_scored on long segments (the kernel whose workgroups share a segment's pages), with test_gpu_scored's
definition and tolerances: every page type and width, units that begin inside a token, columns that fill a unit in part,
tiles that end inside a block, key pieces, ranges, magnitudes over the types' range, and values that are not finite."""

import numpy as np
import pytest
import torch

from llmario_amd.kv import RowRanges
from test_gpu_scored import Call, ranges_of, slopes_of

pytestmark = pytest.mark.gpu

# kv, geometry, prior, new, block, window
FORMS = [
    ("f16", (8, 8, 64, 64), [0], [128], 16, 0),
    ("f16", (12, 4, 64, 64), [37, 5], [90, 1], 16, 50),
    ("f16", (32, 8, 128, 128), [0, 700], [65, 33], 32, 0),
    ("f16", (40, 8, 128, 128), [63], [52], 16, 0),        # five heads: units begin inside a token
    ("f16", (16, 4, 256, 256), [17], [33], 16, 0),
    ("f16", (16, 2, 256, 256), [17, 64], [17, 30], 64, 70),
    ("bf16", (8, 2, 64, 64), [3], [70], 16, 0),
    ("bf16", (32, 8, 128, 128), [0, 31, 1], [64, 65, 66], 16, 0),
    ("bf16", (6, 2, 128, 128), [111], [200], 32, 90),
    ("bf16", (16, 4, 256, 256), [0], [97], 16, 0),
    ("q8_0", (8, 4, 64, 64), [9], [129], 16, 0),
    ("q8_0", (32, 8, 128, 128), [0, 40], [64, 131], 16, 0),
    ("q8_0", (7, 1, 128, 128), [300], [37], 32, 100),
    ("bf16", (71, 1, 64, 64), [20], [9], 16, 0),          # a group wider than a unit's wave
    ("f16", (300, 1, 64, 64), [20], [2], 16, 0),          # .. and than a unit
]
IDS = [f"{f[0]}-{'x'.join(map(str, f[1]))}-{'_'.join(map(str, f[3]))}" for f in FORMS]


@pytest.mark.parametrize("kind", [None, "prefix", "documents", "random", "one", "none"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_forms(form, kind):
    kv, geo, prior, new, bt, window = form
    c = Call(kv, geo, prior, new, bt, seed=11)
    r, sl = ranges_of(kind, c.segs, seed=12), slopes_of(geo[0])
    rows = None if max(new) < 70 else sorted({0, 1, 2, 31, 32, 33, 63, 64, 65, 127, max(new) - 2, max(new) - 1})
    for kw in ({}, {"cap": 2.0, "slopes": sl}, {"cap": 40.0}, {"slopes": sl}):
        kw = dict(kw, window=window, ranges=r)
        c.check(c.run(**kw), rows=rows, **kw)


@pytest.mark.parametrize("kv,geo,prior,new", [
    ("bf16", (32, 8, 128, 128), [6000], [40]), ("f16", (8, 2, 64, 64), [9000], [70]), ("q8_0", (8, 1, 128, 128), [5000], [35]),
    ("bf16", (8, 2, 256, 256), [4000, 100], [50, 40]), ("f16", (5, 1, 128, 128), [12000], [60])])
def test_chunks_on_long_prefixes_in_pieces(kv, geo, prior, new):
    """Few long units: cut into key pieces. Rows that see everything, the first key, the last, one in between, nothing."""
    c = Call(kv, geo, prior, new, seed=13)
    sl = slopes_of(geo[0], 2.0 ** -8)
    rows = [0, 1, 2, 3, 4, 17, new[0] - 1]
    c.check(c.run(slopes=sl, cap=50.0), slopes=sl, cap=50.0, rows=rows)
    lo, hi = [], []
    for p, n in zip(prior, new):
        for j in range(n):
            a, b = [(0, p + n), (0, 1), (p + n - 1, p + n), (p // 2, p // 2 + 1), (5, 5)][j % 5]
            lo.append(a)
            hi.append(b)
    r = RowRanges(lo, hi)
    c.check(c.run(cap=20.0, ranges=r), cap=20.0, ranges=r, rows=rows)


@pytest.mark.parametrize("kv,hd", [("f16", 64), ("bf16", 128), ("q8_0", 128), ("f16", 256)])
def test_scales_of_any_sign(kv, hd):
    c = Call(kv, (8, 2, hd, hd), [50], [70], seed=21, spread=4.0)
    for kw in ({"scale": -0.1}, {"scale": 0.0}, {"scale": -0.2, "cap": 3.0}, {"scale": 0.0, "slopes": slopes_of(8)},
               {"scale": 1.0, "cap": 1e-2}, {"scale": 0.02, "cap": 1e20}):
        c.check(c.run(**kw), rows=[0, 1, 33, 69], **kw)


@pytest.mark.parametrize("kv,geo", [("bf16", (32, 8, 128, 128)), ("f16", (8, 2, 64, 64)), ("q8_0", (16, 4, 128, 128))])
def test_pieces_that_hold_values_that_are_not_finite(kv, geo):
    """A unit cut into key pieces, one of which holds a key of V beyond any number: the rows that do not see it."""
    c = Call(kv, geo, [5000], [40], seed=22)
    lo = [0 if j % 2 else 2001 for j in range(40)]
    r = RowRanges(lo, None)
    clean = c.run(slopes=slopes_of(geo[0], 2.0 ** -9), ranges=r).clone()
    c.hc.store(0, [(0, 0, 1, 2000)], c.k[0][2000:2001].contiguous(), torch.full_like(c.v[0][:1], 3e38 if kv == "q8_0" else float("inf")))
    out = c.run(slopes=slopes_of(geo[0], 2.0 ** -9), ranges=r)
    assert torch.isfinite(out[0::2]).all() and not torch.isfinite(out[1::2]).any()
    assert (out[0::2] - clean[0::2]).abs().max().item() <= 1e-4


def test_short_segments_beside_long_ones():
    """Decode rows in the prompts' launch, in one of their own before it, and a short prompt in theirs: the same rows."""
    for prior, new in (([300, 40, 7, 0], [1, 1, 2, 500]), ([3000] * 20 + [0], [1] * 20 + [150]), ([5000] * 24 + [0, 64], [1] * 24 + [600, 300])):
        for kv, geo in (("bf16", (16, 4, 128, 128)), ("f16", (8, 2, 64, 64))):
            c = Call(kv, geo, prior, new, seed=23)
            c.check(c.run(cap=10.0), cap=10.0, rows=[0, 1, 140, 499])


def refill(c, s, k_mul=1.0, v_mul=1.0, from_pos=0):
    """Sequence s's K and V from a position on times k_mul, v_mul, stored again."""
    t = c.prior[s] + c.new[s]
    c.hc.store(0, [(s, 0, t - from_pos, from_pos)], (c.k[s][from_pos:] * k_mul).contiguous(), (c.v[s][from_pos:] * v_mul).contiguous())
    c.read_back()


SIZES = [("bf16", (8, 2, 128, 128)), ("q8_0", (8, 2, 128, 128)), ("f16", (8, 2, 128, 128)), ("bf16", (8, 2, 64, 64)),
         ("bf16", (4, 1, 256, 256)), ("q8_0", (8, 2, 64, 64))]


@pytest.mark.parametrize("new", [[90], [1]])
@pytest.mark.parametrize("kv,geo", SIZES, ids=[f"{k}-{g[2]}" for k, g in SIZES])
def test_magnitudes(kv, geo, new):
    """K, V and Q far from 1, up to what the pages' type holds: products within the tolerance of their own size."""
    top = {"bf16": 1e30, "q8_0": 1e4, "f16": 1e4}[kv]
    low = {"bf16": 1e-30, "q8_0": 1e-2, "f16": 1e-2}[kv]
    for k_mul, v_mul, q_mul in ((1.0, low, 1.0), (1.0, top, 1.0), (top, 1.0, 1 / top), (low, 1.0, 1 / low), (1.0, 1.0, 0.0)):
        c = Call(kv, geo, [100], new, seed=14)
        c.q *= q_mul
        refill(c, 0, k_mul, v_mul)
        rows = [0, 1, 30, 89]
        c.check(c.run(cap=15.0), cap=15.0, rows=rows)
        c.check(c.run(), rows=rows)


@pytest.mark.parametrize("kv,geo", [x for x in SIZES if x[0] != "f16"], ids=[f"{k}-{g[2]}" for k, g in SIZES if k != "f16"])
def test_magnitudes_that_grow_along_the_sequence(kv, geo):
    """Small first keys, then K (or V) too large for what the first tile suggested: the units are computed again in f32."""
    for k_mul, v_mul in ((3e5, 1.0), (1.0, 3e5)):
        c = Call(kv, geo, [100], [90], seed=15, spread=1e-5 if k_mul > 1 else 1.0)
        refill(c, 0, 1e-3, 1e-3)
        refill(c, 0, 1e3 * k_mul, 1e3 * v_mul, from_pos=70)
        c.check(c.run(cap=15.0), cap=15.0, rows=[0, 1, 30, 89])


@pytest.mark.parametrize("mul", [1e-2, 1e-4, 1e-7, 1e2, 1e4])
@pytest.mark.parametrize("kv,geo", [x for x in SIZES if x[0] != "f16"], ids=[f"{k}-{g[2]}" for k, g in SIZES if k != "f16"])
def test_documents_of_other_magnitudes(kv, geo, mul):
    """Packed documents whose V (then K) is far from the first one's: each row within the tolerance of the V it sees."""
    if kv == "q8_0":
        mul = min(max(mul, 1e-3), 1e3)   # (its scales are f16: 1e-3 of a row at 1e-1 is held to 2^-10 or so, as read back)
    for base in (0.1, 1.0, 30.0):
        c = Call(kv, geo, [0], [190], seed=17)
        refill(c, 0, 1.0, base)
        refill(c, 0, 1.0, base * mul, from_pos=70)
        r = RowRanges.of(c.segs, documents=[[0, 70, 71, 75, 130]])
        for kw in ({"ranges": r}, {"ranges": r, "cap": 15.0}, {"window": 20}):
            c.check(c.run(**kw), rows=[0, 5, 69, 70, 71, 72, 75, 80, 129, 130, 131, 189], **kw)
        refill(c, 0, 1.0, 1.0)
        refill(c, 0, mul, 1.0, from_pos=70)
        c.check(c.run(ranges=r), rows=[0, 69, 70, 72, 80, 130, 189], ranges=r)


@pytest.mark.parametrize("kv,geo", SIZES, ids=[f"{k}-{g[2]}" for k, g in SIZES])
def test_a_head_whose_v_is_zero(kv, geo):
    c = Call(kv, geo, [0], [150], seed=18)
    c.v[0].view(150, geo[1], geo[3])[:, 0] = 0.0
    refill(c, 0)
    out = c.run(cap=15.0)
    c.check(out, cap=15.0, rows=[0, 1, 64, 149])
    if geo[1] > 1:
        assert (out[:, :geo[0] // geo[1]] == 0).all()


@pytest.mark.parametrize("mul", [1e-2, 1e-4, 1e-7, 1e2, 1e4])
@pytest.mark.parametrize("kv,geo", [("bf16", (8, 2, 128, 128)), ("q8_0", (8, 2, 64, 64)), ("bf16", (8, 8, 96, 96)), ("f32", (8, 2, 64, 64)), ("bf16", (4, 2, 80, 80)), ("q8_0", (4, 2, 96, 96))],
                         ids=lambda x: x if isinstance(x, str) else str(x[2]))
def test_documents_of_other_magnitudes_in_short_segments(kv, geo, mul):
    """The same in the unit launch: decode rows and drafted tokens."""
    if kv == "q8_0":
        mul = min(max(mul, 1e-3), 1e3)
    for base in (0.1, 1.0, 30.0):
        c = Call(kv, geo, [171, 70], [5, 1], seed=17)
        for s in range(2):
            refill(c, s, 1.0, base)
            refill(c, s, 1.0, base * mul, from_pos=50)
        lo, hi = [0, 50, 100, 49, 52, 50], [50, 51, 175, 52, 70, 71]
        for kw in ({"ranges": RowRanges(lo, hi)}, {"ranges": RowRanges(lo, hi), "cap": 15.0}, {"window": 20}):
            c.check(c.run(**kw), **kw)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("form", [f for f in FORMS if f[4] == 16 and not f[5] and f[1][0] < 50], ids=lambda f: f"{f[0]}-{f[1][2]}-{f[3][0]}")
def test_values_that_are_not_finite(form, bad):
    """K and V of a few keys are not finite. Rows that do not see them: as if they were zero. Rows that do: not finite
    where the value reaches (V), whatever else the unit holds."""
    kv, geo, prior, new, bt, _ = form
    c = Call(kv, geo, prior, new, bt, seed=16)
    total = prior[0] + new[0]
    hide = [3, total // 2]
    lo, hi = [], []
    for s, start, n, p0 in c.segs:
        for j in range(n):
            pos = p0 + j
            if s == 0 and j % 3 == 0:
                lo.append(0)                    # sees key 3
                hi.append(max(pos + 1, 4))
            elif s == 0 and j % 3 == 1:
                lo.append(4)
                hi.append(total // 2)
            else:
                lo.append(total // 2 + 1 if s == 0 else 0)
                hi.append(max(pos + 1, total // 2 + 2) if s == 0 else pos + 1)
    r = RowRanges(lo, hi)
    clean = c.run(cap=9.0, ranges=r).clone()
    c.check(clean, cap=9.0, ranges=r)
    for pos in hide:
        k, v = c.k[0][pos:pos + 1].clone(), c.v[0][pos:pos + 1].clone()
        v.fill_(3e38 if kv == "q8_0" else bad)   # (a q8_0 row whose scale overflows)
        c.hc.store(0, [(0, 0, 1, pos)], k, v)
    out = c.run(cap=9.0, ranges=r)
    sees = torch.tensor([any(a <= p < b for p in hide) and t < new[0] for t, (a, b) in enumerate(zip(lo, hi))], device="cuda")
    assert not torch.isfinite(out[sees]).any() and torch.isfinite(out[~sees]).all()
    d = (out[~sees] - clean[~sees]).abs().max().item()
    assert d <= 1e-4, d   # another kernel's rounding at the most: tolerances above allow 2 * (hd / 16 + 12) 2^-24 (|q k| + 10) max|v|
    if kv != "q8_0":
        return
    k = c.k[0][3:4].clone().fill_(3e38)
    c.hc.store(0, [(0, 0, 1, 3)], k, c.v[0][3:4].contiguous())
    out = c.run(cap=9.0, ranges=r)
    hid = torch.tensor([t < new[0] and not any(a <= p < b for p in hide) for t, (a, b) in enumerate(zip(lo, hi))], device="cuda")
    assert torch.isfinite(out[hid]).all() and (out[hid] - clean[hid]).abs().max().item() <= 1e-4
