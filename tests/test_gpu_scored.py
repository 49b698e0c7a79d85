"""lmh_attend_scored against its definition in 64 bits: scores capped by a tanh, biased by distance, rows that see
ranges of keys of their own (prefix and document masks, windows, single keys, nothing), on every page type and
layout, at the sizes where the tiling can go wrong.

Tolerance of a row: each score is off by at most
    err = (hd / 16 + 12) 2^-24 (sum |q k| scale + |s| + |bias| + 1)
(f32 sums in at most hd / 16 + 8 steps; Q held to 2^-22 or better, the tanh, the bias and the exponent's argument by a
few roundings of their size), which moves the output by at most 2 sum(w err) max|v|; weights in two 11-bit parts, the
exponential and the sums add 2^-20 max|v|."""

import numpy as np
import pytest
import torch

from llmario_amd import _native as N
from llmario_amd.kv import HipKvCache, Layer, LmhError, RowRanges, Segments

pytestmark = pytest.mark.gpu


class Call:
    """A cache of one layer with sequences of prior + new stored tokens, and the call's rows."""

    def __init__(self, kv, geo, prior, new, bt=16, seed=0, window_layer=0, spread=1.0):
        self.kv, self.geo, self.prior, self.new = kv, geo, prior, new
        n_head, n_kv, hd, hdv = geo
        rng = np.random.default_rng(seed)
        totals = [p + n for p, n in zip(prior, new)]
        layers = [Layer(n_head, n_kv, hd, hdv, window_layer)] + ([Layer(n_head, n_kv, hd, hdv)] if window_layer else [])
        self.hc = HipKvCache(layers, max_ctx=max(totals) + bt, n_seqs=len(prior), kv_type=kv, block_tokens=bt, n_batch=max(totals))
        self.k, self.v, self.segs, start = [], [], [], 0
        for s, t in enumerate(totals):
            self.hc.reserve(s, t)
            k = torch.from_numpy(rng.standard_normal((t, n_kv * hd)).astype(np.float32)).cuda()
            v = torch.from_numpy(rng.standard_normal((t, n_kv * hdv)).astype(np.float32)).cuda()
            self.hc.store(0, [(s, 0, t, 0)], k, v)
            self.k.append(k)
            self.v.append(v)
            self.segs.append((s, start, new[s], prior[s]))
            start += new[s]
        self.n_rows = start
        self.q = torch.from_numpy((spread * rng.standard_normal((start, n_head, hd))).astype(np.float32)).cuda()
        self.read_back()

    def read_back(self):
        """K and V as the pages hold them."""
        for s, (p, n) in enumerate(zip(self.prior, self.new)):
            self.hc.gather(0, [(s, 0, p + n, 0)], self.k[s], self.v[s])
        torch.cuda.synchronize()

    def run(self, scale=None, q=None, out=None, **kw):
        n_head, _, hd, hdv = self.geo
        out = torch.full((self.n_rows, n_head, hdv), 7.0, device="cuda") if out is None else out
        self.hc.attend_scored(0, Segments(self.segs), self.q if q is None else q, out, 1 / hd ** 0.5 if scale is None else scale, **kw)
        torch.cuda.synchronize()
        return out

    def check(self, out, scale=None, window=0, cap=0.0, slopes=None, ranges=None, rows=None):
        n_head, n_kv, hd, hdv = self.geo
        scale = 1 / hd ** 0.5 if scale is None else scale
        out = out.double().cpu().numpy()
        assert np.isfinite(out).all()
        sl = slopes.double().cpu().numpy() if slopes is not None else None
        worst = 0.0
        for s, start, n, p0 in self.segs:
            ks = self.k[s].double().cpu().numpy().reshape(-1, n_kv, hd)
            vs = self.v[s].double().cpu().numpy().reshape(-1, n_kv, hdv)
            for j in range(n) if rows is None else [x for x in rows if x < n]:
                t, pos = start + j, p0 + j
                lo = max(ranges.lo[t] if ranges is not None and ranges.lo is not None else 0, pos + 1 - window if window else 0)
                hi = ranges.hi[t] if ranges is not None and ranges.hi is not None else pos + 1
                if lo >= hi:
                    assert (out[t] == 0).all(), (t, "sees nothing")
                    continue
                q = self.q[t].double().cpu().numpy().reshape(n_kv, -1, hd)
                k, v = ks[lo:hi], vs[lo:hi]
                x = np.einsum("hgd,khd->hgk", q, k) * scale
                mag = np.einsum("hgd,khd->hgk", np.abs(q), np.abs(k)) * abs(scale)
                if cap:
                    x = cap * np.tanh(x / cap)
                bias = np.zeros_like(x)
                if sl is not None:
                    bias = sl.reshape(n_kv, -1, 1) * np.abs(pos - np.arange(lo, hi))
                err = (hd / 16 + 12) * 2.0 ** -24 * (mag + np.abs(x) + np.abs(bias) + 1)
                x = x - bias
                w = np.exp(x - x.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                want = np.einsum("hgk,khd->hgd", w, v).reshape(n_head, hdv)
                top = np.abs(v).max(axis=(0, 2))[:, None]
                tol = ((2 * (w * err).sum(-1) + 2.0 ** -20) * top).reshape(n_head)
                d = np.abs(out[t] - want).max(-1)
                assert (d <= tol).all(), (t, pos, lo, hi, float((d / tol).max()), float(d.max()))
                worst = max(worst, float((d / tol).max()))
        return worst


def slopes_of(n_head, top=0.5):
    return torch.tensor([top * 2.0 ** (-8.0 * h / n_head) for h in range(n_head)], device="cuda")


def ranges_of(kind, segs, seed=0):
    rng = np.random.default_rng(seed)
    if kind is None:
        return None
    if kind == "prefix":
        return RowRanges.of(segs, prefix=[int(rng.integers(0, p + n + 1)) for _, _, n, p in segs])
    if kind == "documents":
        return RowRanges.of(segs, documents=[sorted(set(rng.integers(0, p + n, 4).tolist())) for _, _, n, p in segs])
    lo, hi = [], []
    for _, _, n, p in segs:
        for pos in range(p, p + n):
            a = int(rng.integers(0, p + n))
            lo.append(a)
            hi.append(a + 1 if kind == "one" else a if kind == "none" else int(rng.integers(0, p + n + 1)))
    return RowRanges(lo, hi)


# kv, geometry, prior, new, block, window
FORMS = [
    ("f32", (8, 8, 64, 64), [255], [1], 16, 0),
    ("f32", (12, 4, 128, 128), [0, 40, 15], [1, 33, 2], 16, 0),
    ("f32", (4, 1, 256, 256), [70, 3], [3, 1], 32, 20),
    ("f32", (8, 2, 100, 100), [31, 500], [1, 7], 16, 0),
    ("f16", (32, 8, 128, 128), [0, 15, 16, 17, 700], [1, 1, 1, 1, 1], 16, 0),
    ("f16", (40, 8, 128, 128), [300, 0], [5, 90], 32, 64),
    ("f16", (32, 32, 64, 64), [100, 31], [40, 1], 64, 0),
    ("f16", (16, 4, 256, 256), [33, 200], [70, 1], 16, 0),
    ("f16", (12, 4, 96, 96), [5], [131], 16, 0),
    ("f16", (8, 4, 32, 32), [64], [77], 16, 33),
    ("f16", (4, 4, 192, 192), [50], [20], 16, 0),
    ("f16", (32, 8, 192, 128), [120], [19], 16, 0),
    ("bf16", (32, 8, 128, 128), [0, 31, 32, 900], [1, 1, 9, 1], 16, 0),
    ("bf16", (16, 4, 256, 256), [100, 3], [33, 1], 16, 50),
    ("bf16", (12, 4, 96, 96), [40], [55], 32, 0),
    ("bf16", (8, 8, 64, 64), [0], [150], 16, 0),
    ("bf16", (6, 2, 192, 192), [77], [18], 16, 0),
    ("bf16", (4, 2, 32, 32), [77], [18], 16, 0),
    ("bf16", (8, 2, 192, 128), [9], [41], 16, 0),
    ("q8_0", (32, 8, 128, 128), [0, 500, 33], [1, 1, 21], 16, 0),
    ("q8_0", (16, 4, 64, 64), [15], [90], 32, 0),
    ("q8_0", (4, 2, 256, 256), [47], [40], 16, 30),
    ("q8_0", (4, 2, 192, 192), [47], [40], 16, 0),
    # the row layout: on matrix cores, then on the slower kernel
    ("f16", (32, 32, 80, 80), [30, 200], [20, 1], 16, 0),
    ("bf16", (8, 2, 80, 80), [63], [30], 16, 25),
    ("f16", (4, 2, 40, 48), [63], [30], 16, 0),
    ("bf16", (12, 4, 112, 112), [200], [3], 32, 0),
    ("f16", (4, 2, 160, 160), [40], [35], 16, 0),
    ("bf16", (4, 1, 200, 200), [90], [9], 16, 0),
    ("f16", (4, 2, 64, 128), [90], [9], 16, 0),
    ("bf16", (4, 2, 256, 144), [90], [9], 16, 0),
    ("q8_0", (12, 4, 96, 96), [100], [20], 16, 0),
    ("f16", (8, 2, 100, 100), [120], [5], 16, 0),
    ("bf16", (8, 2, 64, 64), [61], [20], 8, 0),
    ("f32", (4, 2, 50, 50), [61], [20], 16, 17),
    ("f16", (2, 1, 400, 320), [30], [5], 16, 0),
    ("q8_0", (4, 2, 64, 64), [30], [11], 4, 0),
    # groups wider than a unit, one head
    ("bf16", (71, 1, 64, 64), [90], [3], 16, 0),
    ("f16", (1, 1, 128, 128), [513], [2], 16, 0),
]
IDS = [f"{f[0]}-{'x'.join(map(str, f[1]))}-{'_'.join(map(str, f[3]))}-bt{f[4]}" + (f"-w{f[5]}" if f[5] else "") for f in FORMS]


@pytest.mark.parametrize("kind", [None, "prefix", "documents", "random"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_scores_and_ranges(form, kind):
    kv, geo, prior, new, bt, window = form
    c = Call(kv, geo, prior, new, bt)
    r = ranges_of(kind, c.segs)
    sl = slopes_of(geo[0])
    for kw in ({}, {"cap": 5.0}, {"slopes": sl}, {"cap": 30.0, "slopes": sl}):
        if kind is None or kw:
            kw = dict(kw, window=window, ranges=r)
            c.check(c.run(**kw), **kw)


WIDTHS = [(kv, hd, hdv) for kv in ("f16", "bf16") for hd, hdv in ((32, 32), (64, 64), (96, 96), (128, 128), (192, 192), (256, 256), (192, 128),
                                                                   (40, 40), (80, 80), (120, 112), (160, 160), (240, 256))] + \
    [("q8_0", d, d) for d in (64, 128, 192, 256)] + [("f32", d, d) for d in (60, 128, 200)]


@pytest.mark.parametrize("new", [1, 15])
@pytest.mark.parametrize("kv,hd,hdv", WIDTHS)
def test_every_width(kv, hd, hdv, new):
    """One column block (a decode row) and two (a run of drafted tokens) of every instance."""
    c = Call(kv, (8, 2, hd, hdv), [83, 5], [new, new], seed=31)
    r = ranges_of("random", c.segs, seed=32)
    sl = slopes_of(8)
    c.check(c.run(cap=6.0, slopes=sl), cap=6.0, slopes=sl)
    c.check(c.run(ranges=r), ranges=r)


@pytest.mark.parametrize("kind", ["one", "none"])
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_rows_that_see_one_key_or_none(form, kind):
    kv, geo, prior, new, bt, _ = form
    c = Call(kv, geo, prior, new, bt, seed=1)
    r = ranges_of(kind, c.segs, seed=2)
    c.check(c.run(cap=4.0, ranges=r), cap=4.0, ranges=r)


LONG = [("f16", (32, 8, 128, 128), [9000], [1]), ("bf16", (12, 2, 128, 128), [20000, 40], [3, 1]), ("q8_0", (64, 8, 128, 128), [8000], [1]),
        ("f32", (16, 2, 128, 128), [7000], [1]), ("f16", (4, 1, 80, 80), [12000], [2]), ("bf16", (4, 2, 256, 256), [6000], [4]),
        ("q8_0", (4, 1, 96, 96), [5000], [1]), ("bf16", (71, 1, 64, 64), [9000], [2])]


@pytest.mark.parametrize("kv,geo,prior,new", LONG, ids=[f"{f[0]}-{'x'.join(map(str, f[1]))}" for f in LONG])
def test_long_contexts_in_pieces(kv, geo, prior, new):
    """Units cut into key pieces, whose partials a merge launch combines: rows that see all of them, one, or none."""
    c = Call(kv, geo, prior, new)
    sl = slopes_of(geo[0], 2.0 ** -9)
    c.check(c.run(slopes=sl, cap=50.0), slopes=sl, cap=50.0)
    lo = [max(0, p + j - 70 * (j + 1)) for p, n in zip(prior, new) for j in range(n)]
    r = RowRanges(lo, None)
    c.check(c.run(slopes=sl, ranges=r), slopes=sl, ranges=r)
    # a row of all its keys beside rows that see the first key, the last one or nothing
    hi = [p + n for p, n in zip(prior, new) for _ in range(n)]
    edge = [0, hi[0] - 1, hi[0], 0]
    r = RowRanges([0] + [edge[i % 4] for i in range(1, c.n_rows)], [hi[0]] + [1 if i % 4 == 0 else hi[i] for i in range(1, c.n_rows)])
    c.check(c.run(cap=20.0, ranges=r), cap=20.0, ranges=r)


@pytest.mark.parametrize("kv,geo,prior,new,kind", [
    ("bf16", (32, 8, 128, 128), [0, 0], [700, 333], "prefix"), ("f16", (16, 4, 64, 64), [0], [2500], "documents"),
    ("q8_0", (8, 2, 128, 128), [130], [600], "prefix"), ("bf16", (8, 2, 256, 256), [0, 100], [500, 300], "prefix"),
    ("f16", (8, 8, 80, 80), [0], [900], "documents"), ("f32", (8, 2, 64, 64), [0], [600], "prefix")])
def test_prompts(kv, geo, prior, new, kind):
    """Prompts of hundreds of rows: several rounds of units, checked on rows spread over them."""
    c = Call(kv, geo, prior, new)
    r = ranges_of(kind, c.segs, seed=5)
    rows = sorted(set(list(range(0, max(new), 37)) + [n - 1 for n in new] + [0, 1]))
    c.check(c.run(cap=30.0, ranges=r), cap=30.0, ranges=r, rows=rows)
    sl = slopes_of(geo[0])
    c.check(c.run(slopes=sl, ranges=r), slopes=sl, ranges=r, rows=rows)


UNSEEN = [f for f in FORMS if f[2] in ([0, 31, 32, 900], [0, 15, 16, 17, 700], [0, 500, 33], [30, 200], [63], [33, 200], [100, 3],
                                       [0, 40, 15], [100], [120], [5], [61], [15], [47])]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("form", UNSEEN, ids=[f"{f[0]}-{'x'.join(map(str, f[1]))}-{'_'.join(map(str, f[3]))}-bt{f[4]}" for f in UNSEEN])
def test_what_a_row_does_not_see_may_hold_anything(form, bad):
    """Keys of sequence 0 that its rows do not see are not finite: before the range, after it, and between."""
    kv, geo, prior, new, bt, _ = form
    c = Call(kv, geo, prior, new, bt, seed=3)
    total = prior[0] + new[0]
    hide = sorted({0, total // 3, total - 1}) if total > 3 else [0]
    r = ranges_of("random", c.segs, seed=4)
    for t in range(new[0]):   # sequence 0's rows see a gap between hidden keys
        gaps = [(a + 1, b) for a, b in zip([-1] + hide, hide + [total])]
        r.lo[t], r.hi[t] = gaps[t % len(gaps)]
    clean = c.run(cap=9.0, ranges=r).clone()
    c.check(clean, cap=9.0, ranges=r)
    for pos in hide:
        k, v = c.k[0][pos:pos + 1].clone(), c.v[0][pos:pos + 1].clone()
        if bad == bad or kv != "q8_0":   # (a q8_0 row of NaN has no code)
            k.fill_(bad)
            v.fill_(bad)
        else:
            k.fill_(3e38)
            v.fill_(3e38)
        c.hc.store(0, [(0, 0, 1, pos)], k, v)
    out = c.run(cap=9.0, ranges=r)
    assert torch.isfinite(out).all()
    c.check(out, cap=9.0, ranges=r)


@pytest.mark.parametrize("kv", ["f16", "bf16", "q8_0", "f32"])
def test_without_shaping_as_attend(kv):
    geo = (16, 4, 128, 128)
    c = Call(kv, geo, [40, 300], [20, 1])
    a, b = c.run(), torch.empty(c.n_rows, 16, 128, device="cuda")
    c.hc.attend(0, c.segs, c.q, b, 1 / 128 ** 0.5)
    torch.cuda.synchronize()
    # attend's Q on bf16 pages keeps 16 bits: scores of |s| <= 8 within 2^-13, outputs within 2^-12 max|v|
    assert (a - b).abs().max().item() <= 2.0 ** -12 * 5.5


def test_scales_and_slopes_of_any_sign():
    c = Call("f16", (8, 2, 128, 128), [100], [20], spread=8.0)
    sl = slopes_of(8) * torch.tensor([1.0, -1.0] * 4, device="cuda") * 0.01
    for kw in ({"scale": -0.1}, {"scale": 0.0}, {"scale": 0.3, "cap": 50.0}, {"scale": -0.3, "cap": 10.0}, {"slopes": sl},
               {"scale": 0.05, "slopes": sl, "cap": 20.0}):
        c.check(c.run(**kw), **kw)


@pytest.mark.parametrize("cap", [1e-3, 0.5, 1e4, 1e30])
def test_caps_far_below_and_above_the_scores(cap):
    for kv in ("f16", "f32", "q8_0"):
        c = Call(kv, (8, 2, 64, 64), [60], [9], spread=4.0)
        c.check(c.run(cap=cap), cap=cap)


def test_a_cap_holds_scores_that_would_overflow_the_exponential():
    c = Call("f32", (8, 2, 64, 64), [60], [9], spread=1e4)
    c.check(c.run(cap=50.0), cap=50.0)
    c.q.zero_()
    c.check(c.run(cap=50.0), cap=50.0)


def test_a_window_layer():
    c = Call("f16", (8, 2, 64, 64), [0], [90], window_layer=40)
    r = RowRanges.of(c.segs, documents=[[0, 30, 77]])
    c.check(c.run(window=40, ranges=r, cap=9.0), window=40, ranges=r, cap=9.0)
    r = RowRanges.of(c.segs, prefix=[60])
    c.check(c.run(window=25, ranges=r), window=25, ranges=r)
    for window in (0, 41):
        with pytest.raises(LmhError):
            c.run(window=window)


def test_arrays_at_any_float_address_and_nothing_behind_them():
    c = Call("bf16", (12, 4, 80, 80), [100, 30], [5, 40])
    q = torch.zeros(c.q.numel() + 3, device="cuda")
    q[1:1 + c.q.numel()] = c.q.flatten()
    out = torch.full((c.n_rows * 12 * 80 + 9,), 5.0, device="cuda")
    c.run(q=q[1:], out=out[3:], cap=3.0)
    want = c.run(cap=3.0)
    n = want.numel()
    assert torch.equal(out[3:3 + n].view_as(want), want)
    assert (out[:3] == 5.0).all() and (out[3 + n:] == 5.0).all()


def test_same_bits_again_and_on_another_stream():
    for kv, geo, prior, new in (("f16", (32, 8, 128, 128), [9000, 70], [1, 40]), ("q8_0", (4, 1, 96, 96), [3000], [2])):
        c = Call(kv, geo, prior, new)
        r = ranges_of("prefix", c.segs)
        a = c.run(cap=20.0, ranges=r)
        assert torch.equal(a, c.run(cap=20.0, ranges=r))
        s = torch.cuda.Stream()
        b = torch.empty_like(a)
        torch.cuda.synchronize()
        c.hc.attend_scored(0, c.segs, c.q, b, 1 / geo[2] ** 0.5, cap=20.0, ranges=r, stream=s)
        s.synchronize()
        assert torch.equal(a, b)


def test_many_calls_of_different_ranges_in_flight():
    """More calls than staging slots, enqueued without waiting: each has its own ranges."""
    c = Call("f16", (8, 2, 64, 64), [200], [30])
    ranges = [RowRanges([i] * 30, None) for i in range(40)]
    outs = [torch.empty(30, 8, 64, device="cuda") for _ in ranges]
    for r, o in zip(ranges, outs):
        c.hc.attend_scored(0, c.segs, c.q, o, 0.125, ranges=r)
    torch.cuda.synchronize()
    for r, o in zip(ranges, outs):
        c.check(o, scale=0.125, ranges=r, rows=[0, 29])


def test_refusals():
    c = Call("f16", (8, 2, 64, 64), [20], [4])
    n = c.n_rows
    for kw in ({"cap": -1.0}, {"cap": float("inf")}, {"cap": float("nan")}, {"scale": float("inf")}, {"scale": float("nan")},
               {"cap": 1e-38, "scale": 1e10}, {"cap": 3e38}, {"ranges": RowRanges(None, [25] * n)}):
        with pytest.raises(LmhError) as e:
            c.run(**kw)
        assert e.value.status == N.INVALID_ARGUMENT
    for kw in ({"ranges": RowRanges([0] * (n + 1), None)}, {"slopes": torch.zeros(7, device="cuda")}, {"slopes": torch.zeros(8)},
               {"slopes": torch.zeros(8, device="cuda", dtype=torch.float64)}):
        with pytest.raises(ValueError):
            c.run(**kw)
    out = torch.empty(n, 8, 64, device="cuda")
    with pytest.raises(LmhError):
        c.hc.attend_scored(1, c.segs, c.q, out, 1.0, slopes=torch.zeros(8, device="cuda"))   # no such layer
    with pytest.raises(LmhError):
        c.hc.attend_scored(0, [(0, 0, 13, 20)], c.q, out, 1.0)   # beyond the reserved blocks
    lib, p = N.lib(), N.ScoreParams(N.ABI_VERSION, 0, 1.0, 0.0, None, None, None, 0)
    import ctypes as C
    segs = Segments(c.segs)
    args = (c.hc.h, 0, segs.arr, segs.n, C.c_void_p(c.q.data_ptr()), C.c_void_p(out.data_ptr()))
    assert lib.lmh_attend_scored(*args, None, None) == N.INVALID_ARGUMENT
    for field, value in (("abi_version", 99), ("reserved0", 1), ("slopes", c.q.data_ptr() + 2)):
        bad = N.ScoreParams(N.ABI_VERSION, 0, 1.0, 0.0, None, None, None, 0)
        setattr(bad, field, value)
        assert lib.lmh_attend_scored(*args, C.byref(bad), None) == N.INVALID_ARGUMENT
    assert lib.lmh_attend_scored(None, *args[1:], C.byref(p), None) == N.INVALID_ARGUMENT
    assert lib.lmh_attend_scored(c.hc.h, 0, segs.arr, segs.n, None, args[5], C.byref(p), None) == N.INVALID_ARGUMENT
    assert lib.lmh_attend_scored(c.hc.h, 0, segs.arr, 0, None, None, C.byref(p), None) == N.OK   # no rows
    c.check(c.run(cap=2.0), cap=2.0)   # the handle still works


def test_capture_is_refused():
    c = Call("f16", (8, 2, 64, 64), [20], [4])
    out = c.run(cap=2.0)
    g = torch.cuda.CUDAGraph()
    refused = None
    with torch.cuda.graph(g):
        try:
            c.hc.attend_scored(0, c.segs, c.q, out, 0.125, cap=2.0)
        except LmhError as e:
            refused = e.status
        out.add_(0.0)
    assert refused == N.UNSUPPORTED
    torch.cuda.synchronize()
