"""lmh_attend_scored's work list on the CPU (lmh_plan_scored: the planner alone, no device), over rows that see
ranges of keys of their own: prefixes, documents, single keys, nothing. Every (row, query head) sits in one unit
(or one decode item of its row and KV head), and the waves of its unit, or of the unit's key pieces, walk every page
the row sees once; block ids carried in the records equal the table's; pieces have a merge over exactly their slots."""

import ctypes as C
import random

import numpy as np
import pytest

from llmario_amd import _native as N
from llmario_amd.kv import RowRanges
from test_plan import KV, NO_SLOT, contiguous_table


def scored_plan(kv, geo, bt, table, segs, lo, hi, window=0, n_cu=256, per_cu=8, whole=0):
    n_seqs, bps = table.shape
    tab = np.ascontiguousarray(table, dtype=np.int32)
    d = N.PlanDesc(N.ABI_VERSION, KV[kv], *geo, bt, n_cu, 0, n_seqs, bps, tab.ctypes.data_as(C.c_void_p),
                   window, 0.1, 0, N.AttendTuning(N.ABI_VERSION, 0, 0, 0, 0, 0, whole, 0))
    arr = (N.Seg * max(len(segs), 1))(*[N.Seg(*s) for s in segs])
    r = RowRanges(lo, hi)
    lo_p = C.cast(r.lo, C.c_void_p) if r.lo is not None else None
    hi_p = C.cast(r.hi, C.c_void_p) if r.hi is not None else None
    c, n_items, n_prompts = N.PlanWaveCounts(), N.u64(), N.u64()
    counts = (C.byref(c), C.byref(n_items), C.byref(n_prompts))
    rc = N.lib().lmh_plan_scored(C.byref(d), arr, len(segs), lo_p, hi_p, per_cu, None, 0, None, 0, None, 0, None, 0, *counts)
    if rc != N.OK and not (c.n_waves or n_items.value or n_prompts.value):
        return rc, None, None, None, None, c
    waves, items = np.zeros((c.n_waves, 10), np.uint32), np.zeros((n_items.value, 8), np.uint32)
    prompts = np.zeros((n_prompts.value, 10), np.uint32)
    merges = np.zeros((c.n_merges, 6), np.uint32)
    at = lambda a: a.ctypes.data_as(C.c_void_p)
    rc = N.lib().lmh_plan_scored(C.byref(d), arr, len(segs), lo_p, hi_p, per_cu, at(waves), len(waves), at(items), len(items),
                                 at(prompts), len(prompts), at(merges), len(merges), *counts)
    return rc, waves, items, prompts, merges, c


def seen(segs, lo, hi, window):
    """(sequence, position, first key, key after the last) of every row."""
    out = []
    for s, _, n, p0 in segs:
        for pos in range(p0, p0 + n):
            t = len(out)
            a = max(lo[t] if lo is not None else 0, pos + 1 - window if window and pos + 1 > window else 0)
            out.append((s, pos, a, hi[t] if hi is not None else pos + 1))
    return out


def check(kv, geo, bt, table, segs, lo, hi, window, waves, items, prompts, merges, c):
    n_head, n_kv, _, _ = geo
    group, rows = n_head // n_kv, seen(segs, lo, hi, window)
    step = 1 if kv == "f32" else 2
    pages = {}     # (row, head) -> pages its unit's waves walk
    slots = {}     # (row, head) -> slots its pieces leave
    W, at = c.waves_per_wg, 0
    assert not (len(waves) + len(prompts) and len(items)) and (len(waves) == 0 or len(waves) % W == 0)
    while at < len(waves):
        seq, row0, pos0, page0, _, slot, _, _, head, cols = (int(x) for x in waves[at])
        n = cols >> 16 & 0xFF
        if n == 0:
            assert not waves[at].any()
            at += 1
            continue
        assert at // W == (at + n - 1) // W and (n == 1 or c.shared)
        page = page0
        for j in range(n):
            r = [int(x) for x in waves[at + j]]
            assert (r[0], r[1], r[2], r[5], r[8]) == (seq, row0, pos0, slot, head) and r[9] == (cols & ~0xFF00) | j << 8
            assert r[3] == page and r[4] > 0 and (j + 1 == n or r[4] % step == 0)
            assert r[6] == table[seq, page * 16 // bt] >= 0 and r[7] == table[seq, min(page + 1, page + r[4] - 1) * 16 // bt] >= 0
            page += r[4]
        assert table[seq, (page - 1) * 16 // bt] >= 0
        kvh, c_off, n_col, k = head & 0xFFFF, head >> 16, cols & 0xFF, cols >> 24
        assert 0 < n_col <= 16 * c.col_blocks and (k > 1) == (slot != NO_SLOT)
        for col in range(c_off, c_off + n_col):
            t, h = row0 + col // group, kvh * group + col % group
            assert rows[t][0] == seq and rows[t][1] == pos0 + col // group
            pages.setdefault((t, h), []).append((page0, page))
            if k:
                assert slot + (col // group) * k < c.slots
                slots.setdefault((t, h), []).append(slot + (col // group) * k)
        at += n
    cols = 256 if geo[2] == 128 else 128
    assert all(int(a[7]) + 3 >= int(b[7]) for a, b in zip(prompts, prompts[1:]))   # the longest first (in 64-key tiles)
    for u in prompts:
        seq, kvh, row0, pos0, c_off, n_col, page0, n_pages, slot, k = (int(x) for x in u)
        assert 0 < n_col <= cols and n_pages > 0 and (k > 1) == (slot != NO_SLOT)
        assert all(table[seq, p * 16 // bt] >= 0 for p in (page0, page0 + n_pages - 1))
        for col in range(c_off, c_off + n_col):
            t, h = row0 + col // group, kvh * group + col % group
            assert rows[t][0] == seq and rows[t][1] == pos0 + col // group
            pages.setdefault((t, h), []).append((page0, page0 + n_pages))
            if k:
                assert slot + (col // group) * k < c.slots
                slots.setdefault((t, h), []).append(slot + (col // group) * k)
    for it in items:
        row, kvh, h0, p0, p1, slot, seq, blk0 = (int(x) for x in it)
        assert seq == rows[row][0] and blk0 == table[seq, p0 // 16 * 16 // bt] >= 0
        assert p0 == p1 or rows[row][2] <= p0 < p1 <= rows[row][3]
        for h in range(h0, min(h0 + c.ng, group)):
            pages.setdefault((row, kvh * group + h), []).append((p0, p1))
            if slot != NO_SLOT:
                slots.setdefault((row, kvh * group + h), []).append(slot)
    merged = {}
    for row, kvh, h0, slot0, n_split, nh in (tuple(int(x) for x in m) for m in merges):
        for h in range(h0, min(h0 + (nh or c.ng), group)):
            assert (row, kvh * group + h) not in merged
            merged[(row, kvh * group + h)] = list(range(slot0, slot0 + n_split))
    assert {k: sorted(v) for k, v in slots.items()} == merged
    for t, (_, pos, a, b) in enumerate(rows):
        for h in range(n_head):
            got = sorted(pages[(t, h)])
            assert all(x[1] == y[0] for x, y in zip(got, got[1:])), (t, h, got)   # in a row, none twice
            if a < b and len(items):
                assert got[0][0] == a and got[-1][1] == b
            elif a < b:
                assert got[0][0] * 16 <= a and got[-1][1] * 16 >= b, (t, h, got, a, b)
            if len(waves) and len(rows) * group == 1 and a < b:   # a unit walks no page that none of its columns sees
                assert got[0][0] == a // 16 and got[-1][1] == (b - 1) // 16 + 1


GEOS = [("f16", (32, 8, 128, 128)), ("bf16", (16, 4, 256, 256)), ("q8_0", (8, 8, 64, 64)), ("f32", (12, 4, 64, 64)),
        ("f16", (32, 32, 80, 80)), ("bf16", (40, 8, 128, 128)), ("q8_0", (6, 2, 96, 96)), ("f16", (8, 1, 300, 300)),
        ("bf16", (71, 1, 64, 64)), ("f16", (1, 1, 128, 128))]
BATCHES = [([255], [1]), ([0], [1]), ([15, 16, 17, 700], [1, 1, 1, 1]), ([0, 40], [300, 57]), ([500, 3000, 9], [1, 70, 1]),
           ([9000], [1]), ([20000, 3], [5, 2]), ([0], [2000])]


def make_ranges(kind, segs, seed):
    rng = random.Random(seed)
    if kind == "prefix":
        return RowRanges.of(segs, prefix=[rng.randint(0, p + n) for _, _, n, p in segs])
    if kind == "documents":
        return RowRanges.of(segs, documents=[sorted(rng.sample(range(p + n), min(p + n, rng.randint(1, 6)))) for _, _, n, p in segs])
    lo, hi = [], []
    for _, _, n, p in segs:
        for pos in range(p, p + n):
            a = rng.randint(0, p + n)
            if kind == "one":
                a = min(a, p + n - 1)
            lo.append(a)
            hi.append(a + 1 if kind == "one" else a if kind == "none" else rng.randint(0, p + n))
    return RowRanges(lo, hi)


@pytest.mark.parametrize("kind", ["none", "one", "random", "prefix", "documents", "causal"])
@pytest.mark.parametrize("kv,geo", GEOS, ids=[f"{k}-{'x'.join(map(str, g))}" for k, g in GEOS])
def test_every_row_walks_what_it_sees(kv, geo, kind):
    for b, (prior, new) in enumerate(BATCHES):
        for bt in (16, 64, 4):
            if bt == 4 and sum(new) > 400:
                continue
            segs, start = [], 0
            for s, (p, n) in enumerate(zip(prior, new)):
                segs.append((s, start, n, p))
                start += n
            table = contiguous_table([p + n for p, n in zip(prior, new)], bt)
            r = RowRanges() if kind == "causal" else make_ranges(kind, segs, b)
            lo, hi = (None if x is None else list(x) for x in (r.lo, r.hi))
            for window, n_cu, per_cu, whole in ((0, 256, 8, 0), (333, 80, 4, 0), (0, 12, 16, 1)):
                rc, waves, items, prompts, merges, c = scored_plan(kv, geo, bt, table, segs, lo, hi, window, n_cu, per_cu, whole)
                assert rc == N.OK
                tiles = bt >= 16 and not (kv == "q8_0" and geo[2] == 96) and geo[2] <= 256
                assert (len(waves) + len(prompts) > 0) == tiles and (len(items) > 0) != tiles
                check(kv, geo, bt, table, segs, lo, hi, window, waves, items, prompts, merges, c)


def test_units_walk_their_documents_only():
    """Decode rows that see their last document, and packed documents: the pages walked are about those seen."""
    n = 48
    segs = [(i, i, 1, 8000) for i in range(n)]
    table = contiguous_table([8001] * n, 16)
    rc, waves, _, _, _, _ = scored_plan("bf16", (40, 8, 128, 128), 16, table, segs, [7900] * n, None)
    assert rc == N.OK and int(waves[:, 4].sum()) == n * 8 * (8000 // 16 - 7900 // 16 + 1)
    r = RowRanges.of([(0, 0, 8192, 0)], documents=[list(range(0, 8192, 512))])
    table = contiguous_table([8192], 16)
    rc, waves, _, prompts, _, c = scored_plan("f16", (16, 4, 64, 64), 16, table, [(0, 0, 8192, 0)], list(r.lo), list(r.hi))
    assert rc == N.OK and len(waves) == 0 and len(prompts) == 4 * 8192 // 32   # 128 columns of a group of 4: 32 rows a unit
    assert int(prompts[:, 7].sum()) == 4 * 16 * sum(2 * (i + 1) for i in range(16))


def test_refused_ranges():
    table = contiguous_table([21, 21], 16)
    segs = [(0, 0, 4, 17), (1, 4, 1, 9)]
    geo = (8, 2, 64, 64)
    assert scored_plan("f16", geo, 16, table, segs, None, [18, 21, 21, 21, 10])[0] == N.OK
    assert scored_plan("f16", geo, 16, table, segs, None, [18, 22, 21, 21, 10])[0] == N.INVALID_ARGUMENT   # past its segment
    assert scored_plan("f16", geo, 16, table, segs, None, [18, 21, 21, 21, 11])[0] == N.INVALID_ARGUMENT
    assert scored_plan("f16", geo, 16, table, segs, [0xffffffff] * 5, None)[0] == N.OK                    # sees nothing
    with pytest.raises(ValueError):
        RowRanges([1, 2], [3])
    with pytest.raises(ValueError):
        RowRanges([-1], [3])
    with pytest.raises(ValueError):
        RowRanges.of([(0, 0, 4, 17)], prefix=[22])


def test_row_ranges_of_a_batch():
    r = RowRanges.of([(0, 0, 5, 2), (1, 5, 3, 0)], prefix=[4, None], documents=[[0, 3, 6], None])
    assert list(r.lo) == [0, 3, 3, 3, 6, 0, 0, 0]
    assert list(r.hi) == [3, 4, 5, 6, 7, 1, 2, 3]     # the prefix ends at its row's document
    r = RowRanges.of([(0, 0, 5, 2)], prefix=[5])
    assert list(r.lo) == [0] * 5 and list(r.hi) == [5, 5, 5, 6, 7]
