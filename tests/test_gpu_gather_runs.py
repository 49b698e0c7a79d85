"""Reads of 16-bit page tiles in runs (lmh_kv_gather, lmh_kv_gather_encoded): the rows stored, bit for bit, for runs that
begin and end inside a tile, single rows, several heads and widths, arrays of 16-byte alignment or not, and nothing
written past the rows."""

import pytest
import torch

from llmario_amd.kv import HipKvCache, Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f16", "bf16"])
@pytest.mark.parametrize("geo", [(4, 2, 128, 128), (8, 8, 64, 64), (3, 3, 96, 96), (2, 1, 256, 256), (4, 2, 192, 128), (6, 2, 32, 32)])
@pytest.mark.parametrize("bt", [16, 64])
def test_rows_come_back(kv, geo, bt):
    n_head, n_kv, hd, hdv = geo
    lens = [1, 100, 16, 37]
    hc = HipKvCache([Layer(*geo)] * 2, max_ctx=128, n_seqs=len(lens), kv_type=kv, block_tokens=bt)
    dt = torch.float16 if kv == "f16" else torch.bfloat16
    ks, vs = [], []
    for s, n in enumerate(lens):
        hc.reserve(s, n)
        ks.append(torch.randn(n, n_kv * hd, device="cuda"))
        vs.append(torch.randn(n, n_kv * hdv, device="cuda"))
        hc.store(1, [(s, 0, n, 0)], ks[s], vs[s])
    for picks in ([(1, 0, 100)], [(0, 0, 1), (3, 5, 1), (1, 15, 2), (2, 0, 16)], [(1, 3, 90), (3, 31, 6)]):
        segs, at = [], 0
        for s, p, n in picks:
            segs.append((s, at, n, p))
            at += n
        want_k = torch.cat([ks[s][p:p + n] for s, p, n in picks]).to(dt)
        want_v = torch.cat([vs[s][p:p + n] for s, p, n in picks]).to(dt)
        for off in (0, 8, 1):   # elements: 16-byte aligned rows, then not
            for enc in (True, False):
                t = dt if enc else torch.float32
                k, v = (torch.full((off + at * n_kv * d + 24,), 3.0, dtype=t, device="cuda") for d in (hd, hdv))
                (hc.gather_encoded if enc else hc.gather)(1, segs, k[off:], v[off:])
                torch.cuda.synchronize()
                for got, want in ((k, want_k), (v, want_v)):
                    end = off + want.numel()
                    assert torch.equal(got[off:end].to(dt).view_as(want), want)
                    assert (got[:off] == 3.0).all() and (got[end:] == 3.0).all()
