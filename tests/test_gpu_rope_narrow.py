"""lmh_qk_rope_store on heads narrower than a wave (under 64 dims), both pairings: Q and K against the rotation in 64
bits. At positions under 64 an f32 angle is off by at most 64 * 2^-23, the products by 2^-22 of the pair."""

import numpy as np
import pytest
import torch

from llmario_amd.kv import HipKvCache, Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("hd,rot", [(32, 32), (32, 16), (8, 8), (48, 48), (60, 20)])
def test_narrow_heads(hd, rot, neox):
    n, heads, n_kv = 37, 4, 2
    hc = HipKvCache([Layer(heads, n_kv, hd, hd)], max_ctx=64, n_seqs=1, kv_type="f32")
    hc.reserve(0, n)
    rng = np.random.default_rng(hd + rot)
    q, k, v = (rng.standard_normal((n, h, hd)).astype(np.float32) for h in (heads, n_kv, n_kv))
    dev = [torch.from_numpy(x).cuda() for x in (q, k, v)]
    q_out, k_out, v_out = (torch.empty_like(x) for x in dev)
    hc.qk_rope_store(0, [(0, 0, n, 0)], *dev, q_out, rot_dim=rot, neox=neox)
    hc.gather(0, [(0, 0, n, 0)], k_out, v_out)
    torch.cuda.synchronize()
    i = np.arange(rot // 2)
    ang = np.arange(n)[:, None] * 10000.0 ** (-2.0 * i / rot)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)
    for got, x in ((q_out, q), (k_out, k)):
        want = x.astype(np.float64)
        want[..., a], want[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
        assert np.abs(got.double().cpu().numpy() - want).max() <= (64 * 2.0 ** -23 + 2.0 ** -22) * 1.5 * np.abs(x).max()
    assert np.array_equal(v_out.cpu().numpy(), v)
