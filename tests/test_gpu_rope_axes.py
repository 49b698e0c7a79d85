"""lmh_qk_rope_store_axes against its definition in 64 bits: positions of one to four axes, sections one after the
other or by turns, frequencies of the whole rotation or of each axis, every page type and kernel (aligned runs, single
rows, widths off the fast paths), and together with lmh_attend_scored over several steps.

Tolerance: with norm weights near 1 the norm is off by at most (hd / 64 + 8) 2^-24 of a value, cos and sin by 2^-23
(their argument's rounding, 2^-24 of half a turn times pi, and their own) plus 2^-24 for attn_factor, the two products
and their sum by 2^-23: Q within (hd / 64 + 20) 2^-24 of the pair's norm. K on 16-bit pages adds half a step of the
type; on q8_0 half a code, amax / 254, and the scale's own 2^-11."""

import math

import numpy as np
import pytest
import torch

from llmario_amd import _native as N
from llmario_amd.kv import HipKvCache, Layer, LmhError, RowRanges

pytestmark = pytest.mark.gpu


def axis_of(sections, interleaved):
    n = len(sections)
    if not interleaved:
        return [a for a in range(n) for _ in range(sections[a])]
    return [i % n if i % n and i < n * sections[i % n] else 0 for i in range(sum(sections))]


def rotate64(x, w, pos, sections, *, rot, theta, neox, interleaved=False, own_freq=False, freq_scale=1.0, attn_factor=1.0,
             freq_div=None, eps=1e-6):
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    y, axes, seen = x.copy(), axis_of(sections, interleaved), [0] * len(sections)
    for i, a in enumerate(axes):
        e = -seen[a] / sections[a] if own_freq else -2.0 * i / rot
        seen[a] += 1
        # (the angle is the position times a frequency given in f32 parameters; exact in 64 bits to 2^-20 of a turn at 2^31)
        ang = pos[a].astype(np.float64) * float(np.float32(freq_scale)) * float(np.float32(theta)) ** e
        if freq_div is not None:
            ang = ang / float(np.float32(freq_div[i]))
        c, s = (np.cos(ang) * float(np.float32(attn_factor)))[:, None], (np.sin(ang) * float(np.float32(attn_factor)))[:, None]
        p, q = (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)
        y[..., p], y[..., q] = x[..., p] * c - x[..., q] * s, x[..., p] * s + x[..., q] * c
    return y


def grid_positions(n, axes, seed, far=0):
    rng = np.random.default_rng(seed)
    pos = np.empty((axes, n), np.int32)
    for a in range(axes):
        pos[a] = far + rng.integers(0, 3 * n + 40, n)
    return pos


def run(kv, heads, n_kv, hd, prior, new, sections, *, bt=16, rot=0, neox=False, norm=False, seed=0, far=0, q_stride=0, freq_div=None, **kw):
    rng = np.random.default_rng(seed)
    rot = rot or hd
    hc = HipKvCache([Layer(heads, n_kv, hd, hd)], max_ctx=max(p + n for p, n in zip(prior, new)) + bt, n_seqs=len(prior), kv_type=kv,
                    block_tokens=bt)
    segs, at = [], 0
    for s, (p, n) in enumerate(zip(prior, new)):
        hc.reserve(s, p + n)
        segs.append((s, at, n, p))
        at += n
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    q = rng.standard_normal((at, heads, q_stride or hd)).astype(np.float32)
    k, v = (rng.standard_normal((at, n_kv, hd)).astype(np.float32) for _ in range(2))
    wq, wk = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)) if norm else (None, None)
    pos = grid_positions(at, len(sections), seed + 1, far)
    q_out = torch.full((at, heads, hd), 9.0, device="cuda")
    hc.qk_rope_store_axes(0, segs, dev(q), dev(k), dev(v), q_out, dev(pos), sections, rot_dim=rot, neox=neox, q_stride=q_stride,
                          q_norm=dev(wq) if norm else None, k_norm=dev(wk) if norm else None,
                          freq_div=dev(freq_div) if freq_div is not None else None, **kw)
    k_got, v_got = (torch.empty(at, n_kv, hd, device="cuda") for _ in range(2))
    hc.gather(0, segs, k_got, v_got)
    torch.cuda.synchronize()
    opt = dict(rot=rot, neox=neox, freq_div=freq_div, theta=kw.get("theta", 10000.0), interleaved=kw.get("interleaved", False),
               own_freq=kw.get("own_freq", False), freq_scale=kw.get("freq_scale", 1.0), attn_factor=kw.get("attn_factor", 1.0))
    factor = max(1.0, abs(opt["attn_factor"]))
    for got, x, w, is_q in ((q_out, q[..., :hd], wq, True), (k_got, k, wk, False)):
        want = rotate64(x, w, pos, sections, **opt)
        size = np.abs(x if w is None else want).max(-1, keepdims=True) * 1.5 * factor   # a pair's norm is at most sqrt 2 of the largest
        tol = (hd / 64 + 20) * 2.0 ** -24 * size
        if not is_q:
            tol = held(want, tol, kv)
        d = np.abs(got.double().cpu().numpy() - want)
        assert (d <= tol).all(), (is_q, float((d / tol).max()), np.unravel_index((d / tol).argmax(), d.shape))
    tol = held(v.astype(np.float64), np.zeros_like(v[..., :1], dtype=np.float64), kv)
    assert (np.abs(v_got.double().cpu().numpy() - v) <= tol).all()


def held(want, tol, kv):
    """The tolerance of values that are `tol` off and then held in the pages' type."""
    if kv == "q8_0":
        b = np.abs(want).reshape(*want.shape[:-1], -1, 32)
        amax = b.max(-1, keepdims=True)
        step = (amax / 254 + amax * 2.0 ** -11 + 2.0 ** -24 * 127) * np.ones_like(b)
        return step.reshape(want.shape) * 1.001 + 2 * tol
    half = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}[kv]
    return (np.abs(want) + tol) * half + tol + (2.0 ** -25 if kv == "f16" else 0.0)


KINDS = [("f16", 128, 16), ("bf16", 128, 16), ("q8_0", 128, 32), ("f32", 128, 16), ("f16", 64, 16), ("bf16", 256, 16), ("q8_0", 64, 16),
         ("f32", 256, 16), ("f16", 96, 16), ("bf16", 80, 16), ("q8_0", 96, 16), ("f32", 64, 4), ("bf16", 192, 16), ("f16", 512, 16), ("bf16", 32, 16)]


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("kv,hd,bt", KINDS)
def test_three_axes(kv, hd, bt, neox):
    """Runs of four aligned tokens, unaligned edges and single rows; sections in turn and interleaved."""
    half = hd // 2
    third = half // 3
    for norm, prior, new in ((False, [0], [1]), (True, [3, 16], [1, 1]), (True, [0, 5], [9, 30]), (False, [2, 8, 100], [70, 1, 4])):
        run(kv, 8, 2, hd, prior, new, [half - 2 * third, third, third], bt=bt, neox=neox, norm=norm)
        run(kv, 8, 2, hd, prior, new, [half - 2 * third, third, third], bt=bt, neox=neox, norm=norm, interleaved=True, theta=1e6)


@pytest.mark.parametrize("sections,rot,kw", [
    ([64], 128, {}), ([32, 32], 128, {}), ([16, 16, 16, 16], 128, {}), ([0, 64], 128, {}), ([40, 0, 24], 128, {}), ([8, 12, 12], 64, {}),
    ([11, 21, 32], 128, {"own_freq": True}), ([16, 16], 64, {"own_freq": True, "interleaved": True}), ([22, 21, 21], 128, {"interleaved": True}),
    ([44, 20, 0], 128, {"interleaved": True}), ([16, 16, 16, 16], 128, {"interleaved": True}), ([1, 1, 1], 6, {}), ([3, 1, 1], 10, {"interleaved": True}),
    ([24, 20, 20], 128, {"freq_scale": 0.25, "attn_factor": 1.2}), ([64], 128, {"interleaved": True})])
@pytest.mark.parametrize("neox", [False, True])
def test_axes_and_sections(sections, rot, kw, neox):
    run("bf16", 6, 2, 128, [7], [21], sections, rot=rot, neox=neox, **kw)


def test_frequency_divisors_and_a_wider_query():
    div = (1.0 + np.arange(64) / 7.0).astype(np.float32)
    run("f16", 6, 2, 128, [7], [21], [24, 20, 20], freq_div=div, neox=True)
    run("f32", 6, 2, 128, [0], [40], [24, 20, 20], q_stride=256, norm=True)


@pytest.mark.parametrize("far", [1000000, 2000000000, -5000])
def test_far_and_negative_positions(far):
    """Angles of far positions are formed in 64 bits. (Positions of 2^31 turn a pair by up to 3.4e8 turns: 2^-24 of one.)"""
    for hd in (128, 80):
        run("f32", 4, 2, hd, [0], [12], [hd // 4, hd // 4], far=far, neox=True)


def test_axes_alike_turn_as_the_sequence_position_does():
    """Every axis holding the sequence position: lmh_qk_rope_store, but for the rounding of its f32 angles, which at
    positions under 100 is below 100 * 2^-23 in the first pair."""
    hc = HipKvCache([Layer(8, 2, 128, 128)] * 2, max_ctx=128, n_seqs=1, kv_type="f32")
    hc.reserve(0, 100)
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(100, h, 128, device="cuda", generator=g) for h in (8, 2, 2))
    pos = torch.arange(100, dtype=torch.int32, device="cuda").repeat(3, 1).contiguous()
    a, b = torch.empty_like(q), torch.empty_like(q)
    hc.qk_rope_store_axes(0, [(0, 0, 100, 0)], q, k, v, a, pos, [24, 20, 20])
    hc.qk_rope_store(1, [(0, 0, 100, 0)], q, k, v, b)
    torch.cuda.synchronize()
    assert (a - b).abs().max().item() <= 100 * 2.0 ** -23 * 1.5 * q.abs().max().item()


def test_refusals():
    hc = HipKvCache([Layer(8, 2, 128, 128)], max_ctx=64, n_seqs=1, kv_type="f16")
    hc.reserve(0, 20)
    q, k, v = (torch.randn(4, h, 128, device="cuda") for h in (8, 2, 2))
    out, pos = torch.empty_like(q), torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    segs = [(0, 0, 4, 3)]
    ok = dict(positions=pos, sections=[24, 20, 20])
    hc.qk_rope_store_axes(0, segs, q, k, v, out, **ok)
    for bad in (dict(sections=[24, 20, 21]), dict(sections=[24, 20, 19]), dict(sections=[20, 22, 22], interleaved=True), dict(theta=0.0),
                dict(theta=float("inf")), dict(theta=-2.0), dict(freq_scale=float("nan")), dict(rot_dim=130), dict(rot_dim=3)):
        with pytest.raises(LmhError) as e:
            hc.qk_rope_store_axes(0, segs, q, k, v, out, **{**ok, **bad})
        assert e.value.status == N.INVALID_ARGUMENT
    for bad in (dict(positions=pos[:2].contiguous()), dict(positions=pos.long()), dict(positions=pos.cpu()), dict(positions=pos.t()),
                dict(sections=[16] * 5), dict(sections=[]), dict(sections=[-1, 30, 35])):
        with pytest.raises(ValueError):
            hc.qk_rope_store_axes(0, segs, q, k, v, out, **{**ok, **bad})
    import ctypes as C
    lib, seg = N.lib(), (N.Seg * 1)(N.Seg(0, 0, 4, 3))
    at = lambda t: C.c_void_p(t.data_ptr())

    def call(axes, flags=N.ROPE_APPLY):
        p = N.RopeParams(N.ABI_VERSION, flags, 128, 0, 1e-6, 10000.0, 1.0, 1.0, None, None, None)
        return lib.lmh_qk_rope_store_axes(hc.h, 0, seg, 1, at(q), at(k), at(v), at(out), C.byref(p), C.byref(axes) if axes else None, None)

    def axes(**kw):
        x = N.RopeAxes(N.ABI_VERSION, 3, 0, (N.u32 * 4)(24, 20, 20, 0), 0, pos.data_ptr())
        for f, value in kw.items():
            setattr(x, f, value)
        return x

    assert call(axes()) == N.OK
    assert call(None) == N.INVALID_ARGUMENT and call(axes(), flags=0) == N.INVALID_ARGUMENT
    for kw in (dict(abi_version=99), dict(n_axes=0), dict(n_axes=5), dict(n_axes=2), dict(flags=4), dict(reserved0=1), dict(positions=None),
               dict(positions=pos.data_ptr() + 2), dict(sections=(N.u32 * 4)(24, 20, 0, 20)), dict(sections=(N.u32 * 4)(0xffffffff, 65, 0, 0))):
        assert call(axes(**kw)) == N.INVALID_ARGUMENT, kw


def test_capture_is_refused():
    hc = HipKvCache([Layer(8, 2, 128, 128)], max_ctx=64, n_seqs=1, kv_type="f16")
    hc.reserve(0, 4)
    q, k, v = (torch.randn(4, h, 128, device="cuda") for h in (8, 2, 2))
    out, pos = torch.zeros_like(q), torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    hc.qk_rope_store_axes(0, [(0, 0, 4, 0)], q, k, v, out, pos, [24, 20, 20])
    torch.cuda.synchronize()
    refused = None
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        try:
            hc.qk_rope_store_axes(0, [(0, 0, 4, 0)], q, k, v, out, pos, [24, 20, 20])
        except LmhError as e:
            refused = e.status
        out.add_(0.0)
    assert refused == N.UNSUPPORTED


def test_another_rotation_after_one_and_back():
    """The table of turns kept from the latest call is not another rotation's."""
    hc = HipKvCache([Layer(8, 2, 128, 128)], max_ctx=64, n_seqs=1, kv_type="f32")
    hc.reserve(0, 40)
    q, k, v = (torch.randn(40, h, 128, device="cuda") for h in (8, 2, 2))
    pos = torch.randint(0, 500, (3, 40), dtype=torch.int32, device="cuda")
    outs = []
    for kw in ({}, {"theta": 1e6}, {"freq_scale": 0.5}, {"rot_dim": 64, "sections": [12, 10, 10]}, {"interleaved": True, "sections": [22, 21, 21]},
               {"sections": [20, 22, 22]}, {"own_freq": True}, {}):
        out = torch.empty_like(q)
        hc.qk_rope_store_axes(0, [(0, 0, 40, 0)], q, k, v, out, pos, **{"sections": [24, 20, 20], **kw})
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[-1])
    assert all(not torch.equal(outs[0], o) for o in outs[1:-1])


@pytest.mark.parametrize("kv", ["f16", "bf16", "f32"])
def test_an_image_prompt_and_its_answer(kv):
    """Both operators as a layer runs them: a prompt of text and an image (positions of three axes, the prefix's tokens
    see each other), then tokens decoded one by one at positions that go on after the image's, through the cache, against
    the same in 64 bits on the K and V that the pages hold."""
    heads, n_kv, hd, n, steps = 8, 2, 128, 75, 3
    rng = np.random.default_rng(8)
    hc = HipKvCache([Layer(heads, n_kv, hd, hd)], max_ctx=128, n_seqs=1, kv_type=kv)
    pos = np.concatenate([np.tile(np.arange(5), (3, 1)), np.stack([np.full(60, 5), 5 + np.arange(60) // 10, 5 + np.arange(60) % 10]),
                          np.tile(15 + np.arange(10), (3, 1))], axis=1).astype(np.int32)
    prefix, cap, scale = 65, 30.0, hd ** -0.5
    done = 0
    for new in [n] + [1] * steps:
        segs, n_rows = hc.prepare_batch([(0, new)])
        q, k, v = (torch.from_numpy(rng.standard_normal((new, h, hd)).astype(np.float32)).cuda() for h in (heads, n_kv, n_kv))
        p = pos if done == 0 else np.full((3, 1), 25 + done - n, np.int32)
        q_out, out = torch.empty_like(q), torch.empty_like(q)
        hc.qk_rope_store_axes(0, segs, q, k, v, q_out, torch.from_numpy(p).cuda(), [24, 20, 20], neox=True)
        r = RowRanges.of(segs, prefix=[prefix]) if done == 0 else None
        hc.attend_scored(0, segs, q_out, out, scale, cap=cap, ranges=r)
        hc.commit_batch(segs)
        ks, vs = (torch.empty(done + new, n_kv, hd, device="cuda") for _ in range(2))
        hc.gather(0, [(0, 0, done + new, 0)], ks, vs)
        torch.cuda.synchronize()
        want_q = rotate64(q.cpu().numpy(), None, p, [24, 20, 20], rot=hd, theta=10000.0, neox=True)
        assert np.abs(q_out.double().cpu().numpy() - want_q).max() <= 22 * 2.0 ** -24 * 1.5 * float(q.abs().max())
        ks, vs = ks.double().cpu().numpy(), vs.double().cpu().numpy()
        qs = q_out.double().cpu().numpy()
        for j in range(new):
            hi = max(done + j + 1, prefix) if done == 0 and j < prefix else done + j + 1
            for h in range(heads):
                s = cap * np.tanh(ks[:hi, h // 4] @ qs[j, h] * scale / cap)
                w = np.exp(s - s.max())
                want = (w / w.sum()) @ vs[:hi, h // 4]
                mag = (np.abs(ks[:hi, h // 4]) @ np.abs(qs[j, h])) * scale
                tol = (2 * (hd / 16 + 12) * 2.0 ** -24 * (mag.max() + np.abs(s).max() + 1) + 2.0 ** -20) * np.abs(vs[:hi]).max()
                assert np.abs(out[j, h].double().cpu().numpy() - want).max() <= tol
        done += new
    assert hc.len(0) == n + steps
