"""The rotary operator against float64: both layouts, parts of the head, types, strides, in place, far positions, and
as it is used: 4-bit projections, rotary and the attention between them."""
import math

import numpy as np
import pytest
import torch

from cleffa_amd import AttnPlan, Mx4Matrix, Rotary, TextAttention, mx4_gemm
from tests import mx4_ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
EPS = 1e-6


def _say(*a):
    print("[rotary]", *a, flush=True)


def _np(x):
    return x.detach().cpu().double().numpy()


def _turned(x, pos, f, layout, magnitude=1.0, norm=None):
    """float64 [T][heads][hd] turned, and the length of each dim's pair (of a dim that does not turn: its magnitude)."""
    n, hd = 2 * len(f), x.shape[2]
    if norm is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + EPS) * norm
    pos = pos.reshape(len(pos), -1)
    ang = np.array([[int(p[j % pos.shape[1]]) * f[j] for j in range(n // 2)] for p in pos])[:, None]
    i = np.arange(n // 2)
    a, b = (i, i + n // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y, size = x.copy(), np.abs(x)
    c, s = magnitude * np.cos(ang), magnitude * np.sin(ang)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = abs(magnitude) * np.hypot(x[..., a], x[..., b])
    return y, size


def _check(got, want, size, f, pos):
    """The angle's fraction of a turn goes to f32 (2^-25 turns, 2^-22 radians), sine and cosine are off by 2^-22 at most, the norm, its
    weight and the rotation round ten times at most (2^-24 each), f16's smallest step is 2^-24; the float64 angle of a far position is off
    by 2^-51 of itself in both."""
    far = np.abs(pos).max(initial=0) * f.max() * 2.0 ** -50
    lim = size * (2.0 ** -21 + 10 * 2.0 ** -24 + far)
    lim = lim + (np.abs(want) + lim) * HALF_STEP[got.dtype] + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    d = np.abs(_np(got) - want)
    assert (d <= lim).all(), f"{d.max()} off, {(d / np.maximum(lim, 1e-300)).max()} of what is allowed"


def _inputs(T, nh, nkv, hd, dtype, seed, norm=True):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q, k = (torch.randn(T, n, hd, generator=g, device="cuda").to(dtype) for n in (nh, nkv))
    w = [1 + 0.1 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)] if norm else [None, None]
    return q, k, w[0], w[1]


def _freq(n, theta=1e7):
    return theta ** (-2 * np.arange(n // 2) / n)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,n_rot", [(2, 2), (6, 4), (64, 64), (72, 72), (72, 36), (80, 40), (128, 128), (128, 2), (192, 64), (256, 64), (256, 256), (256, 250), (256, 34), (250, 250), (66, 64)])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_rotation(layout, hd, n_rot, norm):
    f = _freq(n_rot)
    for dtype in TYPES.values():
        T, nh, nkv = 5, 7, 3
        q, k, qw, kw = _inputs(T, nh, nkv, hd, dtype, hd + n_rot, norm)
        pos = torch.randint(0, 20000, (T,), dtype=torch.int32, device="cuda")
        _say(layout, hd, n_rot, dtype, norm)
        q_out, k_out = Rotary(n_rot, layout=layout).apply(q, k, pos, qw, kw)
        for x, out, w in ((q, q_out, qw), (k, k_out, kw)):
            want, size = _turned(_np(x), pos.cpu().numpy(), f, layout, norm=None if w is None else _np(w))
            _check(out, want, size, f, pos.cpu().numpy())
        # in place, the same bits
        q_in, k_in = q.clone(), k.clone()
        Rotary(n_rot, layout=layout).apply(q_in, k_in, pos, qw, kw, q_out=q_in, k_out=k_in)
        assert torch.equal(q_in, q_out) and torch.equal(k_in, k_out)
        if not norm and n_rot < hd:
            assert torch.equal(q_out[..., n_rot:], q[..., n_rot:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T", [0, 1, 3, 64, 1000])
def test_lengths_and_axes(layout, T):
    for axes in (1, 2, 3, 4):
        q, k, qw, kw = _inputs(T, 24, 4, 256, torch.bfloat16, T)
        pos = torch.randint(-50, 4000, (T, axes), dtype=torch.int32, device="cuda")
        _say("lengths", layout, T, axes)
        q_out, k_out = Rotary(64, layout=layout, axes=axes).apply(q, k, pos, qw, kw)
        for x, out, w in ((q, q_out, qw), (k, k_out, kw)):
            want, size = _turned(_np(x), pos.cpu().numpy(), _freq(64), layout, norm=_np(w)) if T else (np.zeros((0, x.shape[1], 256)),) * 2
            _check(out, want, size, _freq(64), pos.cpu().numpy())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_positions(layout):
    """Positions to the ends of int32: the whole turns drop out."""
    pos = torch.tensor([0, 1, -1, 130000, 1 << 20, 123456789, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32, device="cuda")
    q, k, _, _ = _inputs(len(pos), 3, 1, 64, torch.float32, 3, False)
    f = _freq(64, 1e4)
    q_out, k_out = Rotary(64, theta=1e4, layout=layout).apply(q, k, pos)
    for x, out in ((q, q_out), (k, k_out)):
        _check(out, *_turned(_np(x), pos.cpu().numpy(), f, layout), f, pos.cpu().numpy().astype(np.int64))
    # negated positions turn back
    p = torch.randint(0, 500000, (len(pos),), dtype=torch.int32, device="cuda")
    r = Rotary(64, theta=1e4, layout=layout)
    back, _ = r.apply(r.apply(q, None, p)[0], None, -p)
    size = np.hypot(_np(q), 0).max(-1, keepdims=True) * 2 ** 0.5
    assert (np.abs(_np(back) - _np(q)) <= 2 * size * 2.0 ** -20).all()


@pytest.mark.parametrize("scaling", [{"kind": "linear", "factor": 4}, {"kind": "base", "factor": 8.0}, {"kind": "parts", "factor": 16, "original": 4096},
                                     {"kind": "parts", "factor": 8, "original": 8192, "low": 1, "high": 4}])
def test_scaled(scaling):
    n, s = 64, scaling["factor"]
    f = _freq(n)
    if scaling["kind"] == "linear":
        f = f / s
    elif scaling["kind"] == "base":
        f = _freq(n, 1e7 * s ** (n / (n - 2)))
    else:
        r = scaling["original"] * f / (2 * math.pi)
        keep = np.clip((r - 1) / (scaling.get("high", 32) - 1), 0, 1)
        f = keep * f + (1 - keep) * f / s
    rotary = Rotary(n, scaling=scaling)
    assert rotary.magnitude == (0.1 * math.log(s) + 1 if scaling["kind"] == "parts" else 1)
    q, k, qw, kw = _inputs(9, 4, 2, 128, torch.float32, 5)
    pos = torch.randint(0, 200000, (9, 1), dtype=torch.int32, device="cuda")
    _say("scaled", scaling)
    q_out, _ = rotary.apply(q, k, pos, qw, kw)
    _check(q_out, *_turned(_np(q), pos.cpu().numpy(), f, "half", rotary.magnitude, _np(qw)), f, pos.cpu().numpy())
    table = Rotary(n, freqs=f, magnitude=rotary.magnitude)
    _check(table.apply(q, k, pos, qw, kw)[0], *_turned(_np(q), pos.cpu().numpy(), f, "half", rotary.magnitude, _np(qw)), f, pos.cpu().numpy())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lead", [0, 8, 3])
def test_strides(dtype, lead):
    """Heads inside wider rows, at odd elements, heads ahead of rows, one norm alone: what is not turned stays as it was."""
    T, nh, nkv, hd = 6, 5, 2, 64
    t = TYPES[dtype]
    g = torch.Generator(device="cuda")
    g.manual_seed(lead)
    rows = torch.randn(T, lead + (2 * nh + 2 * nkv) * hd + 16, generator=g, device="cuda").to(t)
    kept = rows.clone()
    pos = torch.arange(100, 100 + T, dtype=torch.int32, device="cuda")
    w = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
    r = Rotary(32, layout="half")
    q, k = Rotary.heads(rows[:, lead:], nh, nkv, hd)
    want_q, want_k = _turned(_np(q), pos.cpu().numpy(), _freq(32), "half"), _turned(_np(k), pos.cpu().numpy(), _freq(32), "half", norm=_np(w))
    _say("strides", dtype, lead)
    r.apply(q, k, pos, None, w, q_out=q, k_out=k)
    _check(q, *want_q, _freq(32), pos.cpu().numpy())
    _check(k, *want_k, _freq(32), pos.cpu().numpy())
    q0, k0 = Rotary.heads(kept[:, lead:], nh, nkv, hd)
    q.copy_(q0)
    k.copy_(k0)
    assert torch.equal(rows, kept)
    # [heads][T][hd] in and out
    qt = q0.transpose(0, 1).contiguous()
    out = torch.empty_like(qt)
    r.apply(qt.transpose(0, 1), None, pos, q_out=out.transpose(0, 1))
    _check(out.transpose(0, 1), *want_q, _freq(32), pos.cpu().numpy())


def test_bad_values_stay_in_their_pair_or_head():
    q, k, qw, kw = _inputs(4, 3, 1, 64, torch.bfloat16, 2)
    q[1, 2, 5], q[2, 0, 63] = float("nan"), float("inf")
    pos = torch.arange(1, 5, dtype=torch.int32, device="cuda")
    out = _np(Rotary(32, layout="half").apply(q, None, pos)[0])
    bad = ~np.isfinite(out)
    want = np.zeros_like(bad)
    want[1, 2, [5, 21]], want[2, 0, 63] = True, True
    assert np.array_equal(bad, want)
    normed = ~np.isfinite(_np(Rotary(32, layout="half").apply(q, None, pos, qw)[0]))
    assert normed[1, 2].all() and normed[2, 0, 63] and normed.any(-1).sum() == 2


def test_rows_beyond_32_bits():
    """2^20 rows of 4.5 GB, in place: the last ones and those across 2^32 bytes as a call on them alone."""
    T, nh, nkv, hd = 1 << 20, 14, 3, 128
    _say("large", T)
    qkv = torch.randn(T, (nh + 2 * nkv) * hd, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    r = Rotary(128, layout="interleaved", scaling={"kind": "linear", "factor": 8.0})
    q, k = r.heads(qkv, nh, nkv, hd, gated=False)
    at = [0, (1 << 32) // (2 * qkv.shape[1]) - 32, T - 64]
    want = [r.apply(q[t:t + 64].contiguous(), k[t:t + 64].contiguous(), pos[t:t + 64].contiguous()) for t in at]
    v = [qkv[t:t + 64, (nh + nkv) * hd:].clone() for t in at]
    r.apply(q, k, pos, q_out=q, k_out=k)
    for t, (wq, wk), wv in zip(at, want, v):
        assert torch.equal(q[t:t + 64], wq) and torch.equal(k[t:t + 64], wk) and torch.equal(qkv[t:t + 64, (nh + nkv) * hd:], wv)


def test_in_a_graph():
    q, k, qw, kw = _inputs(33, 24, 4, 256, torch.bfloat16, 4)
    pos = torch.arange(33, dtype=torch.int32, device="cuda")
    r = Rotary(64, layout="interleaved")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r.apply(q, k, pos, qw, kw, q_out=q_out, k_out=k_out)
    for i in range(3):
        pos.add_(1000)
        g.replay()
        want = r.apply(q, k, pos, qw, kw)
        torch.cuda.synchronize()
        assert torch.equal(q_out, want[0]) and torch.equal(k_out, want[1])


@pytest.mark.parametrize("four_bit", [True, False], ids=["x4", "xbf16"])
def test_a_layer(four_bit):
    """Quantised activations, the QKV product, norm and rotary in its rows, the attention without its own, and the output
    projection into the residual; beside it the same rows through the attention's own prologue."""
    nh, nkv, H, lens = 8, 2, 512, [70, 1, 133]
    T, cu = sum(lens), np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    att, plain = TextAttention(nh, nkv, n_rot=64), TextAttention(nh, nkv, n_rot=0)
    w_qkv = Mx4Matrix.quantised(torch.randn(att.row, H, generator=g, device="cuda") / H ** 0.5)
    w_o = Mx4Matrix.quantised(torch.randn(H, nh * 256, generator=g, device="cuda") / (nh * 256) ** 0.5)
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    res = torch.randn(T, H, generator=g, device="cuda")
    qw, kw = (1 + 0.1 * torch.randn(256, generator=g, device="cuda") for _ in range(2))
    plan = AttnPlan(cu)
    pos3 = torch.from_numpy(np.repeat(np.concatenate([np.arange(n) for n in lens])[:, None], 3, 1).astype(np.int32)).cuda()
    _say("a layer", four_bit)
    X = Mx4Matrix.quantised(x) if four_bit else x
    qkv = att.project(X, w_qkv, plan, prologue=False)
    xv, wv = (_np(X.values(out_dtype="f32")) if four_bit else _np(x)), _np(w_qkv.values(out_dtype="f32"))
    want = xv @ wv.T
    assert (np.abs(_np(qkv) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -17 * (np.abs(xv) @ np.abs(wv).T)).all()
    # the prologue behind the product, and the whole pass: the same
    planes = att.planes(plan.kvT)
    att.project(X, w_qkv, plan, qw, kw, pos3, k_plane=planes[0], vt_plane=planes[1])
    own = att.forward(qkv, qw, kw, pos3, plan)
    assert torch.equal(att.forward(qkv, qw, kw, pos3, plan, k_plane=planes[0], vt_plane=planes[1], stage="core"), own)
    rows = qkv.clone()
    q, k = Rotary.heads(rows, nh, nkv, 256)
    Rotary(64, theta=1e7, axes=3).apply(q, k, pos3, qw, kw, q_out=q, k_out=k)
    out = plain.forward(rows, None, None, pos3, plan)
    d = (out.float() - own.float()).abs()
    assert d.max() <= 2e-2 and d.mean() <= 2e-3     # the path's own tolerance: q and k are rounded to bf16 once more
    a = Mx4Matrix.quantised(out)
    code, scale = mx4_ref.quantise(_np(out))
    av, ov = mx4_ref.values(code, scale), _np(w_o.values(out_dtype="f32"))
    y = res.clone()
    mx4_gemm(a, w_o, Y=y, residual=y)
    want = av @ ov.T + _np(res)
    off = 32 * 2.0 ** -23 * (np.abs(av) @ np.abs(ov).T)
    assert (np.abs(_np(y) - want) <= off + 2.0 ** -23 * np.abs(want)).all()
