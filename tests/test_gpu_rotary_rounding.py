"""Rotary outputs in bf16 from f32 heads: rounded once, where rows in bf16 were rounded before."""
import numpy as np
import pytest
import torch

from cleffa_amd import Mx4Matrix, Rotary, mx4_gemm
from tests.test_gpu_rotary import EPS, _check, _freq, _inputs, _np, _turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,n_rot", [(2, 2), (6, 4), (72, 36), (80, 40), (128, 128), (256, 64), (256, 250), (250, 250), (66, 64)])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_bf16_from_f32(layout, hd, n_rot, norm):
    print("[rotary] bf16 from f32", layout, hd, n_rot, norm, flush=True)
    f, r = _freq(n_rot), Rotary(n_rot, layout=layout)
    for T, nh, nkv in ((5, 7, 3), (513, 3, 1)):
        q, k, qw, kw = _inputs(T, nh, nkv, hd, torch.float32, hd + n_rot, norm)
        pos = torch.randint(0, 20000, (T,), dtype=torch.int32, device="cuda")
        q_out, k_out = torch.empty_like(q, dtype=torch.bfloat16), torch.empty_like(k, dtype=torch.bfloat16)
        assert r.apply(q, k, pos, qw, kw, q_out=q_out, k_out=k_out)[0] is q_out
        for x, out, w in ((q, q_out, qw), (k, k_out, kw)):
            _check(out, *_turned(_np(x), pos.cpu().numpy(), f, layout, norm=None if w is None else _np(w)), f, pos.cpu().numpy())
        # an output that is made takes the given one's type
        made = r.apply(q, k, pos, qw, kw, k_out=k_out)[0]
        assert made.dtype == torch.bfloat16 and torch.equal(made, q_out)
        # into heads of wider rows, at an odd element: nothing else is written
        wide = torch.full((T, nh * (hd + 3) + 5), 7.0, dtype=torch.bfloat16, device="cuda")
        view = wide[:, 3:3 + nh * (hd + 3)].unflatten(1, (nh, hd + 3))[:, :, :hd]
        r.apply(q, None, pos, qw, q_out=view)
        _check(view, *_turned(_np(q), pos.cpu().numpy(), f, layout, norm=None if qw is None else _np(qw)), f, pos.cpu().numpy())
        view.fill_(7)
        assert (wide == 7).all()


def test_projected_heads_are_rounded_once():
    """Quantised activations, the product in f32, norm and rotary: each output within one rounding to bf16 of the value in 64 bits. (From rows
    in bf16 it would be two: some of these outputs are off by more.)"""
    T, H, nh, nkv, hd, n = 40, 544, 4, 2, 256, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    W = Mx4Matrix.quantised(torch.randn((2 * nh + 2 * nkv) * hd, H, generator=g, device="cuda") / H ** 0.5)
    X = Mx4Matrix.quantised(torch.randn(T, H, generator=g, device="cuda"))
    w = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
    pos = torch.arange(1000, 1000 + T, dtype=torch.int32, device="cuda")
    print("[rotary] rounded once", flush=True)
    r, x, wv = Rotary(n), _np(X.values()), _np(W.values(out_dtype="f32"))
    q, k = Rotary.heads(mx4_gemm(X, W, out="f32"), nh, nkv, hd)
    out = r.apply(q, k, pos, w, w, q_out=torch.empty(T, nh, hd, dtype=torch.bfloat16, device="cuda"))
    exact = Rotary.heads(torch.from_numpy(x @ wv.T), nh, nkv, hd)
    # f32 sums of five steps and up to 16 joined waves; the norm passes a head's errors on at most twice, times weight / rms
    off = Rotary.heads(torch.from_numpy(21 * 2.0 ** -23 * (np.abs(x) @ np.abs(wv).T)), nh, nkv, hd)
    twice = r.apply(*(t.bfloat16() for t in (q, k)), pos, w, w)
    for got, t, e, double in zip(out, exact, off, twice):
        want, size = _turned(t.numpy(), pos.cpu().numpy(), _freq(n), "half", norm=_np(w))
        rms = np.sqrt((t.numpy() ** 2).mean(-1, keepdims=True) + EPS)
        lim = 2 * np.abs(_np(w)).max() / rms * np.linalg.norm(e.numpy(), axis=-1, keepdims=True) + size * (2.0 ** -21 + 10 * 2.0 ** -24)
        lim = lim + (np.abs(want) + lim) * 2.0 ** -8
        assert got.dtype == torch.bfloat16 and (np.abs(_np(got) - want) <= lim).all()
        assert (np.abs(_np(double) - want) > lim).any()
