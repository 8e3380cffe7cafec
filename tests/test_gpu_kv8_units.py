"""The 8-bit paged cache's attention over pages of different scales, with bounds that are small next to the outputs:
a unit or a rescaling that is wrong by a factor of two shows."""
import numpy as np
import pytest
import torch

from cleffa_amd import Kv8Cache, Kv8Plan, TextAttention
from tests import kv8_ref as ref
from tests.test_gpu_kv8 import HALF_STEP, HD, PAGE, _cache_values, _int, _np, _qkv, _say, _sequence

pytestmark = pytest.mark.gpu
V_FAR = [2.0 ** 13, 2.0 ** -60, 1.0, 2.0 ** -20, 2.0 ** 12, 2.0 ** -62, 2.0 ** -3]
V_NEAR = [1.0, 4.0, 0.25, 8.0, 0.125, 2.0, 2.0 ** 5, 2.0 ** -4]
K_FAR = [2.0 ** 6, 2.0 ** -30, 1.0, 2.0 ** -55, 2.0 ** 5, 2.0 ** -3, 2.0 ** 7]
FORMS = {"token": 1, "question": 20, "prompt": 70}


def attend(q, k, v, first, scale):
    """Outputs [n][nh][256] of causal attention in float64 and how far each may be off before its own rounding. A query's element is
    off by half a step, 2^-11 of itself (2^-25 where it is subnormal) and 2^-18 of f32 arithmetic, so key i's score by
    d_i = scale sum |q k_i| (2^-11 + 2^-18) + scale sum |k_i| 2^-25 and its weight by the factor exp(+-d_i); the sum of the weights lies
    between sum w exp(-d) and sum w exp(d), whose logarithms are at most D = log sum w exp(d) (their product is at least 1). A weight's
    own rounding is 2^-11, or 2^-28 of the row's largest where that is more."""
    n, nh = q.shape[:2]
    out, off = np.zeros_like(q), np.zeros_like(q)
    for h in range(nh):
        kk, vv = k[h * k.shape[0] // nh], v[h * k.shape[0] // nh]
        for i in range(n):
            m = first + i + 1
            s = kk[:m] @ q[i, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            d = scale * (np.abs(kk[:m]) @ np.abs(q[i, h]) * (2.0 ** -11 + 2.0 ** -18) + np.abs(kk[:m]).sum(-1) * 2.0 ** -25)
            move = np.expm1(d + np.log((w * np.exp(d)).sum()))
            a = np.abs(vv[:m])
            out[i, h] = w @ vv[:m]
            off[i, h] = (w * (move + (1 + move) * 2.0 ** -11 + 2.0 ** -16)) @ a + 2.0 ** -28 * w.max() * a.sum(0)
    return out, off


def _rows(T, nh, nkv, seed, q_scale, k_scale, v_scale):
    """Queries and keys about 0, values about 1, times their scales (a number, or one a row)."""
    x = _qkv(T, nh, nkv, seed)[0].float()
    x[:, :2 * nh * HD] *= q_scale
    at = (2 * nh + nkv) * HD
    x[:, 2 * nh * HD:at] *= torch.as_tensor(k_scale, dtype=torch.float32, device="cuda").reshape(-1, 1)
    x[:, at:] = (1 + 0.5 * x[:, at:]) * torch.as_tensor(v_scale, dtype=torch.float32, device="cuda").reshape(-1, 1)
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("form,whole", [(f, w) for f in FORMS for w in (False, True) if f != "token" or not w])
@pytest.mark.parametrize("which,mags", [("v", V_FAR), ("v", V_FAR[::-1]), ("v", V_NEAR), ("v", V_NEAR[::-1]), ("k", K_FAR), ("k", K_FAR[::-1])])
def test_pages_of_different_magnitude(form, which, mags, whole):
    """Pages whose values, or keys, differ by powers of two, cached page by page or in one prompt whose own rows see
    them; outputs in f32, so that only the path's own roundings count."""
    nh, nkv, new = 4, 2, FORMS[form]
    q_scale = 2.0 ** -2 if which == "v" else 2.0 ** -8
    _say("magnitudes of", which, mags[0], form, whole)
    cache, model = Kv8Cache(1, nkv, 12, 1, 12), ref.Cache(12, 1, 12)
    cache.k[0].fill_(0x7f)
    cache.v[0].fill_(0xff)
    att = TextAttention(nh, nkv, HD, 0)
    n = PAGE * len(mags)
    size = np.concatenate([np.repeat(mags, PAGE), np.ones(new)])
    ones = np.ones(n + new)
    x = _rows(n + new, nh, nkv, 5, q_scale, size if which == "k" else ones, size if which == "v" else ones)
    # blocks of 128 rows are of passes of more than 8,192 (row, head) pairs
    spare = 2049 if form == "prompt" else 0
    passes = [n + new] if whole else [n, new]
    at = 0
    for m in passes:
        first = int(model.len[0])
        T = m + (spare if at + m == n + new else 0)
        plan = Kv8Plan(cache, T, nh, 1 if form == "token" and m == 1 else 32 if form == "question" and whole else None)
        plan.update(_int([m]))
        model.plan([m], T)
        qkv = torch.zeros(T, att.row, dtype=torch.bfloat16, device="cuda")
        qkv[:m] = x[at:at + m]
        out = att.forward_kv8(qkv, None, None, None, plan, cache, 0, out_dtype="f32", gate=False)
        at += m
    torch.cuda.synchronize()
    plan.check()
    kk, vv = _sequence(cache, _cache_values(cache), model, 0, n + new)
    q = _np(qkv.float())[:m, :2 * nh * HD].reshape(m, nh, 2, HD)[:, :, 0]
    want, off = attend(q, kk, vv, first, HD ** -0.5)
    off = off + HALF_STEP["f32"] * (np.abs(want) + off)
    tight = np.median(off, -1) / np.median(np.abs(want), -1)
    assert tight.max() < 0.03, "the bound says too little"
    d = np.abs(_np(out)[:m].reshape(want.shape) - want)
    with np.errstate(invalid="ignore"):   # a first token's value of 0
        _say(f"largest error {np.nanmax(d / off):.3f} of its bound, which is {tight.max():.4f} of the outputs")
    assert (d <= off).all()
