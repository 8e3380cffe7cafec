"""The rotary of the 8-bit paged cache's keys: a code may differ from the definition's only where f32 arithmetic of the
path's own precision can tell the two apart."""
import numpy as np
import pytest
import torch

from cleffa_amd import Kv8Cache, Kv8Plan, TextAttention, rope_inv_freq
from tests import kv8_ref as ref
from tests.test_gpu_kv8 import HD, PAGE, _int, _np, _qkv, _say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("most,trig", [(1 << 10, 1.3), (1 << 21, 1.3), (1 << 22, 2.9), (1 << 26, 6.0), (1 << 31, 180.0)])
def test_codes_of_rotated_keys(most, trig):
    """Keys without norm at positions of three axes up to ``most``. x = a cos - b sin (and b cos + a sin): sine and cosine
    are off by trig * 2^-24 (1.3 up to angles of 2^21, 2.8 up to 2^22, the reduction of farther ones more), the inner product and
    the sum by half a step each. Codes are monotone in the value, so each lies between those of the ends."""
    nh, nkv, T = 4, 4, 4096
    _say("rotary up to", most)
    cache = Kv8Cache(1, nkv, T // PAGE, 1, T // PAGE)
    plan = Kv8Plan(cache, T, nh)
    plan.update(_int([T]))
    qkv, _, _ = _qkv(T, nh, nkv, 7)
    rng = np.random.default_rng(most)
    pos = rng.integers(0, most, (T, 3)).astype(np.int32)
    pos[::3] = (most * np.exp(-rng.uniform(0, 12, (len(pos[::3]), 3)))).astype(np.int64).clip(0, most - 1)
    TextAttention(nh, nkv).forward_kv8(qkv, None, None, _int(pos), plan, cache, 0, stage="append")
    torch.cuda.synchronize()
    pages = _np(cache.tables)[0]
    codes = ref.decode(cache.k[0].cpu().numpy())[pages]                    # [page][nkv][4][64][64]
    got = codes[:, :, 0].transpose(0, 2, 1, 3).reshape(T, nkv, 64)         # the 64 rotated dims
    s = np.repeat(_np(cache.k_scale[0])[pages], PAGE, 0)[..., None]
    k = _np(qkv.float())[:, 2 * nh * HD:(2 * nh + nkv) * HD].reshape(T, nkv, HD)
    a, b = k[..., :32], k[..., 32:64]
    ang = (pos[:, np.arange(32) % 3].astype(np.float32) * rope_inv_freq(1e7, 64)).astype(np.float64)[:, None]
    x = np.concatenate([a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)], -1)
    both = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    off = (both * (trig + 0.5) + np.abs(x) * 0.5) * 2.0 ** -24 * (1 + 2.0 ** -10)
    lo, hi = ref.round_e4m3((x - off) / s), ref.round_e4m3((x + off) / s)
    wrong = (got < lo) | (got > hi)
    _say(int((lo != hi).sum()), "codes may go either way,", int(wrong.sum()), "of", wrong.size, "are wrong")
    assert not wrong.any()


def _borders(x):
    """The distance of each x (|x| < 448) to the nearest border between two codes."""
    _, e = np.frexp(x)
    step = 2.0 ** (np.maximum(e - 1, -6) - 3)
    return (0.5 - np.abs(x / step - np.rint(x / step))) * step


def near_borders(T, heads, trig, least=1.0, most=1.5, most_pos=1 << 20, seed=0, tries=1 << 16):
    """Keys a, b [T][heads][32] (bf16 values), positions [T] and which of their rotated elements [T][heads][64] lie between
    ``least`` and ``most`` times the error away from a border that sine and cosine trig * 2^-24 off give them."""
    rng = np.random.default_rng(seed)
    pos = rng.integers(0, most_pos, T)
    ang = (pos.astype(np.float32)[:, None] * rope_inv_freq(1e7, 64)).astype(np.float64)
    a, b = np.full((T, heads, 32), 64.0), np.full((T, heads, 32), 64.0)
    for t in range(T):
        for i in range(32):
            p, q = (np.rint(rng.uniform(128, 256, tries)) * rng.choice([-1.0, 1.0], tries) for _ in range(2))   # eight bits: bf16 values
            c, s = np.cos(ang[t, i]), np.sin(ang[t, i])
            good = np.zeros(tries, bool)
            for x in (p * c - q * s, q * c + p * s):
                off = ((np.abs(p) + np.abs(q)) * (trig + 0.5) + np.abs(x) * 0.5) * 2.0 ** -24
                d = _borders(x)
                good |= (d > least * off) & (d <= most * off)
            at = np.flatnonzero(good)[:heads]
            a[t, :len(at), i], b[t, :len(at), i] = p[at], q[at]
    return a, b, pos, ang


def test_codes_near_a_border():
    """Keys that are chosen to rotate to just beside a border between two codes: sine and cosine within 4e-7 leave every
    code as the definition has it, an error of one and a half times that would not."""
    heads, T, trig = 4, 64, 4e-7 * 2.0 ** 24
    _say("keys near borders")
    a, b, pos, ang = near_borders(T, heads, trig)
    x = np.concatenate([a * np.cos(ang)[:, None] - b * np.sin(ang)[:, None], b * np.cos(ang)[:, None] + a * np.sin(ang)[:, None]], -1)
    off = ((np.abs(np.concatenate([a] * 2, -1)) + np.abs(np.concatenate([b] * 2, -1))) * (trig + 0.5) + np.abs(x) * 0.5) * 2.0 ** -24
    sure = _borders(x) > off
    close = sure & (_borders(x) <= 1.5 * off)
    assert close.sum() > 1000
    k = np.zeros((T, heads, HD))
    k[..., :32], k[..., 32:64], k[..., 200] = a, b, 448.0                   # the page's scale is 1
    cache = Kv8Cache(1, heads, 1, 1, 1)
    plan = Kv8Plan(cache, T, heads)
    plan.update(_int([T]))
    att = TextAttention(heads, heads)
    qkv = torch.zeros(T, att.row, dtype=torch.bfloat16, device="cuda")
    qkv[:, 2 * heads * HD:3 * heads * HD] = torch.tensor(k.reshape(T, -1), dtype=torch.bfloat16, device="cuda")
    assert np.array_equal(_np(qkv.float())[:, 2 * heads * HD:3 * heads * HD].reshape(k.shape), k)
    att.forward_kv8(qkv, None, None, _int(np.repeat(pos[:, None], 3, 1)), plan, cache, 0, stage="append")
    torch.cuda.synchronize()
    assert (_np(cache.k_scale[0]) == 1).all()
    got = ref.decode(cache.k[0].cpu().numpy())[0][:, 0].transpose(1, 0, 2)  # [T][heads][64]
    wrong = sure & (got != ref.round_e4m3(x))
    _say(int(close.sum()), "codes near a border,", int(wrong.sum()), "of", int(sure.sum()), "are wrong")
    assert not wrong.any()
