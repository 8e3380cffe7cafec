"""The 8-bit paged cache's attention at the ends of its range, in each of its three forms: scores of any size, tokens
that are not numbers."""
import numpy as np
import pytest
import torch

from cleffa_amd import Kv8Cache, Kv8Plan, TextAttention
from tests import kv8_ref as ref
from tests.test_gpu_kv8 import HALF_STEP, HD, PAGE, _cache_values, _int, _np, _qkv, _say, _sequence

pytestmark = pytest.mark.gpu
# new tokens, pass rows, max_new: blocks of 16, 32 and 128 rows for two q heads a kv head
FORMS = {"token": (1, 1, 1), "question": (20, 20, None), "prompt": (40, 4097, None)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [300.0, 6000.0, 8000.0, 10000.0, 60000.0])
def test_scores_of_any_size(form, size):
    """Queries and keys of equal elements, up to the largest that f16 holds: scores of 2^16 to 2^36, in pages of
    different scales. A row's largest keys share its weight, all others are further off than f32 or f64 can tell from 0;
    their weights are equal, so an output is off by the half steps of f16 weights (2^-11) and of its own."""
    nh, nkv, n = 2, 1, 200
    new, T, max_new = FORMS[form]
    _say("scores", form, size)
    cache, model = Kv8Cache(1, nkv, 8, 1, 8), ref.Cache(8, 1, 8)
    att = TextAttention(nh, nkv, HD, 0)
    base = 2.0 ** np.floor(np.log2(size))
    for m, rows, hint in ((n, n, None), (new, T, max_new)):
        plan = Kv8Plan(cache, rows, nh, hint)
        plan.update(_int([m]))
        before = int(model.len[0])
        model.plan([m], rows)
        qkv, _, _ = _qkv(rows, nh, nkv, m)
        qkv[:, :HD], qkv[:, 2 * HD:3 * HD] = size, -size       # one head looks for the largest key, the other for the least
        t = before + np.arange(rows)
        key = base * (0.5 + t % 5 / 8) * np.array([0.25, 1, -0.5, 0.125, 1])[t // PAGE % 5]
        qkv[:, 2 * nh * HD:2 * nh * HD + HD] = torch.tensor(key, dtype=torch.bfloat16, device="cuda")[:, None]
        out = att.forward_kv8(qkv, None, None, None, plan, cache, 0, gate=False)
    torch.cuda.synchronize()
    kk, vv = _sequence(cache, _cache_values(cache), model, 0, n + new)
    got = _np(out.float())[:new].reshape(new, nh, HD)
    q = _np(qkv.float())[:new, :2 * nh * HD].reshape(new, nh, 2, HD)[:, :, 0]
    for i in range(new):
        s = q[i] @ kk[0, :n + i + 1].T * HD ** -0.5
        far = s.max(-1, keepdims=True) - s
        assert ((far == 0) | (far > 200)).all()
        w = (far == 0) / (far == 0).sum(-1, keepdims=True)
        want, room = w @ vv[0, :n + i + 1], w @ np.abs(vv[0, :n + i + 1])
        assert (np.abs(got[i] - want) <= room * (2.0 ** -11 + HALF_STEP["bf16"] + 2.0 ** -16)).all(), (i, np.abs(got[i] - want).max())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("what", ["row", "row of infinities", "same dim"])
def test_tokens_that_are_not_numbers(form, what):
    """A token whose query and key are NaN or infinite, with norms and without: finite outputs, a flag at its
    sequence's first row, and the other sequence's rows as they are without it."""
    nh, nkv = 2, 1
    new, T, max_new = FORMS[form]
    T += new
    outs = []
    for bad in (False, True):
        _say("not numbers", form, what, bad)
        cache = Kv8Cache(1, nkv, 12, 2, 6)
        norm = what != "same dim"
        att = TextAttention(nh, nkv, HD, 64 if norm else 0)
        first = Kv8Plan(cache, 140, nh)
        first.update(_int([70, 70]))
        qkv, qn, kn = _qkv(140, nh, nkv, 1)
        if not norm:
            qn = kn = None
        att.forward_kv8(qkv, qn, kn, first.pos3, first, cache, 0, stage="append")
        plan = Kv8Plan(cache, T, nh, max_new)
        plan.update(_int([new, new]))
        qkv, _, _ = _qkv(T, nh, nkv, 2)
        if bad:
            t = new + new // 2
            if what == "same dim":
                qkv[t, 7] = qkv[t, 2 * HD + 7] = qkv[t, 2 * nh * HD + 7] = float("inf")
            else:
                for at in (slice(0, HD), slice(2 * HD, 3 * HD), slice(2 * nh * HD, (2 * nh + 2 * nkv) * HD)):
                    qkv[t, at] = float("nan") if what == "row" else float("inf")
        ovf = torch.zeros(T, dtype=torch.int32, device="cuda")
        out = att.forward_kv8(qkv, qn, kn, plan.pos3, plan, cache, 0, ovf=ovf)[:2 * new]
        torch.cuda.synchronize()
        want = np.zeros(T, np.int32)
        want[new] = bad
        assert np.array_equal(_np(ovf), want)
        assert torch.isfinite(out.float()).all(), "rows " + str((~torch.isfinite(out.float())).any(1).nonzero().flatten().tolist())
        outs.append(out)
    assert torch.equal(outs[0][:new].view(torch.int16), outs[1][:new].view(torch.int16))
