"""Three position axes that differ: the rotary operator and the attention's own prologue turn each pair by the same one."""
import numpy as np
import pytest
import torch

from cleffa_amd import AttnPlan, Rotary, TextAttention
from tests.test_gpu_rotary import _freq, _np, _turned

pytestmark = pytest.mark.gpu


def test_axes_as_in_the_prologue():
    nh, nkv, T = 4, 2, 150
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    att, plain, plan = TextAttention(nh, nkv, n_rot=64), TextAttention(nh, nkv, n_rot=0), AttnPlan([0, 70, T])
    qkv = torch.randn(T, att.row, generator=g, device="cuda").bfloat16()
    qw, kw = (1 + 0.1 * torch.randn(256, generator=g, device="cuda") for _ in range(2))
    pos3 = torch.randint(0, 3000, (T, 3), generator=g, device="cuda", dtype=torch.int32)
    print("[rotary] axes", flush=True)
    own = att.forward(qkv, qw, kw, pos3, plan)
    rows = qkv.clone()
    q, k = Rotary.heads(rows, nh, nkv, 256)
    Rotary(64, theta=1e7, axes=3).apply(q, k, pos3, qw, kw, q_out=q, k_out=k)
    f = _freq(64)
    want, size = _turned(_np(Rotary.heads(qkv, nh, nkv, 256)[1]), pos3.cpu().numpy(), f, "half", norm=_np(kw))
    assert (np.abs(_np(k) - want) <= size * 2.0 ** -20 + (np.abs(want) + size * 2.0 ** -20) * 2.0 ** -8).all()
    d = (plain.forward(rows, None, None, pos3, plan).float() - own.float()).abs()
    assert d.max() <= 2e-2 and d.mean() <= 2e-3      # the path's own tolerance: q and k are rounded to bf16 once more
    # axes in another order are not
    q, k = Rotary.heads(rows.copy_(qkv), nh, nkv, 256)
    Rotary(64, theta=1e7, axes=3).apply(q, k, pos3.flip(1).contiguous(), qw, kw, q_out=q, k_out=k)
    assert (plain.forward(rows, None, None, pos3, plan).float() - own.float()).abs().max() > 2e-2
