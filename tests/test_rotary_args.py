"""Refusals of the rotary operator's outputs in bf16, without a GPU."""
import ctypes

import pytest
import torch

from cleffa_amd import Rotary, _lib
from tests.test_mx4 import _refused, _rotary_args

AWAY = ctypes.c_void_p(1 << 24)


@pytest.mark.parametrize("over,msg", [
    (dict(bf16_out=1), "bf16_out"), (dict(bf16_out=1, type=1), "bf16_out"), (dict(bf16_out=2, type=2), "bf16_out"), (dict(bf16_out=-1, type=2), "bf16_out"),
    (dict(bf16_out=1, type=2), "in place"), (dict(bf16_out=1, type=2, out=ctypes.c_void_p((1 << 24) + 1)), "aligned"),
    (dict(bf16_out=1, type=2, x=ctypes.c_void_p((1 << 20) + 2), out=AWAY), "aligned"),
])
def test_bf16_out_refusals(over, msg):
    a = _rotary_args(**over)
    setattr(a, "k.out", AWAY)
    _refused(_lib.load().clef_hip_rotary, a, msg)


def test_bf16_outputs_need_only_their_own_alignment():
    a = _rotary_args(bf16_out=1, type=2, out=ctypes.c_void_p((1 << 24) + 2), pos=None)
    setattr(a, "k.out", ctypes.c_void_p((1 << 26) + 2))
    _refused(_lib.load().clef_hip_rotary, a, "pos")     # the check behind the heads'


def test_output_types():
    r, pos = Rotary(32, device="cpu"), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64)
    half, other = q.bfloat16(), q.half()
    for args, kw in (((q, None, pos), dict(q_out=other)), ((half, None, pos), dict(q_out=q)), ((half, None, pos), dict(q_out=other)),
                     ((q, q, pos), dict(q_out=half.clone(), k_out=q)), ((q, q, pos), dict(q_out=q, k_out=half)), ((q, half, pos), dict(q_out=half, k_out=half))):
        with pytest.raises(TypeError, match="dtype"):
            r.apply(*args, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        r.apply(q, q, pos, q_out=half, k_out=half.clone())


@pytest.mark.parametrize("n,theta,factor", [(4, 1e7, 1e151), (64, 1e300, 1e9), (4, 1e300, 1e9)])
def test_a_base_beyond_f64_is_refused(n, theta, factor):
    """It would make every frequency but the first zero."""
    with pytest.raises(RuntimeError, match="too large"):
        Rotary(n, theta=theta, scaling={"kind": "base", "factor": factor}, device="cpu")
    assert (Rotary(n, theta=1e7, scaling={"kind": "base", "factor": 1e100}, device="cpu").freq > 0).all()
