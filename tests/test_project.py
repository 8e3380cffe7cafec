"""TextAttention.project without a GPU: what a call does beside the product."""
import builtins
from types import SimpleNamespace

import pytest
import torch

from cleffa_amd import Mx4Matrix, TextAttention, mx4


@pytest.mark.parametrize("four_bit", [True, False])
def test_a_call_imports_nothing(four_bit, monkeypatch):
    """An import statement inside costs every call 0.9 us of host time, 16-bit weights too."""
    monkeypatch.setattr(mx4, "_launch", lambda fn, a, dev, stream: None)
    att = SimpleNamespace(device=torch.device("cpu"), row=4, nh=1, nkv=1, hd=256, n_rot=0)
    x = Mx4Matrix(8, 64, device="cpu")
    W = Mx4Matrix(4, 64, device="cpu") if four_bit else torch.zeros(4, 64, dtype=torch.bfloat16)
    names, real = [], builtins.__import__

    def watch(name, globals=None, *a):
        if globals and globals.get("__name__", "").startswith("cleffa_amd"):
            names.append(name)
        return real(name, globals, *a)
    monkeypatch.setattr(builtins, "__import__", watch)
    if four_bit:
        TextAttention.project(att, x, W, SimpleNamespace(T=8), prologue=False)
    else:
        with pytest.raises(TypeError, match="4 bits"):
            TextAttention.project(att, x, W, SimpleNamespace(T=8), prologue=False)
    assert names == []
