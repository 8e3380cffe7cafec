"""Where calls make their results, planes and tables: in the memory of the stream that they are given, not of the current one, whose
own work may still use it, or take it again before the call has run."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

from cleffa_amd import AttnPlan, Kv8Cache, Kv8Plan, Mx4Matrix, Rotary, TextAttention, VisionAttention, mx4, mx4_gemm, rotary, vision_positions
from cleffa_amd import workloads
from cleffa_amd.gemm import gemm
from cleffa_amd.omni import OmniAttention, OmniPlan
from cleffa_amd.prefix_cache import PrefixEntry

MAKERS = ("empty", "empty_like", "zeros")


@contextlib.contextmanager
def _made(monkeypatch, where):
    """A list of where() at each tensor that is made."""
    made = []
    with monkeypatch.context() as m:
        for name in MAKERS:
            real = getattr(torch, name)
            m.setattr(torch, name, lambda *a, _real=real, **k: (made.append(where()), _real(*a, **k))[1])
        yield made


def test_made_on_the_given_stream(monkeypatch):
    """Without a GPU: a stream whose context is watched, launches that do nothing."""
    current = []

    @contextlib.contextmanager
    def context(s):
        current.append(s)
        yield
        current.pop()
    monkeypatch.setattr(torch.cuda, "stream", context)
    launched = []
    for module in (mx4, rotary):
        monkeypatch.setattr(module, "_launch", lambda fn, a, dev, stream: launched.append(stream))
    s, where = object(), lambda: current[-1] if current else None
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    m, q, pos = Mx4Matrix(4, 64, device="cpu"), torch.zeros(4, 2, 64), torch.zeros(4, dtype=torch.int32)
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    att = SimpleNamespace(device=torch.device("cpu"), row=4, nh=1, nkv=1, hd=256, n_rot=0)
    calls = [lambda **k: Mx4Matrix.quantised(x, **k), lambda **k: Mx4Matrix.from_codes(codes, scales, **k), lambda **k: m.to_codes(**k), lambda **k: m.values(**k),
             lambda **k: mx4_gemm(x, m, **k), lambda **k: Rotary(32, device="cpu").apply(q, q, pos, **k),
             lambda **k: TextAttention.project(att, x, m, SimpleNamespace(T=4), prologue=False, **k)]
    for call in calls:
        for stream in (s, None):
            with _made(monkeypatch, where) as made:
                call(stream=stream)
            assert made and all(w is stream for w in made)
            assert launched.pop() is stream


@pytest.mark.gpu
def test_calls_on_another_stream(monkeypatch):
    """All calls that make something, on a stream beside the current one: made there, and the current stream's result."""
    s = torch.cuda.Stream()
    T, H, nh, nkv, E = 40, 256, 4, 2, 16 * 72
    w = workloads.text_inputs([T], nh, nkv, seed=1)
    d = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in w.items()}
    att, plan = TextAttention(nh, nkv), AttnPlan([0, T])
    vis, vplan, pos2 = VisionAttention(), AttnPlan([0, 16], causal=False), torch.from_numpy(vision_positions([0, 16], [4])).cuda()
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    x, W, vqkv = (torch.randn(*n, generator=g, device="cuda").bfloat16() for n in ((T, H), (att.row, H), (16, 3 * E)))
    omni, oplan, oqkv = OmniAttention(8, 1), OmniPlan([0, T]), torch.randn(T, 10 * 128, generator=g, device="cuda")
    ones, pos = torch.ones(128, device="cuda"), torch.arange(T, dtype=torch.int32, device="cuda")
    X4, W4 = Mx4Matrix.quantised(x), Mx4Matrix.quantised(W)
    q, r = torch.randn(T, nh, 256, generator=g, device="cuda").bfloat16(), Rotary(64)
    codes = X4.to_codes()
    prep = dict(q_norm=d["q_norm"], k_norm=d["k_norm"], pos3=d["pos3"])

    def eight_bit(**k):
        cache = Kv8Cache(1, nkv, 4, 1, 2)
        p = Kv8Plan(cache, T, nh, T).update(torch.full((1,), T, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        with _made(monkeypatch, torch.cuda.current_stream) as made:
            out = att.forward_kv8(d["qkv"], d["q_norm"], d["k_norm"], d["pos3"], p, cache, **k)
        return out, made

    def grown(**k):
        entry = PrefixEntry(2, nkv)
        entry.reserve(100, 0)
        for t in (*entry.K, *entry.Vt):
            t.fill_(3)
        torch.cuda.synchronize()
        with _made(monkeypatch, torch.cuda.current_stream) as made:
            entry.reserve(2000, 96, **k)
        return (*(t[:, :96] for t in entry.K), *(t[:, :, :96] for t in entry.Vt)), made

    plain = {
        "forward": lambda **k: att.forward(d["qkv"], d["q_norm"], d["k_norm"], d["pos3"], plan, **k), "gemm": lambda **k: gemm(x, W, **k),
        "project": lambda **k: att.project(x, W, plan, **prep, **k), "project 4 bits": lambda **k: att.project(X4, W4, plan, **prep, **k),
        "vision": lambda **k: vis.forward(vqkv, None, pos2, vplan, **k), "omni": lambda **k: omni.forward(oqkv, ones, ones, d["pos3"], oplan, **k),
        "quantised": lambda **k: Mx4Matrix.quantised(x, **k), "from codes": lambda **k: Mx4Matrix.from_codes(*codes, **k),
        "to codes": lambda **k: X4.to_codes(**k), "values": lambda **k: X4.values(**k), "product": lambda **k: mx4_gemm(x, W4, **k),
        "rotary": lambda **k: r.apply(q, q, pos, **k),
    }

    def watched(call):
        def run(**k):
            with _made(monkeypatch, torch.cuda.current_stream) as made:
                return call(**k), made
        return run
    for name, call in {**{n: watched(c) for n, c in plain.items()}, "8 bits": eight_bit, "prefix": grown}.items():
        print("[streams]", name, flush=True)
        want = call()[0]
        torch.cuda.synchronize()
        got, made = call(stream=s)
        s.synchronize()
        assert made and all(w == s for w in made), name
        got, want = (t.to_codes() if isinstance(t, Mx4Matrix) else (t,) if isinstance(t, torch.Tensor) else t for t in (got, want))
        for a, b in zip(got, want):
            assert torch.equal(a, b), name
