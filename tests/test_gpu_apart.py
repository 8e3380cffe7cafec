"""Outputs beside what is read, in the same rows: nothing of it overlaps, so the calls are taken and right."""
import pytest
import torch

from cleffa_amd import Mx4Matrix, Rotary, mx4_gemm

pytestmark = pytest.mark.gpu


def _randn(*shape, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


@pytest.mark.parametrize("T", [1, 5, 300])
def test_product_beside_its_rows(T):
    K, N = 96, 104
    print("[apart] product", T, flush=True)
    W = Mx4Matrix.quantised(_randn(N, K))
    wide = _randn(T, K + N + 16, seed=2).bfloat16()
    kept, X, Y = wide.clone(), wide[:, :K], wide[:, K + 8:K + 8 + N]
    want = mx4_gemm(X.contiguous(), W)
    mx4_gemm(X, W, Y=Y)
    assert torch.equal(Y, want)
    Y.copy_(kept[:, K + 8:K + 8 + N])
    assert torch.equal(wide, kept)
    # Y ahead of X, in every second row's place
    two = torch.zeros(2 * T, 104, dtype=torch.bfloat16, device="cuda")
    two[1::2, :K] = X
    assert torch.equal(mx4_gemm(two[1::2, :K], W, Y=two[0::2, :N]), want)
    assert torch.equal(two[1::2, :K], X)
    # the residual behind Y's columns
    f = _randn(T, 2 * N + 4, seed=3)
    r = f[:, N + 4:]
    want = mx4_gemm(X, W, residual=r.contiguous())
    mx4_gemm(X, W, Y=f[:, :N], residual=r)
    assert torch.equal(f[:, :N], want)


@pytest.mark.parametrize("T", [1, 6])
def test_rotary_beside_its_heads(T):
    nh, nkv, hd = 4, 2, 64
    r, pos = Rotary(hd), torch.arange(T, dtype=torch.int32, device="cuda")
    rows = _randn(T, (2 * nh + 2 * nkv) * hd).bfloat16()
    kept = rows.clone()
    q, k = Rotary.heads(rows, nh, nkv, hd)
    want = r.apply(q, k, pos)
    print("[apart] rotary", T, flush=True)
    # q into the gates' places, k into the values'
    gates, values = rows[:, :2 * nh * hd].unflatten(1, (nh, 2 * hd))[:, :, hd:], rows[:, (2 * nh + nkv) * hd:].unflatten(1, (nkv, hd))
    r.apply(q, k, pos, q_out=gates, k_out=values)
    assert torch.equal(gates, want[0]) and torch.equal(values, want[1])
    assert torch.equal(q, Rotary.heads(kept, nh, nkv, hd)[0]) and torch.equal(k, Rotary.heads(kept, nh, nkv, hd)[1])
    # heads of [q | k | v] each, in place
    trio = _randn(T, 3 * nh * hd, seed=4)
    tq, tk = (trio.unflatten(1, (nh, 3, hd))[:, :, i] for i in range(2))
    want = r.apply(tq.contiguous(), tk.contiguous(), pos)
    r.apply(tq, tk, pos, q_out=tq, k_out=tk)
    assert torch.equal(tq, want[0]) and torch.equal(tk, want[1])
    # heads ahead of rows, both outputs in one buffer
    both = torch.zeros(nh + nkv, T, hd, dtype=torch.bfloat16, device="cuda")
    want = r.apply(q, k, pos)
    r.apply(q, k, pos, q_out=both[:nh].transpose(0, 1), k_out=both[nh:].transpose(0, 1))
    assert torch.equal(both[:nh].transpose(0, 1), want[0]) and torch.equal(both[nh:].transpose(0, 1), want[1])


def test_overlaps_are_refused():
    W = Mx4Matrix.quantised(_randn(64, 64))
    x = _randn(8, 72).bfloat16()
    with pytest.raises(RuntimeError, match="Y overlaps X"):
        mx4_gemm(x[:, :64], W, Y=x[:, 8:72])
    q = _randn(8, 3, 64).bfloat16()
    pos = torch.arange(8, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        Rotary(64).apply(q, q, pos, q_out=q, k_out=q)
    with pytest.raises(RuntimeError, match="overlaps"):
        Rotary(64).apply(q[:4], None, pos[:4], q_out=q[2:6])
