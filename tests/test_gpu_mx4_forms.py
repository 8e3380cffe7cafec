"""Every form of the 4-bit product (mx4_forms.py) on what the forms differ in: rows that lie apart, ragged columns, NaN blocks, scales far
apart, graphs, streams. Against the sums in float64 of the values that codes stand for, within the bound of test_gpu_mx4.py."""
import pytest
import torch

from cleffa_amd import Mx4Matrix, mx4_gemm
from tests import mx4_forms

pytestmark = pytest.mark.gpu

FORMS = [("x4", f, *s) for f, s in mx4_forms.X4.items()] + [("xbf16", f, *s) for f, s in mx4_forms.X16.items()]
every_form = pytest.mark.parametrize("kind,form,T,N", FORMS, ids=[f"{k} {f}" for k, f, _, _ in FORMS])


def _k(form):
    """Columns for a form: 21 K tiles, two or three for each of eight waves, or ten in three scale groups; the last one of 32 columns alone."""
    return 2592 if form.startswith("rows") else 1184


def _say(*a):
    print("[mx4 forms]", *a, flush=True)


def _codes(rows, K, seed, lo=121, hi=130):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randint(0, 256, (rows, K // 2), generator=g, device="cuda", dtype=torch.uint8),
            torch.randint(lo, hi, (rows, K // 32), generator=g, device="cuda", dtype=torch.uint8))


def _values(codes, scales):
    """float64 of flat codes and scale bytes, from the format's definition."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    v = torch.cat([grid, -grid])[torch.stack([codes & 15, codes >> 4], -1).flatten(1).int()]
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127))
    return v * s.repeat_interleave(32, 1)


def _rows(T, K, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(T, K, generator=g, device="cuda").bfloat16()


def _operands(kind, T, N, K, seed):
    """X, W as mx4_gemm takes them and their values in float64."""
    wc = _codes(N, K, seed)
    if kind == "xbf16":
        x = _rows(T, K, seed + 1)
        return x, Mx4Matrix.from_codes(*wc), x.double(), _values(*wc)
    xc = _codes(T, K, seed + 1)
    return Mx4Matrix.from_codes(*xc), Mx4Matrix.from_codes(*wc), _values(*xc), _values(*wc)


def _want(kind, x, w):
    """The sums, and how far f32 sums may be off: a rounding of the magnitudes' sum for each step of 128 or 32 and each of 16 joined parts."""
    return x @ w.T, (-(-x.shape[1] // (32 if kind == "xbf16" else 128)) + 16) * 2.0 ** -23 * (x.abs() @ w.abs().T)


def _check(y, want, off, residual=None):
    if residual is not None:      # its addition rounds once more
        want = want + residual.double()
        off = off + 2.0 ** -24 * (want.abs() + off)
    lim = off + (want.abs() + off) * (2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -24)
    assert bool(((y.double() - want).abs() <= lim).all())


@every_form
def test_values_and_strides(kind, form, T, N):
    """Outputs in both types, with a residual and in its place; rows of X, Y and the residual that lie apart, Y at odd elements, and at whole lines (where
    stores go past the caches): what lies between stays as it was."""
    K = _k(form)
    _say("strides", kind, form, T, N, K)
    X, W, x, w = _operands(kind, T, N, K, T + N)
    want, off = _want(kind, x, w)
    if kind == "xbf16":
        wide = torch.full((T, K + 40), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, 16:16 + K] = X
        X = wide[:, 16:16 + K]
    _check(mx4_gemm(X, W), want, off)
    lines = -(-N // 64) * 64 + 64
    for dtype, row, lead in ((torch.bfloat16, N + 21, 1), (torch.bfloat16, lines, 0), (torch.float32, N + 21, 3), (torch.float32, lines, 0)):
        y = torch.full((T + 2, row), 3.0, dtype=dtype, device="cuda")
        mx4_gemm(X, W, Y=y[1:-1, lead:lead + N])
        _check(y[1:-1, lead:lead + N], want, off)
        y[1:-1, lead:lead + N] = 3
        assert (y == 3).all()
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    for row, lead in ((N + 5, 2), (lines, 0)):
        r = torch.randn(T, row, generator=g, device="cuda")
        kept, part = r.clone(), r[:, lead:lead + N]
        _check(mx4_gemm(X, W, residual=part), want, off, part)
        mx4_gemm(X, W, Y=part, residual=part)
        _check(part, want, off, kept[:, lead:lead + N])
        part.copy_(kept[:, lead:lead + N])
        assert torch.equal(r, kept)


@every_form
def test_bad_values(kind, form, T, N):
    """NaN blocks of W, first, last and in the middle, make their columns NaN, and of X their rows; nothing else."""
    K = _k(form)
    _say("bad values", kind, form)
    wc, ws = _codes(N, K, 7)
    ws[0, 0] = ws[N // 2, K // 64] = ws[N - 1, K // 32 - 1] = 255
    cols, rows = [0, N // 2, N - 1], [0, T // 2, T - 1]
    if kind == "xbf16":
        X = _rows(T, K, 8)
        x = X.double().clone()
        X[0, 0] = X[T // 2, K // 2] = X[T - 1, K - 1] = float("nan")
    else:
        xc, xs = _codes(T, K, 8)
        x = _values(xc, xs)
        xs[0, 0] = xs[T // 2, K // 64] = xs[T - 1, K // 32 - 1] = 255
        X = Mx4Matrix.from_codes(xc, xs)
    y = mx4_gemm(X, Mx4Matrix.from_codes(wc, ws), out="f32")
    bad = torch.zeros(T, N, dtype=torch.bool, device="cuda")
    bad[:, cols] = True
    bad[rows] = True
    assert torch.equal(y.isnan(), bad)
    clean = ws.clone()
    clean[clean == 255] = 127
    want, off = _want(kind, x, _values(wc, clean))
    lim = off + (want.abs() + off) * 2.0 ** -24
    assert bool(((y.double() - want).abs() <= lim)[~bad].all())


@every_form
def test_scales_far_apart(kind, form, T, N):
    """Blocks between 2^-100 and 2^20 of W against activations that bring them back: no block's scale is lost or taken twice."""
    K = _k(form)
    _say("scales", kind, form)
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    e = torch.randint(-100, 21, (K // 32,), generator=g, device="cuda")
    (wc, _), (xc, _) = _codes(N, K, 10), _codes(T, K, 11)
    ws, xs = ((127 + s * e).to(torch.uint8).expand(n, -1).contiguous() for s, n in ((1, N), (-1, T)))
    x, w = _values(xc, xs), _values(wc, ws)
    if kind == "xbf16":
        X = x.bfloat16()
        assert torch.equal(X.double(), x)
    else:
        X = Mx4Matrix.from_codes(xc, xs)
    _check(mx4_gemm(X, Mx4Matrix.from_codes(wc, ws), out="f32"), *_want(kind, x, w))


@every_form
def test_graphs_and_streams(kind, form, T, N):
    """The same bits again, from a graph replayed with other work between, and on two streams at once."""
    K = _k(form)
    _say("graphs", kind, form)
    X, W, _, _ = _operands(kind, T, N, K, 13)
    first = mx4_gemm(X, W)
    assert torch.equal(mx4_gemm(X, W), first)
    y = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mx4_gemm(X, W, Y=y)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.mm(torch.ones(64, 64, device="cuda"), torch.ones(64, 64, device="cuda"))
        torch.cuda.synchronize()
        assert torch.equal(y, first)
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[torch.zeros_like(first) for _ in range(3)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(3):
        for s, out in zip(streams, outs):
            mx4_gemm(X, W, Y=out[i], stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for out in outs for o in out)


@pytest.mark.parametrize("T,N", mx4_forms.FEW)
@pytest.mark.parametrize("kind", ["x4", "xbf16"])
def test_few_rows(kind, T, N):
    for K in (32, 160, 1184, 5120):
        _say("few rows", kind, T, N, K)
        X, W, x, w = _operands(kind, T, N, K, T + N + K)
        want, off = _want(kind, x, w)
        _check(mx4_gemm(X, W, out="f32"), want, off)
        _check(mx4_gemm(X, W), want, off)
        r = torch.ones(T, N, device="cuda")
        _check(mx4_gemm(X, W, residual=r), want, off, r)


def test_scale_bytes_beyond_the_types():
    """Scale bytes 253 and 254, from elsewhere: with X in bf16 a weight that bf16 does not hold is an infinity, all others are exact; in 4 bits nothing is
    lost that the sums hold."""
    K = 32
    codes = torch.arange(16, dtype=torch.uint8, device="cuda")
    wc = (codes | codes << 4)[:, None].expand(16, K // 2).contiguous()
    for s in (252, 253, 254):
        ws = torch.full((16, 1), s, dtype=torch.uint8, device="cuda")
        W, w = Mx4Matrix.from_codes(wc, ws), _values(wc, ws)[:, 0]
        x = torch.zeros(1, K, device="cuda")
        x[0, 3] = 2.0 ** -8
        limit = torch.finfo(torch.bfloat16).max
        held = torch.where(w.abs() <= limit, w, torch.sign(w) * float("inf"))
        got = mx4_gemm(x.bfloat16(), W, out="f32")[0].double()
        over = held.isinf()
        assert (s > 252) == bool(over.any())
        # an infinite weight times the row's zeros is NaN
        assert not bool(got[over].isfinite().any()) and torch.equal(got[~over], w[~over] * 2.0 ** -8)
        X = Mx4Matrix.quantised(x)
        assert torch.equal(mx4_gemm(X, W, out="f32")[0].double(), w * 2.0 ** -8)
