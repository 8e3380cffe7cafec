"""4-bit matrices on the GPU against the format's definition in float64: codes and scales bit for bit, values exactly,
products within the roundings of f32 sums."""
import numpy as np
import pytest
import torch

from cleffa_amd import Mx4Matrix, _lib, mx4_gemm
from tests import mx4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _say(*a):
    print("[mx4]", *a, flush=True)


def _rows(rows, K, seed, dtype=torch.bfloat16, spread=3):
    """Normal values times powers of two by block and by channel."""
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, K)) * np.exp2(r.integers(-spread, spread + 1, (rows, K // 32))).repeat(32, 1) * np.where(r.random(K) < 0.03, 8, 1)
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


def _np(x):
    return x.detach().cpu().double().numpy()


def _matrix(code, scale):
    """From reference codes; the buffers' unused bytes hold NaN scales and the largest codes."""
    rows, K = code.shape
    m = Mx4Matrix(rows, K)
    m.codes.fill_(0x77)
    m.scales.fill_(255)
    return m._pack(torch.from_numpy(ref.flat(code)).cuda(), torch.from_numpy(np.ascontiguousarray(scale)).cuda(), 0, None)


def _held(m):
    codes, scales = m.to_codes()
    return ref.unflat(codes.cpu().numpy()), scales.cpu().numpy()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 64), (16, 128), (17, 96), (33, 544), (5, 5120), (100, 1056)])
def test_quantise_and_values(rows, K, dtype):
    _say("quantise", rows, K, dtype)
    x = _rows(rows, K, rows + K, TYPES[dtype])
    code, scale = ref.quantise(_np(x))
    m = Mx4Matrix(rows, K)
    m.codes.fill_(0x77)
    m.scales.fill_(255)
    got_code, got_scale = _held(m.quantise(x.cuda()))
    assert np.array_equal(got_scale, scale)
    assert np.array_equal(got_code, code)
    want = ref.values(code, scale)
    for out in ("bf16", "f32"):
        assert np.array_equal(_np(m.values(out_dtype=out)), want)
    # values of values are the same
    assert np.array_equal(_held(Mx4Matrix.quantised(m.values(out_dtype="f32")))[0] & 7, code & 7) or (scale == 0).any()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantise_borders(dtype):
    """Ties, largest values next to the scale's borders, zeros of both signs, the smallest and largest magnitudes."""
    t = TYPES[dtype]
    info = torch.finfo(t)
    blocks = []
    for e in (0, -3, 4):
        for most in (4, 5, 6, 6.5, 7, 7.5, 3.5, 3.75, 1.0):
            tie = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 0.24, 0.26, 0.74, 0.76, 1.24, 1.26, 2.49, 2.51] * 2) * np.where(np.arange(32) < 16, 1, -1)
            tie = np.clip(tie, -most, most)
            tie[31] = most
            blocks.append(tie * 2.0 ** e)
    for v in (info.max, info.tiny, info.smallest_normal / 8, info.max * 0.874, 0.0):
        b = np.zeros(32)
        b[5], b[6], b[7] = v, -v / 2, v / 3
        blocks.append(b)
    blocks.append(np.full(32, -0.0))
    x = torch.from_numpy(np.array(blocks)).to(t)
    x = torch.cat([x, -x])
    code, scale = ref.quantise(_np(x))
    _say("borders", dtype, x.shape)
    m = Mx4Matrix.quantised(x.cuda())
    got_code, got_scale = _held(m)
    assert np.array_equal(got_scale, scale)
    assert np.array_equal(got_code, code)
    assert np.array_equal(_np(m.values(out_dtype="f32")), ref.values(code, scale))
    assert np.array_equal(_np(m.values()), ref.values(code, scale))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantise_not_finite(dtype, bad):
    x = _rows(20, 160, 3, TYPES[dtype])
    x[2, 33], x[2, 40], x[19, 159] = bad, float("nan"), bad
    code, scale = ref.quantise(_np(x))
    assert (scale == 255).sum() == 2
    m = Mx4Matrix.quantised(x.cuda())
    got_code, got_scale = _held(m)
    assert np.array_equal(got_scale, scale) and np.array_equal(got_code, code)
    for out in ("bf16", "f32"):
        assert np.array_equal(_np(m.values(out_dtype=out)), ref.values(code, scale), equal_nan=True)


def test_quantise_touches_its_rows_alone():
    """Strided rows in, strided rows out, the first rows of a larger matrix: nothing else is written."""
    _say("rows alone")
    wide = torch.full((40, 200), float("nan"), dtype=torch.bfloat16, device="cuda")
    x = _rows(40, 160, 9).cuda()
    wide[:, 8:168] = x
    m = Mx4Matrix.quantised(_rows(40, 160, 10).cuda())
    before = _held(m)
    m.first(16).quantise(wide[:16, 8:168])
    code, scale = ref.quantise(_np(x))
    got = _held(m)
    assert np.array_equal(got[0][:16], code[:16]) and np.array_equal(got[1][:16], scale[:16])
    assert np.array_equal(got[0][16:], before[0][16:]) and np.array_equal(got[1][16:], before[1][16:])
    # rows of the last row tile beyond the matrix stay as they were
    t = Mx4Matrix(3, 96)
    t.codes.fill_(0x5a)
    t.scales.fill_(0x5b)
    t.quantise(x[:3, :96])
    assert (t.codes.view(4, 16, 16)[:, 3:] == 0x5a).all() and (t.scales.view(4, 16, 4)[:, 3:] == 0x5b).all()
    assert (t.codes.view(4, 16, 16)[3, :3] == 0).all() and (t.scales.view(4, 16, 4)[3, :3] == 0).all()
    out = torch.full((40, 200), 7.0, dtype=torch.bfloat16, device="cuda")
    m.quantise(x).values(out=out[:, 8:168])
    assert np.array_equal(_np(out[:, 8:168]), ref.values(code, scale))
    assert (out[:, :8] == 7).all() and (out[:, 168:] == 7).all()


@pytest.mark.parametrize("rows,K", [(1, 32), (31, 96), (48, 1056)])
def test_codes_of_files(rows, K):
    r = np.random.default_rng(rows)
    code, scale = r.integers(0, 16, (rows, K), dtype=np.uint8), r.integers(0, 256, (rows, K // 32), dtype=np.uint8)
    got = _held(_matrix(code, scale))
    assert np.array_equal(got[0], code) and np.array_equal(got[1], scale)
    finite = np.minimum(scale, 252)
    assert np.array_equal(_np(_matrix(code, finite).values(out_dtype="f32")), ref.values(code, finite))
    # 2^-127 * 0.5 is the smallest value: bf16 holds it
    assert np.array_equal(_np(_matrix(code, finite).values()), ref.values(code, finite))


def _operands(T, N, K, seed, bf):
    """X and W as matrices (or a bf16 tensor) and their values in float64."""
    xs, ws = _rows(T, K, seed), _rows(N, K, seed + 1) / K ** 0.5
    wq = ref.quantise(_np(ws))
    if bf:
        return xs.cuda(), _matrix(*wq), _np(xs), ref.values(*wq)
    xq = ref.quantise(_np(xs))
    return _matrix(*xq), _matrix(*wq), ref.values(*xq), ref.values(*wq)


def _off(x, w, bf):
    """How far a sum of products in f32 may be off, each [t][n]. A step of the 4-bit instruction adds 128 exact products to a
    sum, one of the 16-bit instruction 32, up to 16 waves' sums are joined: a rounding each, of at most 2^-23 of what
    is in it, which is at most the sum of the products' magnitudes."""
    mag = np.abs(x) @ np.abs(w).T
    return (-(-x.shape[1] // (32 if bf else 128)) + 16) * 2.0 ** -23 * mag


def _check(y, want, off):
    y = y.detach()
    d = np.abs(_np(y) - want)
    # the store's rounding: half a step of the result's type, of the value that is rounded
    lim = off + (np.abs(want) + off) * (2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -24)
    assert (d <= lim).all(), f"{d.max()} off, {(d / np.maximum(lim, 1e-300)).max()} of what is allowed"


SHAPES = [(1, 1, 32), (1, 16, 128), (1, 100, 5120), (1, 517, 96), (2, 640, 544), (15, 33, 1056), (16, 64, 256), (17, 300, 512), (31, 47, 160), (32, 257, 2048),
          (33, 64, 640), (45, 1024, 1024), (64, 130, 416), (65, 200, 3200), (127, 255, 544), (128, 384, 256), (200, 96, 1120), (257, 513, 768),
          (300, 1000, 672), (520, 777, 2080), (1025, 515, 1536),
          # the larger tiles of both forms, K of one tile to three groups, and between
          (520, 2105, 32), (257, 4099, 544), (1025, 2050, 288), (1025, 2047, 1120), (1025, 4100, 416), (700, 6150, 1056), (2000, 6390, 160), (130, 14300, 672), (2048, 6400, 512), (1900, 6301, 1696), (1100, 5120, 288)]


@pytest.mark.parametrize("T,N,K", SHAPES)
@pytest.mark.parametrize("bf", [False, True], ids=["x4", "xbf16"])
def test_product(T, N, K, bf):
    _say("product", T, N, K, "bf16" if bf else "4 bits")
    X, W, x, w = _operands(T, N, K, T + N + K, bf)
    want, off = x @ w.T, _off(x, w, bf)
    _check(mx4_gemm(X, W, out="f32"), want, off)
    _check(mx4_gemm(X, W), want, off)
    r = torch.randn(T, N, device="cuda")
    # the residual's addition rounds once more
    both = want + _np(r)
    _check(mx4_gemm(X, W, residual=r), both, off + 2.0 ** -24 * (np.abs(both) + off))
    y = r.clone()
    mx4_gemm(X, W, Y=y, residual=y)
    _check(y, both, off + 2.0 ** -24 * (np.abs(both) + off))


@pytest.mark.parametrize("T", [1, 20, 60, 300])
@pytest.mark.parametrize("bf", [False, True], ids=["x4", "xbf16"])
def test_product_strides(T, bf):
    """Rows of X, Y and the residual that lie apart, Y at an odd element: what lies between stays as it was."""
    N, K = 203, 288
    _say("strides", T, bf)
    X, W, x, w = _operands(T, N, K, T, bf)
    if bf:
        wide = torch.full((T, K + 40), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, 16:16 + K] = X
        X = wide[:, 16:16 + K]
    want, off = x @ w.T, _off(x, w, bf)
    for lead, dtype in ((1, torch.bfloat16), (4, torch.float32), (3, torch.float32)):
        y = torch.full((T + 2, N + 21), 3.0, dtype=dtype, device="cuda")
        mx4_gemm(X, W, Y=y[1:-1, lead:lead + N])
        _check(y[1:-1, lead:lead + N], want, off)
        y[1:-1, lead:lead + N] = 3
        assert (y == 3).all()
    r = torch.randn(T, N + 5, device="cuda")
    _check(mx4_gemm(X, W, residual=r[:, 2:2 + N]), want + _np(r[:, 2:2 + N]), off * 1.001 + 2.0 ** -24 * np.abs(want + _np(r[:, 2:2 + N])))


@pytest.mark.parametrize("T", [1, 17, 50, 300])
@pytest.mark.parametrize("bf", [False, True], ids=["x4", "xbf16"])
def test_product_bad_values(T, bf):
    """A NaN block of W makes its column NaN, one of X its row, and nothing else."""
    N, K = 90, 672
    X, W, x, w = _operands(T, N, K, 7, bf)
    code, scale = _held(W)
    scale[41, 20] = 255
    W = _matrix(code, scale)
    row = T - 1
    if bf:
        X[row, 100] = float("inf")
        X[row, 101] = -float("inf")
    else:
        xc, xs = _held(X)
        xs[row, 3] = 255
        X = _matrix(xc, xs)
    _say("bad values", T, bf)
    y = _np(mx4_gemm(X, W, out="f32"))
    bad = np.zeros((T, N), dtype=bool)
    bad[row], bad[:, 41] = True, True
    if bf:   # +inf and -inf times codes that may be zero or of either sign: NaN or an infinity
        assert not np.isfinite(y[row]).any() and np.isnan(y[:, 41]).all()
    else:
        assert np.isnan(y[bad]).all()
    want, off = x @ w.T, _off(x, w, bf)
    assert (np.abs(y - want) <= off + 2.0 ** -23 * np.abs(want))[~bad].all()


@pytest.mark.parametrize("T", [3, 40, 300])
def test_product_scales_far_apart(T):
    """Blocks between 2^-100 and 2^20 of W against activations that bring them back: no block's scale is lost or taken twice."""
    N, K = 70, 512
    r = np.random.default_rng(5)
    e = r.integers(-100, 21, K // 32)
    e[::3] = r.integers(-3, 4, len(e[::3]))
    code_w, code_x = r.integers(0, 16, (N, K), dtype=np.uint8), r.integers(0, 16, (T, K), dtype=np.uint8)
    sw, sx = np.broadcast_to(127 + e, (N, K // 32)).astype(np.uint8), np.broadcast_to(127 - e, (T, K // 32)).astype(np.uint8)
    x, w = ref.values(code_x, sx), ref.values(code_w, sw)
    _say("scales far apart", T)
    _check(mx4_gemm(_matrix(code_x, sx), _matrix(code_w, sw), out="f32"), x @ w.T, _off(x, w, False))
    xb = torch.from_numpy(x.astype(np.float32)).to(torch.bfloat16)
    assert np.array_equal(_np(xb), x)
    _check(mx4_gemm(xb.cuda(), _matrix(code_w, sw), out="f32"), x @ w.T, _off(x, w, True))


@pytest.mark.parametrize("bf", [False, True], ids=["x4", "xbf16"])
@pytest.mark.parametrize("T", [1, 40, 300])
def test_rows_do_not_depend_on_the_others(T, bf):
    """The same call gives the same bits; a captured one too, replayed with other work between, on another stream."""
    N, K = 530, 1056
    X, W, x, w = _operands(T, N, K, 11, bf)
    _say("repeat", T, bf)
    y = mx4_gemm(X, W, out="f32")
    assert torch.equal(mx4_gemm(X, W, out="f32"), y)
    out = torch.empty_like(y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mx4_gemm(X, W, Y=out)
    for _ in range(3):
        out.fill_(float("nan"))
        g.replay()
        torch.mm(torch.ones(64, 64, device="cuda"), torch.ones(64, 64, device="cuda"))
        torch.cuda.synchronize()
        assert torch.equal(out, y)
    s = torch.cuda.Stream()
    out.fill_(0)
    s.wait_stream(torch.cuda.current_stream())
    mx4_gemm(X, W, Y=out, stream=s)
    s.synchronize()
    assert torch.equal(out, y)


def test_quantise_in_a_graph():
    x = _rows(50, 544, 3).cuda()
    m, v = Mx4Matrix(50, 544), torch.empty(50, 544, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.quantise(x).values(out=v)
    for seed in (4, 5, 6):
        y = _rows(50, 544, seed)
        x.copy_(y)
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(_np(v), ref.values(*ref.quantise(_np(y))))


@pytest.mark.parametrize("bf", [False, True], ids=["x4", "xbf16"])
def test_two_streams(bf):
    """Calls that overlap on two streams give what they give alone."""
    calls, alone, out = [], [], []
    for T, N, K, seed in ((300, 2050, 1056, 1), (40, 5000, 2080, 2)):
        X, W = _operands(T, N, K, seed, bf)[:2]
        calls.append((X, W))
        alone.append(mx4_gemm(X, W, out="f32"))
        out.append([torch.zeros_like(alone[-1]) for _ in range(8)])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(8):
        for (X, W), y, s in zip(calls, out, streams):
            mx4_gemm(X, W, Y=y[i], stream=s)
    torch.cuda.synchronize()
    for want, ys in zip(alone, out):
        assert all(torch.equal(y, want) for y in ys)


def test_outputs_beyond_32_bits():
    """Y of more than 2^32 bytes, with rows of X in both types: the rows at both ends and across 2^31 and 2^32 bytes as a call on them alone."""
    T, N, K = _lib.MX4_MAX, 2080, 64
    _say("large Y", T, N, K)
    x = torch.randn(T, K, device="cuda", dtype=torch.bfloat16)
    W, X = Mx4Matrix.quantised(torch.randn(N, K, device="cuda")), Mx4Matrix.quantised(x)
    at = [0, (1 << 31) // (2 * N) // 16 * 16, (1 << 32) // (2 * N) // 16 * 16, T - 64]
    for big in (X, x):
        y = mx4_gemm(big, W)
        for t in at:
            part = x[t:t + 64].contiguous()
            want = mx4_gemm(part if big is x else Mx4Matrix.quantised(part), W, out="f32").double()
            got = y[t:t + 64].double()
            # K of one tile: the forms' sums differ in their order at most, 128 terms, and both round
            mag = part.double().abs() @ W.values().double().abs().T * 2      # 4-bit values of X are off by less than themselves
            assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15 * mag).all()), t
        del y


def test_matrices_beyond_32_bits():
    """A matrix of more than 2^32 bytes of codes: quantised, read back, and as the weight of few and of more rows."""
    N, K = _lib.MX4_MAX, 8320
    _say("large W", N, K)
    x = torch.empty(N, K, device="cuda", dtype=torch.bfloat16)
    x.normal_()
    W = Mx4Matrix.quantised(x)
    tail = Mx4Matrix.quantised(x[-100:].contiguous())
    assert W.codes.numel() > 1 << 32
    v = W.values(out=x)
    want = tail.values()
    assert torch.equal(v[-100:], want)
    del v, x
    for T in (3, 70):
        xb = torch.randn(T, K, device="cuda", dtype=torch.bfloat16)
        X = Mx4Matrix.quantised(xb)
        for rows, values in ((X, X.values()), (xb, xb)):
            y = mx4_gemm(rows, W, out="f32")[:, -100:]
            exact = _np(values) @ _np(want).T
            _check(y, exact, _off(_np(values), _np(want), rows is xb))
            del y


def test_empty():
    W = _operands(1, 20, 64, 1, True)[1]
    assert mx4_gemm(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), W).shape == (0, 20)
    assert mx4_gemm(Mx4Matrix(0, 64), W).shape == (0, 20)
    assert Mx4Matrix(0, 64).quantise(torch.empty(0, 64, device="cuda")).values().shape == (0, 64)
