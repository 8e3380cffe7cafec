"""The interfaces of the 4-bit matrices and of the rotary operator without a GPU: struct layouts, sizes, refusals,
frequency tables and the reference's own arithmetic."""
import ctypes
import math
import re
import subprocess
from pathlib import Path
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from cleffa_amd import Mx4Matrix, Rotary, TextAttention, _lib, mx4_gemm
from tests import mx4_ref

HEADER = Path(__file__).resolve().parents[1] / "include" / "clef_hip_attn.h"
FAKE = ctypes.c_void_p(1 << 20)   # aligned, never read: every case fails a check first
ODD = ctypes.c_void_p((1 << 20) + 1)


def _err():
    return ctypes.create_string_buffer(256)


@pytest.mark.parametrize("name,cls", [("clef_hip_mx4_rows_args", _lib.Mx4RowsArgs), ("clef_hip_mx4_gemm_args", _lib.Mx4GemmArgs),
                                      ("clef_hip_rotary_args", _lib.RotaryArgs)])
def test_struct_layouts(name, cls, tmp_path):
    """The ctypes mirrors have the C compiler's offsets and sizes."""
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"clef_hip_attn.h\"\nint main(void) {\n"
    src += "".join(f'printf("%zu %zu\\n", offsetof({name}, {f}), sizeof((({name} *)0)->{f}));\n' for f, _ in cls._fields_)
    src += f'printf("%zu\\n", sizeof({name}));\nreturn 0;\n}}\n'
    (tmp_path / "l.c").write_text(src)
    subprocess.run(["gcc", "-std=c99", "-I", str(HEADER.parent), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    lines = subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split("\n")
    for (f, _), line in zip(cls._fields_, lines):
        d = getattr(cls, f)
        assert line == f"{d.offset} {d.size}", f
    assert int(lines[len(cls._fields_)]) == ctypes.sizeof(cls)


def test_constants_match_the_header():
    text = HEADER.read_text()
    for name, value in (("MX4_BLOCK", _lib.MX4_BLOCK), ("MX4_MAX", _lib.MX4_MAX), ("ROTARY_ROWS", _lib.ROTARY_ROWS), ("ROTARY_LINEAR", _lib.ROTARY_SCALINGS["linear"]),
                        ("ROTARY_BASE", _lib.ROTARY_SCALINGS["base"]), ("ROTARY_PARTS", _lib.ROTARY_SCALINGS["parts"]),
                        ("ROTARY_HALF", _lib.ROTARY_LAYOUTS["half"]), ("ROTARY_INTERLEAVED", _lib.ROTARY_LAYOUTS["interleaved"])):
        assert int(re.search(rf"#define CLEF_HIP_{name} (\d+)", text).group(1)) == value


def _sizes(rows, K):
    c, s, err = ctypes.c_size_t(0), ctypes.c_size_t(0), _err()
    ok = _lib.load().clef_hip_mx4_sizes(rows, K, ctypes.byref(c), ctypes.byref(s), err, 256)
    return (c.value, s.value) if ok else err.value.decode()


def test_sizes():
    assert _sizes(0, 32) == (0, 0)
    assert _sizes(1, 32) == (1024, 256)
    assert _sizes(17, 544) == (2 * 5 * 1024, 2 * 2 * 256)
    assert _sizes(14336, 5120) == (14336 * 5120 // 2, 14336 * 5120 // 32)
    for args in ((-1, 32), (1, 0), (1, 33), (1, 16), (_lib.MX4_MAX + 1, 32), (1, 2 * _lib.MX4_MAX), (_lib.MX4_MAX, _lib.MX4_MAX)):
        assert _sizes(*args).startswith("hip: "), args
    assert _lib.load().clef_hip_mx4_sizes(1, 32, None, None, None, 0)


def _refused(fn, args, msg):
    err = _err()
    assert not fn(ctypes.byref(args) if args is not None else None, None, err, 256)
    text = err.value.decode()
    assert text.startswith("hip: ") and msg in text, text


@pytest.mark.parametrize("over,msg", [
    (dict(rows=-1), "rows"), (dict(K=48), "multiples of 32"), (dict(K=0), "multiples of 32"), (dict(type=3), "type"), (dict(row=56), "multiple of 8"),
    (dict(row=68), "multiple of 8"), (dict(x=None), "x must be"), (dict(x=ODD), "x must be"), (dict(codes=None), "codes"), (dict(scales=ODD), "scales"),
])
@pytest.mark.parametrize("fn", ["quantise", "values"])
def test_rows_refusals(fn, over, msg):
    a = _lib.Mx4RowsArgs(8, 64, 0, 64, FAKE, FAKE, FAKE)
    for k, v in over.items():
        setattr(a, k, v)
    _refused(getattr(_lib.load(), "clef_hip_mx4_" + fn), a, msg)
    _refused(getattr(_lib.load(), "clef_hip_mx4_" + fn), None, "null")


def test_values_refuse_f16():
    _refused(_lib.load().clef_hip_mx4_values, _lib.Mx4RowsArgs(8, 64, 1, 64, FAKE, FAKE, FAKE), "type")


@pytest.mark.parametrize("over,msg", [
    (dict(T=-1), "rows"), (dict(N=0), "no rows"), (dict(K=40), "multiples of 32"), (dict(y_type=2), "y_type"),
    (dict(y_type=1, residual=FAKE), "f32 Y"), (dict(y_row=99), "rows of Y"), (dict(residual=FAKE, r_row=99), "rows of Y"),
    (dict(x_scales=None), "both"), (dict(x_bf16=FAKE), "in 4 bits or in bf16"), (dict(x_codes=None, x_scales=None), "in 4 bits or in bf16"),
    (dict(x_codes=None, x_scales=None, x_bf16=ODD, x_row=64), "X must be"), (dict(x_codes=None, x_scales=None, x_bf16=FAKE, x_row=60), "X must be"),
    (dict(w_codes=None), "W codes"), (dict(w_scales=ODD), "W codes"), (dict(x_codes=ODD), "X codes"), (dict(y=None), "Y and"), (dict(y=ODD), "Y and"),
])
def test_product_refusals(over, msg):
    a = _lib.Mx4GemmArgs(8, 100, 64, 0, FAKE, FAKE, FAKE, FAKE, None, 0, 100, 0, FAKE, None)
    for k, v in over.items():
        setattr(a, k, v)
    _refused(_lib.load().clef_hip_mx4_gemm, a, msg)
    _refused(_lib.load().clef_hip_mx4_gemm, None, "null")


@pytest.mark.parametrize("at,r_row,y_row,ok", [
    (0, 200, 200, True), (0, 204, 200, False), (400, 200, 200, True), (404, 200, 200, False), (396, 200, 200, False), (-400, 200, 200, True), (-396, 200, 200, False),
    (4 * 200 * 7 + 400, 200, 200, True), (4 * 200 * 7 + 396, 200, 200, False), (4 * 200 * 7 + 396, 100, 200, False), (4 * 200 * 7 + 400, 100, 200, True), (-4 * 800, 100, 200, True),
    (-4 * 799, 100, 200, False), (1000, 200, 200, False), (1200, 200, 200, True), (1200, 200, 201, False),
])
def test_residual_overlap(at, r_row, y_row, ok):
    """The residual is Y, lies apart from it, or between its rows; a call that passes fails at the next check, X's."""
    a = _lib.Mx4GemmArgs(8, 100, 64, 0, FAKE, FAKE, FAKE, FAKE, None, 0, y_row, r_row, 1 << 20, (1 << 20) + at)
    if ok:
        a.x_codes = ODD
    _refused(_lib.load().clef_hip_mx4_gemm, a, "X codes" if ok else "overlap")


def test_no_rows_are_no_work():
    lib, err = _lib.load(), _err()
    assert lib.clef_hip_mx4_gemm(ctypes.byref(_lib.Mx4GemmArgs(0, 8, 32, 0, None, None, None, None, FAKE, 32, 8, 0, None, None)), None, err, 256)
    assert lib.clef_hip_mx4_quantise(ctypes.byref(_lib.Mx4RowsArgs(0, 32, 0, 32, None, None, None)), None, err, 256)
    assert lib.clef_hip_mx4_values(ctypes.byref(_lib.Mx4RowsArgs(0, 32, 0, 32, None, None, None)), None, err, 256)
    assert lib.clef_hip_mx4_pack(0, 32, None, None, None, None, 0, None, err, 256)
    none = (0, None, None, 0, 0, 0, 0, None) * 2
    assert lib.clef_hip_rotary(ctypes.byref(_lib.RotaryArgs(0, 64, 64, 0, 1, 0, 1e-6, 1.0, None, None, *none)), None, err, 256)
    assert lib.clef_hip_rotary(ctypes.byref(_lib.RotaryArgs(4, 64, 64, 0, 1, 0, 1e-6, 1.0, None, None, *none)), None, err, 256)


def _rotary_args(**over):
    heads = dict(heads=4, x=FAKE, out=FAKE, x_row=512, x_head=128, out_row=512, out_head=128, norm=None)
    a = _lib.RotaryArgs(3, 128, 64, 0, 1, 0, 1e-6, 1.0, FAKE, FAKE, *heads.values(), *heads.values())
    for k, v in over.items():
        setattr(a, "q." + k if k in heads else k, v)
    return a


@pytest.mark.parametrize("over,msg", [
    (dict(T=-1), "rows"), (dict(hd=258), "head dim"), (dict(hd=127), "head dim"), (dict(hd=0), "head dim"), (dict(n_rot=130), "n_rot"), (dict(n_rot=0), "n_rot"),
    (dict(n_rot=63), "n_rot"), (dict(layout=2), "layout"), (dict(axes=0), "axes"), (dict(axes=5), "axes"), (dict(type=3), "type"), (dict(eps=-1.0), "eps"),
    (dict(magnitude=math.inf), "magnitude"), (dict(pos=None), "pos"), (dict(freq=None), "freq"), (dict(heads=-1), "heads"), (dict(x=None), "aligned"),
    (dict(out=ODD), "aligned"), (dict(type=2, x=ctypes.c_void_p((1 << 20) + 2)), "aligned"), (dict(norm=ODD), "aligned"), (dict(out_head=64, x_head=64), "overlap"),
    (dict(T=_lib.ROTARY_ROWS + 1), "rows"), (dict(out_row=256, x_row=256), "overlap"), (dict(x_row=-512), "negative"), (dict(x_row=1024), "same strides"), (dict(x_head=256), "same strides"),
])
def test_rotary_refusals(over, msg):
    _refused(_lib.load().clef_hip_rotary, _rotary_args(**over), msg)


def test_rotary_takes_heads_of_rows():
    """[heads][T][hd] strides are no overlap: the call fails at the next check, not at that one."""
    _refused(_lib.load().clef_hip_rotary, _rotary_args(x_row=128, out_row=128, x_head=384, out_head=384, pos=None), "pos")


def test_device_is_needed():
    m = Mx4Matrix(4, 64, device="cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        m.quantise(torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match="GPU"):
        mx4_gemm(torch.zeros(4, 64, dtype=torch.bfloat16), m)
    with pytest.raises(RuntimeError, match="GPU"):
        Rotary(32, device="cpu").apply(torch.zeros(2, 1, 64), None, torch.zeros(2, dtype=torch.int32))


def test_python_refusals():
    m, w = Mx4Matrix(4, 64, device="cpu"), Mx4Matrix(5, 64, device="cpu")
    for x, e in ((torch.zeros(4, 32), ValueError), (torch.zeros(5, 64), ValueError), (torch.zeros(4, 64, dtype=torch.float64), TypeError), (None, TypeError),
                 (torch.zeros(64, 4).T, ValueError), (torch.zeros(4, 68)[:, :64], ValueError), (torch.zeros(4, 72)[:, 1:65], ValueError)):
        with pytest.raises(e):
            m.quantise(x)
    bf = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: mx4_gemm(bf[:, :32], w), lambda: mx4_gemm(bf, bf), lambda: mx4_gemm(bf.float(), w), lambda: mx4_gemm(bf, w, Y=torch.zeros(4, 4)),
                 lambda: mx4_gemm(bf, w, Y=torch.zeros(4, 5, dtype=torch.float16)), lambda: mx4_gemm(bf, w, out="f16"), lambda: m.values(out_dtype="f16"),
                 lambda: mx4_gemm(bf, w, residual=torch.zeros(4, 4)), lambda: m.first(5), lambda: Mx4Matrix(20, 64, device="cpu").first(5),
                 lambda: Mx4Matrix(4, 48, device="cpu"), lambda: Mx4Matrix.from_codes(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            call()
    with pytest.raises(ValueError):
        Rotary(32, layout="pairs", device="cpu")
    for scaling in ({"kind": "other"}, {"factor": 2.0}, {"kind": "linear", "factor": 0.5}, {"kind": "parts", "factor": 2.0}, {"kind": "linear", "rate": 2.0},
                    {"kind": "parts", "factor": 2.0, "original": 100, "low": 4, "high": 4}):
        with pytest.raises((ValueError, RuntimeError)):
            Rotary(32, scaling=scaling, device="cpu")
    r = Rotary(32, axes=3, device="cpu")
    q, pos = torch.zeros(2, 4, 64), torch.zeros(2, 3, dtype=torch.int32)
    for call in (lambda: r.apply(q.double(), None, pos), lambda: r.apply(q, None, pos[:, :2].contiguous()), lambda: r.apply(q, q.half(), pos),
                 lambda: r.apply(q, None, pos.long()), lambda: r.apply(q, None, pos, k_norm=torch.ones(64)), lambda: r.apply(q, None, pos, q_out=q[:, :2]),
                 lambda: r.apply(q, None, pos, q_norm=torch.ones(32)), lambda: r.apply(q[0], None, pos), lambda: r.apply(q.transpose(1, 2), None, pos)):
        with pytest.raises((TypeError, ValueError)):
            call()


def test_project_refuses_mixed_operands():
    att = SimpleNamespace(device=torch.device("cpu"), row=2048)
    with pytest.raises(TypeError, match="4 bits"):
        TextAttention.project(att, Mx4Matrix(8, 64, device="cpu"), torch.zeros(att.row, 64, dtype=torch.bfloat16), SimpleNamespace(T=8))


def test_reference_grid():
    """Every code of the format decodes to its value and codes back to itself, ties go to even codes, and the scale rule's borders."""
    code = np.arange(16, dtype=np.uint8).repeat(2).reshape(1, 32)
    for s in (0, 1, 127, 252):
        v = mx4_ref.values(code, np.array([[s]], dtype=np.uint8))
        c, e = mx4_ref.quantise(v)
        assert e[0, 0] == s and np.array_equal(mx4_ref.values(c, e), v)
    row = np.zeros((1, 32))
    row[0, :9] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25]
    c, e = mx4_ref.quantise(row)
    assert e[0, 0] == 127 and list(c[0, :9] & 7) == [7, 0, 2, 2, 4, 4, 6, 6, 0]
    for most, s in ((7 - 2 ** -40, 127), (7, 128), (6.5, 127), (3.5, 127), (3.5 - 2 ** -40, 126)):
        row[:] = 0
        row[0, 3] = most
        assert mx4_ref.quantise(row)[1][0, 0] == s, most
    assert np.array_equal(mx4_ref.unflat(mx4_ref.flat(code)), code)


@pytest.mark.parametrize("n", [2, 64, 72, 256])
def test_frequency_tables(n):
    two_pi = 2 * math.pi
    j = np.arange(n // 2)
    f = 1e7 ** (-2 * j / n)

    def table(**kw):
        return Rotary(n, theta=1e7, device="cpu", **kw).freq.numpy() * two_pi
    # pow, a product and a division in float64: a few roundings each
    close = dict(rtol=2.0 ** -48, atol=0)
    np.testing.assert_allclose(table(), f, **close)
    np.testing.assert_allclose(table(scaling={"kind": "linear", "factor": 8}), f / 8, **close)
    np.testing.assert_allclose(table(freqs=f * 1.5), f * 1.5, **close)
    if n > 2:
        np.testing.assert_allclose(table(scaling={"kind": "base", "factor": 4.0}), (1e7 * 4 ** (n / (n - 2))) ** (-2 * j / n), rtol=2.0 ** -46)
        # the last pair is stretched by the whole factor
        assert math.isclose(table(scaling={"kind": "base", "factor": 4.0})[-1], f[-1] / 4, rel_tol=1e-12)
    parts = table(scaling={"kind": "parts", "factor": 8.0, "original": 4096, "low": 1, "high": 32})
    r = 4096 * f / two_pi
    want = np.where(r >= 32, f, np.where(r <= 1, f / 8, 0))
    assert np.allclose(parts[want > 0], want[want > 0], **close)
    for i in np.nonzero(want == 0)[0]:
        keep = (r[i] - 1) / 31
        assert math.isclose(parts[i], keep * f[i] + (1 - keep) * f[i] / 8, rel_tol=1e-13)
    assert Rotary(n, scaling={"kind": "parts", "factor": 8.0, "original": 4096}, device="cpu").magnitude == 0.1 * math.log(8) + 1
    assert Rotary(n, scaling={"kind": "parts", "factor": 8.0, "original": 4096}, magnitude=1.0, device="cpu").magnitude == 1
    assert Rotary(n, device="cpu").magnitude == 1
