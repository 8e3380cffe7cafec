"""Overlaps of what a call writes with what it reads: the host's checks against every byte, and the refusals."""
import ctypes
import subprocess
from pathlib import Path

import pytest

from cleffa_amd import _lib
from tests.test_mx4 import _refused, _rotary_args

CSRC = Path(__file__).resolve().parents[1] / "cleffa_amd" / "csrc"
CHECK = r"""
#include <cstdio>
#include <cstdlib>
#include <set>
#include "ranges.h"
using namespace clef_hip;
static std::set<uintptr_t> bytes(const Heads &h) {
    std::set<uintptr_t> s;
    for (long t = 0; t < h.rows; t++)
        for (long i = 0; i < h.heads; i++)
            for (long b = 0; b < h.bytes; b++) s.insert(h.at + t * h.row + i * h.head + b);
    return s;
}
static bool share(const std::set<uintptr_t> &a, const std::set<uintptr_t> &b) {
    for (uintptr_t v : a) if (b.count(v)) return true;
    return false;
}
static int bad = 0, hits = 0;
static void expect(bool got, bool want, const char *what) { hits += want; if (got != want && bad++ < 5) printf("%s: %d, not %d\n", what, got, want); }
int main() {
    srand(1);
    auto r = [](int n) { return (long)(rand() % n); };
    for (int i = 0; i < 200000; i++) {
        const bool same = r(2);
        Rows a{(uintptr_t)(100 + r(60)), 1 + r(5), r(24), 1 + r(9)}, b{(uintptr_t)(100 + r(60)), 1 + r(5), r(24), 1 + r(9)};
        if (same) b.stride = a.stride;
        const auto sa = bytes(Heads{a.at, a.n, a.stride, 1, 0, a.bytes}), sb = bytes(Heads{b.at, b.n, b.stride, 1, 0, b.bytes});
        expect(meet(a, b), share(sa, sb), "rows");
        const uintptr_t lo = 100 + r(80), hi = lo + r(12);
        bool in = false;
        for (uintptr_t v : sa) in |= v >= lo && v < hi;
        expect(meets(a, lo, hi), in, "a range");
    }
    for (int i = 0; i < 200000; i++) {
        const long T = 1 + r(4);
        Heads a{(uintptr_t)(100 + r(200)), T, T > 1 ? r(50) : 0, 1 + r(4), r(30), 1 + r(6)}, b = a;
        b.at = 100 + r(200); b.heads = 1 + r(4); b.head = r(30); b.bytes = 1 + r(6);
        if (r(4) == 0 && T > 1) b.row = r(50);
        const bool want = share(bytes(a), bytes(b)), got = meet(a, b);
        if (a.row == b.row) expect(got, want, "heads");
        else if (want) expect(got, want, "heads of rows of different lengths");    // or refused, where rows as a whole meet
    }
    printf("%d wrong of the checks, %d of them overlap\n", bad, hits);
    return bad != 0;
}
"""


def test_against_every_byte(tmp_path):
    (tmp_path / "c.cpp").write_text(CHECK)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", str(CSRC), str(tmp_path / "c.cpp"), "-o", str(tmp_path / "c")], check=True)
    out = subprocess.run([str(tmp_path / "c")], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert out.stdout.startswith("0 wrong") and int(out.stdout.split()[5]) > 10000


BASE = 1 << 30
P = ctypes.c_void_p


def _product(**over):
    """Y f32 [64][300] of rows 400 apart at BASE; W [300][160], X [64][160], all apart."""
    a = _lib.Mx4GemmArgs(64, 300, 160, 0, P(1 << 24), P(1 << 25), P(1 << 26), P(1 << 27), None, 0, 400, 0, P(BASE), None)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _bf16(at, row=400, **over):
    return _product(x_codes=None, x_scales=None, x_bf16=P(at), x_row=row, **over)


# Y's last byte is 4 * (63 * 400 + 300) behind BASE; W's codes are 19 row tiles x 2 K tiles x 1 KB, its scales 19 x 256 bytes; X's 4 x 2 KB and 1 KB
END = 4 * (63 * 400 + 300)


@pytest.mark.parametrize("args,msg", [
    (_product(w_codes=P(BASE)), "Y overlaps W"), (_product(w_codes=P(BASE - 19 * 2048 + 16)), "Y overlaps W"), (_product(w_scales=P(BASE + END - 16)), "Y overlaps W"),
    (_product(w_scales=P(BASE + 1600 * 7 + 1184)), "Y overlaps W"), (_product(x_codes=P(BASE - 4 * 2048 + 16)), "Y overlaps X"),
    (_product(x_scales=P(BASE + 1600 * 7 + 1200)), "Y overlaps X"), (_product(y_type=1, x_scales=P(BASE + 2 * (63 * 400 + 300) - 24)), "Y overlaps X"),
    (_bf16(BASE), "Y overlaps X"), (_bf16(BASE + 1200, 800, K=224), "Y overlaps X"), (_bf16(BASE + END - 16), "Y overlaps X"), (_bf16(BASE + 1120, 800), "Y overlaps X"),
    (_bf16(BASE + 1200, 808), "Y overlaps X"),
    (_product(y_row=1 << 50), "too far apart"), (_product(residual=P(1 << 28), r_row=1 << 50), "too far apart"), (_bf16(1 << 28, 1 << 50), "too far apart"),
])
def test_product_overlaps(args, msg):
    _refused(_lib.load().clef_hip_mx4_gemm, args, msg)


def _pair(T=6, row=4096, **over):
    """q heads 512 apart and k heads behind them in the same rows, turned in place; f32."""
    a = _lib.RotaryArgs(T, 256, 64, 0, 1, 2, 1e-6, 1.0, P(1 << 24), P(1 << 25), *(4, P(BASE), P(BASE), row, 512, row, 512, None),
                        *(2, P(BASE + 8192), P(BASE + 8192), row, 256, row, 256, None))
    for k, v in over.items():
        setattr(a, k.replace("__", "."), v)
    return a


@pytest.mark.parametrize("args", [
    _pair(k__out=P(BASE)), _pair(q__out=P(BASE + 8192)), _pair(q__out=P(BASE + 4)), _pair(k__x=P(BASE + 8192 - 512 * 4)), _pair(q__out=P(BASE + 4096 * 4 * 5)),
    _pair(q__out=P(1 << 29), k__out=P((1 << 29) + 4 * 200), k__out_head=512), _pair(T=1, k__out=P(BASE + 255 * 4)), _pair(q__out=P(1 << 29), k__out=P(1 << 29)),
    _pair(k__x=P(1 << 28), k__out=P(BASE + 128), k__out_row=4100), _pair(bf16_out=1, q__out=P(BASE + 2 * 1024), k__out=P(1 << 29)),
])
def test_rotary_overlaps(args):
    _refused(_lib.load().clef_hip_rotary, args, "overlaps")


@pytest.mark.parametrize("over", [dict(x_row=1 << 50), dict(out_row=1 << 50), dict(x_head=1 << 50), dict(out_head=1 << 50, out_row=1 << 50)])
def test_rotary_too_far_apart(over):
    _refused(_lib.load().clef_hip_rotary, _rotary_args(**over), "too far apart")


def test_strides_of_no_heads_do_not_count():
    a = _pair(k__heads=0, k__x_row=(1 << 63) - 1, k__out_row=(1 << 63) - 1, q__out=P(BASE + 4))
    _refused(_lib.load().clef_hip_rotary, a, "overlaps")


# 20 rows of 160 values, 240 apart, at BASE; codes 2 x 2 KB, scales 2 x 256 bytes
@pytest.mark.parametrize("fn", ["quantise", "values"])
@pytest.mark.parametrize("type_,codes,scales", [
    (0, BASE, 1 << 24), (0, 1 << 24, BASE), (0, BASE - 4096 + 16, 1 << 24), (0, 1 << 24, BASE + 2 * (19 * 240 + 160) - 16), (2, BASE + 4 * (19 * 240 + 160) - 16, 1 << 24),
    (2, 1 << 24, BASE + 4 * 160), (0, BASE + 320, 1 << 24)])
def test_rows_over_their_matrix(fn, type_, codes, scales):
    a = _lib.Mx4RowsArgs(20, 160, type_, 240, P(BASE), P(codes), P(scales))
    _refused(getattr(_lib.load(), "clef_hip_mx4_" + fn), a, "overlaps")


@pytest.mark.parametrize("fn", ["quantise", "values"])
def test_rows_too_far_apart(fn):
    _refused(getattr(_lib.load(), "clef_hip_mx4_" + fn), _lib.Mx4RowsArgs(20, 160, 0, 1 << 50, P(BASE), P(1 << 24), P(1 << 25)), "too far apart")


@pytest.mark.parametrize("flat_codes,flat_scales", [(BASE, 1 << 24), (1 << 24, BASE), (BASE - 20 * 80 + 16, 1 << 24), (BASE + 4080, 1 << 24), (1 << 24, BASE + 4095), (BASE + 8192, 1 << 24),
                                                    (1 << 24, BASE + 8192 + 511)])
@pytest.mark.parametrize("to_flat", [0, 1])
def test_pack_over_its_matrix(flat_codes, flat_scales, to_flat):
    err = ctypes.create_string_buffer(256)
    assert not _lib.load().clef_hip_mx4_pack(20, 160, flat_codes, flat_scales, BASE, BASE + 8192, to_flat, None, err, 256)
    assert "overlap" in err.value.decode()
