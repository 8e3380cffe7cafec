"""What the 8-bit paged cache's calls are told of their buffers, without a GPU: a plan or workspace that is too short for a
call's sizes is refused before anything is launched."""
import ctypes

import pytest

from cleffa_amd import _lib

FAKE = ctypes.c_void_p(1 << 20)   # aligned, never read: every case fails a check first


def _sizes(n_seq, T, nh, nkv, max_new):
    ints, ws, err = ctypes.c_size_t(0), ctypes.c_size_t(0), ctypes.create_string_buffer(256)
    assert _lib.load().clef_hip_kv8_sizes(n_seq, T, nh, nkv, max_new, ctypes.byref(ints), ctypes.byref(ws), err, 256)
    return ints.value, ws.value


def _args(n_seq, T, nh, nkv, max_new):
    a = _lib.Kv8Args()
    a.nh, a.nkv, a.hd, a.n_rot, a.eps, a.scale, a.T, a.row = nh, nkv, 256, 64, 1e-6, 1 / 16, T, 512 * (nh + nkv)
    a.n_seq, a.max_pages, a.n_pages, a.max_new = n_seq, 16, 64, max_new
    for f in ("qkv", "q_norm", "k_norm", "pos3", "inv_freq", "tables", "k_pages", "v_pages", "k_scale", "v_scale", "plan", "out", "workspace"):
        setattr(a, f, FAKE)
    a.plan_ints, a.workspace_bytes = _sizes(n_seq, T, nh, nkv, max_new)
    return a


@pytest.mark.parametrize("sizes,made_for", [((8, 4096, 24, 4, 0), (8, 1, 24, 4, 0)), ((8, 64, 24, 4, 1), (8, 63, 24, 4, 1)),
                                            ((4096, 300, 16, 4, 0), (1, 300, 16, 4, 0)), ((3, 600, 64, 1, 0), (3, 600, 8, 1, 0))])
def test_a_plan_of_a_smaller_pass_is_refused(sizes, made_for):
    """The kernels read the lists where the call's sizes place them, so a buffer made for less is not looked at."""
    lib = _lib.load()
    for fn in (lib.clef_hip_kv8_append, lib.clef_hip_kv8_attention):
        a, err = _args(*sizes), ctypes.create_string_buffer(256)
        need, a.plan_ints = a.plan_ints, _sizes(*made_for)[0]
        assert a.plan_ints < need
        assert not fn(ctypes.byref(a), None, err, 256)
        assert err.value.decode() == f"hip: plan of {a.plan_ints} int32, {need} are needed"


@pytest.mark.parametrize("fn", ["clef_hip_kv8_append", "clef_hip_kv8_attention"])
def test_a_plan_one_short_is_refused(fn):
    a, err = _args(8, 64, 24, 4, 1), ctypes.create_string_buffer(256)
    a.plan_ints -= 1
    assert not getattr(_lib.load(), fn)(ctypes.byref(a), None, err, 256) and b"are needed" in err.value
    a.plan_ints = 0
    assert not getattr(_lib.load(), fn)(ctypes.byref(a), None, err, 256) and b"are needed" in err.value


def test_status_words_match_the_header():
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parents[1] / "include" / "clef_hip_attn.h").read_text()
    for name in ("STATUS", "FAILED"):
        assert int(re.search(rf"#define CLEF_HIP_KV8_PLAN_{name} (\d+)", text).group(1)) == getattr(_lib, "KV8_PLAN_" + name)
