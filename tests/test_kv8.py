"""The 8-bit paged cache's interface without a GPU: struct layouts, buffer sizes, refusals and the
reference's own arithmetic."""
import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from cleffa_amd import Kv8Cache, Kv8Plan, _lib
from tests import kv8_ref

HEADER = Path(__file__).resolve().parents[1] / "include" / "clef_hip_attn.h"
FAKE = ctypes.c_void_p(1 << 20)   # aligned, never read: every case fails a check first


def _err():
    return ctypes.create_string_buffer(256)


@pytest.mark.parametrize("name,cls", [("clef_hip_kv8_plan_args", _lib.Kv8PlanArgs), ("clef_hip_kv8_args", _lib.Kv8Args),
                                      ("clef_hip_kv8_read_args", _lib.Kv8ReadArgs)])
def test_struct_layouts(name, cls, tmp_path):
    """The ctypes mirrors have the C compiler's offsets and sizes."""
    import subprocess
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
    for name in ("PAGE", "MAX_SEQ", "MAX_ROWS"):
        assert int(re.search(rf"#define CLEF_HIP_KV8_{name} (\d+)", text).group(1)) == getattr(_lib, "KV8_" + name)


def _sizes(*a):
    ints, ws, err = ctypes.c_size_t(0), ctypes.c_size_t(0), _err()
    ok = _lib.load().clef_hip_kv8_sizes(*a, ctypes.byref(ints), ctypes.byref(ws), err, 256)
    return (ints.value, ws.value) if ok else err.value.decode()


def test_sizes():
    small, large = _sizes(8, 8, 24, 4, 1), _sizes(8, 4096, 24, 4, 0)
    assert 0 < small[0] < large[0] and 0 < small[1] <= large[1]
    assert _sizes(1, 0, 8, 8, 0)[0] >= 16                       # a pass of no rows has a header
    assert _sizes(_lib.KV8_MAX_SEQ, _lib.KV8_MAX_ROWS, 128, 1, 0)[0] < 1 << 31


@pytest.mark.parametrize("args,msg", [((0, 8, 24, 4, 1), "sequences"), ((4097, 8, 24, 4, 1), "sequences"), ((8, -1, 24, 4, 1), "pass rows"),
                                      ((8, 262144, 24, 4, 1), "pass rows"), ((8, 8, 24, 5, 1), "head counts"), ((8, 8, 0, 4, 1), "head counts"),
                                      ((8, 8, 129, 1, 1), "head counts"), ((8, 8, 2000, 2000, 1), "nkv")])
def test_sizes_refused(args, msg):
    got = _sizes(*args)
    assert isinstance(got, str) and got.startswith("hip: ") and msg in got


def _plan_args(**over):
    a = _lib.Kv8PlanArgs()
    a.n_seq, a.max_pages, a.n_pages, a.T, a.nh, a.nkv, a.max_new, a.plan_ints = 8, 16, 64, 8, 24, 4, 1, 1 << 20
    for f in ("tables", "free_pages", "state", "state_out", "new_lens", "cu_q", "slots", "plan"):
        setattr(a, f, FAKE)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,msg", [(dict(n_seq=0), "sequences"), (dict(max_pages=0), "table rows"), (dict(max_pages=65537), "table rows"),
                                      (dict(n_pages=0), "pool"), (dict(state=None), "missing"), (dict(slots=None), "missing"),
                                      (dict(cu_q=None), "missing"), (dict(plan_ints=15), "are needed"), (dict(nkv=5), "head counts"),
                                      (dict(plan=ctypes.c_void_p((1 << 20) + 4)), "plan must be")])
def test_plan_refused(over, msg):
    err = _err()
    assert not _lib.load().clef_hip_kv8_plan(ctypes.byref(_plan_args(**over)), None, err, 256)
    assert err.value.decode().startswith("hip: ") and msg in err.value.decode()


def _args(**over):
    a = _lib.Kv8Args()
    a.nh, a.nkv, a.hd, a.n_rot, a.eps, a.scale, a.T, a.row = 24, 4, 256, 64, 1e-6, 1 / 16, 8, 14336
    a.n_seq, a.max_pages, a.n_pages, a.max_new, a.workspace_bytes = 8, 16, 64, 1, 1 << 40
    for f in ("qkv", "q_norm", "k_norm", "pos3", "inv_freq", "tables", "k_pages", "v_pages", "k_scale", "v_scale", "plan", "out", "workspace"):
        setattr(a, f, FAKE)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,msg", [(dict(hd=128), "hd 256"), (dict(nh=25), "head counts"), (dict(n_rot=32), "n_rot"), (dict(row=14000), "qkv row"),
                                      (dict(row=14337), "qkv row"), (dict(qkv=None), "qkv"), (dict(q_norm=None), "both"), (dict(pos3=None), "rotary"),
                                      (dict(k_pages=ctypes.c_void_p((1 << 20) + 8)), "pages"), (dict(v_scale=None), "scales"), (dict(tables=None), "tables"),
                                      (dict(plan=None), "plan"), (dict(inv_freq=ctypes.c_void_p((1 << 20) + 4)), "inv_freq"), (dict(n_pages=1 << 30), "pool"), (dict(eps=float("nan")), "eps"), (dict(n_pages=-1), "pool")])
def test_append_and_attention_refused(over, msg):
    for fn in (_lib.load().clef_hip_kv8_append, _lib.load().clef_hip_kv8_attention):
        err = _err()
        assert not fn(ctypes.byref(_args(**over)), None, err, 256)
        assert err.value.decode().startswith("hip: ") and msg in err.value.decode()


@pytest.mark.parametrize("over,msg", [(dict(out=None), "out must"), (dict(out_type=3), "out_type"), (dict(scale=0.0), "scale"),
                                      (dict(workspace=None), "workspace"), (dict(workspace_bytes=1024), "are needed")])
def test_attention_refused(over, msg):
    err = _err()
    assert not _lib.load().clef_hip_kv8_attention(ctypes.byref(_args(**over)), None, err, 256)
    assert msg in err.value.decode()


@pytest.mark.parametrize("over,msg", [(dict(hd=64), "hd 256"), (dict(kvT=60), "kvT"), (dict(kvT=1 << 30), "kvT"), (dict(cu=None), "cu"),
                                      (dict(vt_plane=None), "planes"), (dict(n_seq=5000), "sequences")])
def test_read_refused(over, msg):
    a = _lib.Kv8ReadArgs()
    a.nkv, a.hd, a.n_seq, a.max_pages, a.n_pages, a.kvT = 4, 256, 8, 16, 64, 64
    for f in ("k_pages", "v_pages", "k_scale", "v_scale", "tables", "state", "cu", "k_plane", "vt_plane"):
        setattr(a, f, FAKE)
    for k, v in over.items():
        setattr(a, k, v)
    err = _err()
    assert not _lib.load().clef_hip_kv8_read(ctypes.byref(a), None, err, 256)
    assert msg in err.value.decode()


def test_null_arguments():
    lib = _lib.load()
    for fn in (lib.clef_hip_kv8_plan, lib.clef_hip_kv8_append, lib.clef_hip_kv8_attention, lib.clef_hip_kv8_read):
        assert not fn(None, None, None, 0)


def test_python_refusals():
    cache = Kv8Cache(2, 4, 16, 3, 8, device="cpu")
    with pytest.raises(ValueError, match="heads"):
        Kv8Plan(cache, 8, 6)
    with pytest.raises(ValueError, match="T -1"):
        Kv8Plan(cache, -1, 8)
    with pytest.raises(ValueError, match="layer 2"):
        cache.layer_args(2)
    with pytest.raises(ValueError, match="hd 256"):
        Kv8Cache(1, 4, 16, 3, 8, hd=128, device="cpu")
    with pytest.raises(ValueError, match="cache sizes"):
        Kv8Cache(1, 4, 16, 5000, 8, device="cpu")
    plan = Kv8Plan(cache, 8, 8)
    with pytest.raises(ValueError, match="new_lens has shape"):
        plan.update(torch.zeros(4, dtype=torch.int32))
    with pytest.raises(TypeError, match="new_lens"):
        plan.update(torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):       # there is no CPU path
        plan.update(torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU"):
        cache.read(0, torch.zeros(4, dtype=torch.int32), torch.zeros(4, 64, 256, dtype=torch.float16), torch.zeros(4, 256, 64, dtype=torch.bfloat16))
    cache.k[0] = cache.k[0][:8]
    with pytest.raises(ValueError, match="k pages"):
        cache.layer_args(0)


def test_reference_codes():
    """The reference's e4m3 against torch's conversion, over every code and between codes."""
    every = torch.arange(256, dtype=torch.uint8)
    want = every.view(torch.float8_e4m3fn).double().numpy()
    got = kv8_ref.decode(every.numpy())
    assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)]) and np.isnan(got[np.isnan(want)]).all()
    x = torch.linspace(-448, 448, 100001)
    x = torch.cat([x, x / 2000]).double()      # f32 values: both sides round once
    assert np.array_equal(kv8_ref.round_e4m3(x.numpy()), x.float().to(torch.float8_e4m3fn).double().numpy())
    assert kv8_ref.page_scale(448.0) == 1 and kv8_ref.page_scale(448.0001) == 2 and kv8_ref.page_scale(0.0) == 2.0 ** -64
