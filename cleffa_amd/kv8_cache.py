"""The 8-bit paged prefix cache on torch device memory: pools, page tables and the pass plan.

``Kv8Cache`` holds, per attention layer, K and V as e4m3 codes in pages of 64 tokens with a power-of-two scale
for each page and kv head, and for all layers the page tables, the stack of free pages and the sequences'
lengths. ``Kv8Plan.update`` plans a pass on the device from the new tokens of each sequence;
``TextAttention.forward_kv8`` appends a layer's keys and values and attends; ``Kv8Cache.read`` brings
pages back into the 16-bit planes that ``TextAttention.forward`` takes. Layouts: include/clef_hip_attn.h.

A serving loop needs no host round trip between its passes:

    cache = Kv8Cache(n_layers, nkv, n_pages, max_seqs, max_pages)
    plan = Kv8Plan(cache, T, nh, max_new=1)
    while ...:
        plan.update(new_lens)                       # state, tables, slots, positions: all on the device
        for l in range(n_layers):
            out = att.forward_kv8(qkv[l], q_norm, k_norm, plan.pos3, plan, cache, l)
"""
import ctypes

import torch

from . import _lib
from .attention import _check, _device, _err, _on, _ptr, init_device

_STATUS = {1: "too few free pages", 2: "more new tokens than the pass has rows", 4: "a sequence would pass its table row",
           8: "lengths, counts or page numbers that cannot be"}


class Kv8Cache:
    """K and V pages of ``n_layers`` layers: ``k[l]`` uint8 [n_pages][nkv][4][64][64] (dim group, token, dim), ``v[l]``
    uint8 [n_pages][nkv][256][64] (dim, token), ``k_scale[l]``, ``v_scale[l]`` float32 [n_pages][nkv]; ``tables``
    int32 [max_seqs][max_pages], ``free`` int32 [n_pages], ``state`` int32 [2 + 2 max_seqs]: {free pages, status of
    the last plan, tokens and pages of each sequence}. allocate=False leaves the layers' lists empty (None),
    for pools that the caller sets."""

    def __init__(self, n_layers, nkv, n_pages, max_seqs, max_pages, hd=256, device="cuda", allocate=True):
        if hd != 256:
            raise ValueError(f"the 8-bit cache supports hd 256 only (got {hd})")
        if n_layers <= 0 or nkv <= 0 or n_pages <= 0 or not 0 < max_seqs <= _lib.KV8_MAX_SEQ or not 0 < max_pages <= 65536:
            raise ValueError(f"bad cache sizes: {n_layers} layers, {nkv} kv heads, {n_pages} pages, {max_seqs} sequences "
                             f"(at most {_lib.KV8_MAX_SEQ}) of {max_pages} pages (at most 65536)")
        self.n_layers, self.nkv, self.n_pages, self.max_seqs, self.max_pages, self.hd = n_layers, nkv, n_pages, max_seqs, max_pages, hd
        self.device = _device(device)
        self.k, self.v, self.k_scale, self.v_scale = ([None] * n_layers for _ in range(4))
        if allocate:
            for l in range(n_layers):
                self.k[l] = torch.empty(self.page_shape("k"), dtype=torch.uint8, device=self.device)
                self.v[l] = torch.empty(self.page_shape("v"), dtype=torch.uint8, device=self.device)
                self.k_scale[l] = torch.ones((n_pages, nkv), dtype=torch.float32, device=self.device)
                self.v_scale[l] = torch.ones((n_pages, nkv), dtype=torch.float32, device=self.device)
        self.tables = torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=self.device)
        # page 0 on top of the stack
        self.free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=self.device)
        self.state = torch.zeros(2 + 2 * max_seqs, dtype=torch.int32, device=self.device)
        self.state[0] = n_pages

    def page_shape(self, which):
        return (self.n_pages, self.nkv, 4, _lib.KV8_PAGE, 64) if which == "k" else (self.n_pages, self.nkv, self.hd, _lib.KV8_PAGE)

    def nbytes(self):
        """Bytes of all layers' pages and scales."""
        return self.n_layers * self.n_pages * self.nkv * 2 * (_lib.KV8_PAGE * self.hd + 4)

    def check_layer(self, layer):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        dev = self.device
        _check(self.k[layer], "k pages", self.page_shape("k"), torch.uint8, dev)
        _check(self.v[layer], "v pages", self.page_shape("v"), torch.uint8, dev)
        _check(self.k_scale[layer], "k_scale", (self.n_pages, self.nkv), torch.float32, dev)
        _check(self.v_scale[layer], "v_scale", (self.n_pages, self.nkv), torch.float32, dev)
        _check(self.tables, "tables", (self.max_seqs, self.max_pages), torch.int32, dev)

    def read(self, layer, cu, k_plane, vt_plane, first_page=None, stream=None):
        """Brings pages back into 16-bit planes (k_plane [nkv][kvT][256] f16, vt_plane [nkv][256][kvT] bf16): of
        sequence r the tokens from page first_page[r] (0 if None) on, into plane rows cu[r] .. cu[r + 1]
        (device int32 [max_seqs + 1], multiples of 8). Other rows are left as they are."""
        self.check_layer(layer)
        dev, kvT = self.device, k_plane.shape[1] if k_plane.dim() == 3 else -1
        _check(self.state, "state", (2 + 2 * self.max_seqs,), torch.int32, dev)
        _check(cu, "cu", (self.max_seqs + 1,), torch.int32, dev)
        if first_page is not None:
            _check(first_page, "first_page", (self.max_seqs,), torch.int32, dev)
        _check(k_plane, "k_plane", (self.nkv, kvT, self.hd), torch.float16, dev)
        _check(vt_plane, "vt_plane", (self.nkv, self.hd, kvT), torch.bfloat16, dev)
        a = _lib.Kv8ReadArgs()
        a.nkv, a.hd, a.n_seq, a.max_pages, a.n_pages, a.kvT = self.nkv, self.hd, self.max_seqs, self.max_pages, self.n_pages, kvT
        a.k_pages, a.v_pages, a.k_scale, a.v_scale = (_ptr(t[layer]) for t in (self.k, self.v, self.k_scale, self.v_scale))
        a.tables, a.state, a.first_page, a.cu = _ptr(self.tables), _ptr(self.state), _ptr(first_page), _ptr(cu)
        a.k_plane, a.vt_plane = _ptr(k_plane), _ptr(vt_plane)
        err = _err()
        with _on(dev, stream) as s:
            _lib.check(_lib.load().clef_hip_kv8_read(ctypes.byref(a), s, err, len(err)), err)
        return k_plane, vt_plane


class Kv8Plan:
    """Device buffers of passes of up to ``T`` rows and nh q heads over a cache: ``cu_q`` [max_seqs + 1], ``slots`` [T]
    (page * 64 + token in page of each pass row), ``pos3`` [T][3], the kernels' work lists and the attention's
    workspace. max_new: the most new tokens of a sequence (None: not known); it selects the attention's form.
    Passes that overlap in time need a plan each."""

    def __init__(self, cache, T, nh, max_new=None):
        if nh <= 0 or nh % cache.nkv:
            raise ValueError(f"{nh} q heads over {cache.nkv} kv heads")
        if T < 0 or (max_new is not None and max_new < 0):
            raise ValueError(f"T {T}, max_new {max_new}")
        lib = _lib.load()
        self.cache, self.T, self.nh, self.max_new = cache, int(T), int(nh), int(max_new or 0)
        ints, ws, err = ctypes.c_size_t(0), ctypes.c_size_t(0), _err()
        _lib.check(lib.clef_hip_kv8_sizes(cache.max_seqs, self.T, self.nh, cache.nkv, self.max_new, ctypes.byref(ints),
                                          ctypes.byref(ws), err, len(err)), err)
        dev = self.device = cache.device
        if dev.type == "cuda":
            init_device(dev)
        self.cu_q = torch.zeros(cache.max_seqs + 1, dtype=torch.int32, device=dev)
        self.slots = torch.full((max(self.T, 1),), -1, dtype=torch.int32, device=dev)[:self.T]
        self.pos3 = torch.zeros((max(self.T, 1), 3), dtype=torch.int32, device=dev)[:self.T]
        self.work = torch.zeros(ints.value, dtype=torch.int32, device=dev)
        self.workspace = torch.empty(ws.value, dtype=torch.uint8, device=dev)
        self.state = None   # the state that the last update wrote

    def update(self, new_lens, pos_off=None, state_out=None, stream=None):
        """Plans a pass: new_lens int32 [max_seqs] on the device (0: the sequence rests, negative: it has ended and
        gives its pages back). Without state_out the cache's state moves on in place; with it, the state after
        the pass goes there and the cache's own stays (tables and free pages change in place either way).
        pos_off int32 [max_seqs]: added to the token indexes for pos3. Does not wait: see status()."""
        c, dev = self.cache, self.device
        _check(new_lens, "new_lens", (c.max_seqs,), torch.int32, dev)
        if pos_off is not None:
            _check(pos_off, "pos_off", (c.max_seqs,), torch.int32, dev)
        out = c.state if state_out is None else state_out
        _check(c.state, "state", (2 + 2 * c.max_seqs,), torch.int32, dev)
        _check(out, "state_out", (2 + 2 * c.max_seqs,), torch.int32, dev)
        _check(c.tables, "tables", (c.max_seqs, c.max_pages), torch.int32, dev)
        _check(c.free, "free", (c.n_pages,), torch.int32, dev)
        a = _lib.Kv8PlanArgs()
        a.n_seq, a.max_pages, a.n_pages, a.T, a.nh, a.nkv, a.max_new = c.max_seqs, c.max_pages, c.n_pages, self.T, self.nh, c.nkv, self.max_new
        a.tables, a.free_pages, a.state, a.state_out = _ptr(c.tables), _ptr(c.free), _ptr(c.state), _ptr(out)
        a.new_lens, a.pos_off = _ptr(new_lens), _ptr(pos_off)
        a.cu_q, a.slots, a.pos3 = _ptr(self.cu_q), _ptr(self.slots), _ptr(self.pos3)
        a.plan, a.plan_ints = _ptr(self.work), self.work.numel()
        err = _err()
        with _on(dev, stream) as s:
            _lib.check(_lib.load().clef_hip_kv8_plan(ctypes.byref(a), s, err, len(err)), err)
        self.state = out
        return self

    def status(self):
        """0, or what kept the last update from planning (waits for it). A pass that could not be planned changes
        nothing: append and attention with it write nothing."""
        return 0 if self.state is None else int(self.state[1])

    def check(self):
        """Raises if the last update could not plan its pass."""
        s = self.status()
        if s:
            raise RuntimeError("hip: the pass could not be planned: " + ", ".join(t for b, t in _STATUS.items() if s & b))
