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
    assert not plan.failed()                        # where the loop waits anyway: no pass was left out
"""
import ctypes

import torch

from . import _lib
from .attention import _arg, _device, _err, _launch, init_device

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
        self._k_shape, self._v_shape = (n_pages, nkv, 4, _lib.KV8_PAGE, 64), (n_pages, nkv, hd, _lib.KV8_PAGE)
        self.k, self.v, self.k_scale, self.v_scale = ([None] * n_layers for _ in range(4))
        if allocate:
            for l in range(n_layers):
                self.k[l] = torch.empty(self._k_shape, dtype=torch.uint8, device=self.device)
                self.v[l] = torch.empty(self._v_shape, dtype=torch.uint8, device=self.device)
                self.k_scale[l] = torch.ones((n_pages, nkv), dtype=torch.float32, device=self.device)
                self.v_scale[l] = torch.ones((n_pages, nkv), dtype=torch.float32, device=self.device)
        self.tables = torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=self.device)
        # page 0 on top of the stack
        self.free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=self.device)
        self.state = torch.zeros(2 + 2 * max_seqs, dtype=torch.int32, device=self.device)
        self.state[0] = n_pages

    def nbytes(self):
        """Bytes of all layers' pages and scales."""
        return self.n_layers * self.n_pages * self.nkv * 2 * (_lib.KV8_PAGE * self.hd + 4)

    def layer_args(self, layer):
        """Addresses of the tables and of a layer's pages and scales, their types and shapes checked."""
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        dev, scales = self.device, (self.n_pages, self.nkv)
        return (_arg(self.tables, "tables", (self.max_seqs, self.max_pages), torch.int32, dev),
                _arg(self.k[layer], "k pages", self._k_shape, torch.uint8, dev), _arg(self.v[layer], "v pages", self._v_shape, torch.uint8, dev),
                _arg(self.k_scale[layer], "k_scale", scales, torch.float32, dev), _arg(self.v_scale[layer], "v_scale", scales, torch.float32, dev))

    def read(self, layer, cu, k_plane, vt_plane, first_page=None, stream=None):
        """Brings pages back into 16-bit planes (k_plane [nkv][kvT][256] f16, vt_plane [nkv][256][kvT] bf16): of
        sequence r the tokens from page first_page[r] (0 if None) on, into plane rows cu[r] .. cu[r + 1]
        (device int32 [max_seqs + 1], multiples of 8). Other rows are left as they are."""
        dev, n, kvT = self.device, self.max_seqs, k_plane.shape[1] if k_plane.dim() == 3 else -1
        tables, k, v, k_scale, v_scale = self.layer_args(layer)
        a = _lib.Kv8ReadArgs(self.nkv, self.hd, n, self.max_pages, self.n_pages, kvT, k, v, k_scale, v_scale, tables,
                             _arg(self.state, "state", (2 + 2 * n,), torch.int32, dev),
                             None if first_page is None else _arg(first_page, "first_page", (n,), torch.int32, dev),
                             _arg(cu, "cu", (n + 1,), torch.int32, dev), _arg(k_plane, "k_plane", (self.nkv, kvT, self.hd), torch.float16, dev),
                             _arg(vt_plane, "vt_plane", (self.nkv, self.hd, kvT), torch.bfloat16, dev))
        _launch(_lib.load().clef_hip_kv8_read, a, dev, stream)
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
        self.workspace_bytes = ws.value
        self.state = None   # the state that the last update wrote (its word 1 is any other plan's too, see status())

    def update(self, new_lens, pos_off=None, state_out=None, stream=None):
        """Plans a pass: new_lens int32 [max_seqs] on the device (0: the sequence rests, negative: it has ended and
        gives its pages back). Without state_out the cache's state moves on in place; with it, the state after
        the pass goes there and the cache's own stays (tables and free pages change in place either way).
        pos_off int32 [max_seqs]: added to the token indexes for pos3. Does not wait: see status()."""
        c, dev, n = self.cache, self.device, self.cache.max_seqs
        out = c.state if state_out is None else state_out
        a = _lib.Kv8PlanArgs(n, c.max_pages, c.n_pages, self.T, self.nh, c.nkv, self.max_new,
                             _arg(c.tables, "tables", (n, c.max_pages), torch.int32, dev), _arg(c.free, "free", (c.n_pages,), torch.int32, dev),
                             _arg(c.state, "state", (2 + 2 * n,), torch.int32, dev), _arg(out, "state_out", (2 + 2 * n,), torch.int32, dev),
                             _arg(new_lens, "new_lens", (n,), torch.int32, dev),
                             None if pos_off is None else _arg(pos_off, "pos_off", (n,), torch.int32, dev),
                             self.cu_q.data_ptr(), self.slots.data_ptr(), self.pos3.data_ptr(), self.work.data_ptr(), self.work.numel())
        _launch(_lib.load().clef_hip_kv8_plan, a, dev, stream)
        self.state = out
        return self

    def status(self):
        """0, or what kept this plan's last update from planning (waits for it). A pass that could not be planned
        changes nothing: append and attention with it write nothing."""
        return int(self.work[_lib.KV8_PLAN_STATUS])

    def failed(self):
        """What kept any of this plan's updates since the last call of failed() from planning, or-ed (waits for
        them): status() of a loop that looks only now and then, or is replayed from a graph."""
        s = int(self.work[_lib.KV8_PLAN_FAILED])
        self.work[_lib.KV8_PLAN_FAILED] = 0
        return s

    def check(self):
        """Raises if the last update could not plan its pass."""
        s = self.status()
        if s:
            raise RuntimeError("hip: the pass could not be planned: " + ", ".join(t for b, t in _STATUS.items() if s & b))
