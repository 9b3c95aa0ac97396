"""The paged context cache: keys and values of the tokens that the expert's context comes from (prompts, camera frames,
answered tokens), for many requests at once, beside the register memory (``ring``) and the source caches (``prepare``).
The reference leaves this part to REKI's prefill.

``PagePool`` keeps which pages a request slot owns; ``pool.append(add, done)`` makes a step's block table and slots on the
GPU (``mkx_page_map``). ``AxesRotary`` turns q and k by positions of several axes (time, height, width), norms them where
the model has q / k norms, and stores k and v in their pages (``mkx_rope_axes``). ``page_attend`` is the attention of the
step's tokens over the cache, causal or not, with a sliding window and first tokens that stay visible
(``mkx_page_attend``). ``PagedCache`` holds the pages of every layer with their pool:

    cache = PagedCache(layers, n_kv_heads, head_dim, n_pages, slots=..., table_cols=..., max_tokens=...)
    m = cache.append(add, done)                        # one launch a step
    for l in range(layers):
        q = cache.store(l, rope, q, k, v, pos, m)      # rotary and store, one launch
        o = cache.attend(l, q, m, max_q=..., window=..., sinks=...)

All calls run on the current stream of their tensors' GPU and can be captured in a HIP graph. None has a backward pass: inputs
that require grad are refused, unless gradients are off. Nothing here runs without libmkx.so.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._lib import (BF16, EINVAL, FP16, MAX_SLOTS, OK, MkxAttendArgs, MkxPageMapArgs, MkxRopeArgs, ROPE_NORM32, ROPE_POS64, check,
                   lib, packer, require_device)

PAGE_ROWS = (16, 32, 64, 128, 256)
_DTYPES = {torch.bfloat16: BF16, torch.float16: FP16}
_rope_args, _attend_args = packer(MkxRopeArgs), packer(MkxAttendArgs)


# the current stream's pointer without a Stream object around it, which takes 1.8 us a call: as long as some launches run;
# the current device without the checks of an initialisation that the tensors' being there has shown
_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice


def _launch(fn, args, device: torch.device, where: str) -> None:
    """On the tensors' GPU and that GPU's current stream, whatever the current device is."""
    index = device.index
    if _device() == index:
        rc = fn(args, _stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(args, _stream(index))
    if rc != OK:
        check(rc, where)


def _require(device: torch.device, **tensors) -> None:
    """Tensors of the operators' GPU, and without gradients to make: none has a backward pass, and a result without a graph would
    pass for a constant."""
    require_device(device, **tensors)
    for name, t in tensors.items():
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires grad, and this has no backward pass: call it under torch.no_grad(), or detach {name}")


def _gpu(device) -> torch.device:
    dev = torch.device(device)
    if dev.type != "cuda":
        raise ValueError(f"the paged cache sits on a GPU, not on {dev}")
    return dev if dev.index is not None else torch.device("cuda", torch.cuda.current_device())


def _ints(t: torch.Tensor, shape: tuple, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape}")
    return t


def _heads(t: torch.Tensor, name: str, hd: int, dtype: torch.dtype | None = None) -> tuple:
    """t [T, N, hd] of a 16-bit type, its sizes, strides and address: each asked for once, as the checks of a small call take
    longer than its launch. A view that the kernels cannot read in 16-byte pieces is copied."""
    shape, dt = t.shape, t.dtype
    if len(shape) != 3 or shape[2] != hd or (dt not in _DTYPES if dtype is None else dt != dtype):
        raise ValueError(f"{name} must be [T, heads, {hd}] {dtype or 'bf16 or fp16'}, got {tuple(shape)} {dt}")
    st, sh, sd = t.stride()
    ptr = t.data_ptr()
    if sd != 1 or (st | sh) & 7 or ptr & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        st, sh, sd = t.stride()
        ptr = t.data_ptr()
    return t, shape, st, sh, ptr


def _result(out: torch.Tensor | None, like: torch.Tensor, shape: torch.Size, name: str, of: str) -> tuple:
    """Where a result goes, its strides and address."""
    if out is None:
        out = torch.empty_like(like, memory_format=torch.contiguous_format)
        n = shape[2]
        return out, shape[1] * n, n, out.data_ptr()
    t, got, st, sh, ptr = _heads(out, name, shape[2], like.dtype)
    if got != shape or t is not out:
        raise ValueError(f"{name} must be like {of}, with heads contiguous and 16-byte aligned")
    return out, st, sh, ptr


def _pages(k: torch.Tensor, v: torch.Tensor, dtype: torch.dtype) -> tuple:
    """The addresses and strides of both, and their shape."""
    shape, strides = k.shape, k.stride()
    if len(shape) != 4 or k.dtype != dtype or v.dtype != dtype or v.shape != shape or v.stride() != strides:
        bad = "k_pages" if len(shape) != 4 or k.dtype != dtype else "v_pages"
        raise ValueError(f"{bad}: k_pages and v_pages must be [n_pages, page_rows, heads, head_dim] {dtype}, alike in shape and strides, got "
                         f"{tuple(shape)} {strides} {k.dtype} and {tuple(v.shape)} {v.stride()} {v.dtype}")
    sp, sr, sh, sd = strides
    kp, vp = k.data_ptr(), v.data_ptr()
    if sd != 1 or (sp | sr | sh) & 7 or (kp | vp) & 15:
        raise ValueError("pages: heads must be contiguous and 16-byte aligned")
    if shape[1] not in PAGE_ROWS:
        raise ValueError(f"pages must have 16, 32, 64, 128 or 256 rows, got {shape[1]}")
    return kp, vp, sp, sr, sh, shape


class PageMap:
    """One step's block table and slots, tensors on the GPU: ``cu`` [B + 1] first token of each slot, ``slots`` [max_tokens]
    int64 cache row of each token (-1: none), ``pos`` [max_tokens] the token's index in its request, ``granted`` [B],
    ``kv_len`` [B] lengths after the step, ``ends`` [2] head and number of the free pages after it, ``table`` and ``queue``
    (the pool's). A map's tensors are written again by the pool's second map after a commit, and by its next map without
    one. Replays of captured maps write the same sets without the pool object's knowing: its own view is right after as many
    replays of the one set as of the other."""

    __slots__ = ("cu", "slots", "pos", "granted", "kv_len", "ends", "table", "queue")


class PagePool:
    """Which pages of a paged cache belong to which request slot. ``map(add, done)`` makes the tables of a step in which slot b
    appends add[b] tokens, or has ended (done[b] != 0: its pages return); ``commit()`` makes the last map the pool's
    state; ``append`` does both. A request is granted its tokens as a whole or not at all (``PageMap.granted``): its pages
    have to fit its table row, and the pages that it and the slots before it asked for have to be free; a slot that is
    refused pages holds up the later ones that need some until it is passed with add = 0. Lengths never visit the host."""

    def __init__(self, slots: int, n_pages: int, page_rows: int, table_cols: int, max_tokens: int, device="cuda"):
        if not 1 <= slots <= MAX_SLOTS:
            raise ValueError(f"slots must be 1 .. {MAX_SLOTS}")
        if page_rows not in PAGE_ROWS:
            raise ValueError("page_rows must be 16, 32, 64, 128 or 256")
        if n_pages < 1 or table_cols < 1 or max_tokens < 1:
            raise ValueError("n_pages, table_cols and max_tokens must be positive")
        dev = self.device = _gpu(device)
        self.slots, self.n_pages, self.page_rows, self.table_cols, self.max_tokens = slots, n_pages, page_rows, table_cols, max_tokens
        i32 = dict(dtype=torch.int32, device=dev)
        self.table = torch.full((slots, table_cols), -1, **i32)
        self.queue = torch.arange(n_pages, **i32)
        self._sets = []
        for _ in range(2):
            m = PageMap()
            m.cu, m.granted, m.kv_len = torch.zeros(slots + 1, **i32), torch.zeros(slots, **i32), torch.zeros(slots, **i32)
            m.slots, m.pos = torch.full((max_tokens,), -1, dtype=torch.int64, device=dev), torch.zeros(max_tokens, **i32)
            m.ends, m.table, m.queue = torch.tensor([0, n_pages], **i32), self.table, self.queue
            self._sets.append(m)
        self._cur = 0  # the set that holds the pool's lengths; a map writes the other one
        self._args = []
        for src, dst in (self._sets, self._sets[::-1]):
            a = MkxPageMapArgs(B=slots, cols=table_cols, n_pages=n_pages, page_rows=page_rows, max_tokens=max_tokens,
                               table_stride=table_cols, table=self.table.data_ptr(), queue=self.queue.data_ptr(),
                               len_in=src.kv_len.data_ptr(), ends_in=src.ends.data_ptr(), len_out=dst.kv_len.data_ptr(),
                               ends_out=dst.ends.data_ptr(), cu=dst.cu.data_ptr(), granted=dst.granted.data_ptr(),
                               slot=dst.slots.data_ptr(), pos=dst.pos.data_ptr())
            self._args.append((a, ctypes.byref(a)))
        self._mapped = False

    @property
    def kv_len(self) -> torch.Tensor:
        """Tokens of each slot."""
        return self._sets[self._cur].kv_len

    @property
    def ends(self) -> torch.Tensor:
        """Head of the free pages in the queue, and their number."""
        return self._sets[self._cur].ends

    def map(self, add: torch.Tensor, done: torch.Tensor | None = None) -> PageMap:
        _ints(add, (self.slots,), "add")
        if done is not None:
            _ints(done, (self.slots,), "done")
        index = self.device.index
        if add.get_device() != index or (done is not None and done.get_device() != index):
            require_device(self.device, add=add, done=done)
        a, ref = self._args[self._cur]
        a.add, a.done = add.data_ptr(), None if done is None else done.data_ptr()
        _launch(lib().mkx_page_map, ref, self.device, "mkx_page_map")
        self._mapped = True
        return self._sets[1 - self._cur]

    def commit(self) -> None:
        if not self._mapped:
            raise RuntimeError("nothing to commit: map a step first")
        self._cur, self._mapped = 1 - self._cur, False

    def append(self, add: torch.Tensor, done: torch.Tensor | None = None) -> PageMap:
        m = self.map(add, done)
        self.commit()
        return m

    def state_dict(self) -> dict:
        """Copies of the pool's state: lengths, table, queue and its ends."""
        return {"len": self.kv_len.clone(), "table": self.table.clone(), "queue": self.queue.clone(), "ends": self.ends.clone()}

    def load_state_dict(self, state: dict) -> None:
        own = {"len": self.kv_len, "table": self.table, "queue": self.queue, "ends": self.ends}
        if set(state) != set(own):
            raise ValueError(f"a pool's state holds {sorted(own)}, got {sorted(state)}")
        for k, t in own.items():
            if tuple(state[k].shape) != tuple(t.shape):
                raise ValueError(f"{k} has shape {tuple(state[k].shape)}, this pool's is {tuple(t.shape)}")
        for k, t in own.items():
            t.copy_(state[k])
        self._mapped = False


class AxesRotary:
    """Rotary positions of several axes. ``axis_of_pair``: the axis that turns each of the head_dim / 2 pairs (pair i =
    elements i and i + head_dim / 2; ``sections`` makes the usual lists); the pair's frequency is theta^(-2 i / head_dim),
    or ``freqs[i]`` radians per position. ``q_norm`` / ``k_norm``: [head_dim] weights of per-head RMS norms ahead of the turn, or
    None. They are copied, and used as 1 + w: a model of plain weights passes w - 1, made in 32 bits. Weights of the
    tokens' type are read as they are, others in 32 bits."""

    def __init__(self, head_dim: int, axis_of_pair, theta: float = 10000.0, freqs=None, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, eps: float = 1e-6, device="cuda"):
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        axis = [int(a) for a in axis_of_pair]
        if len(axis) != head_dim // 2 or min(axis) < 0 or max(axis) > 15:
            raise ValueError(f"axis_of_pair needs {head_dim // 2} axes of 0 .. 15")
        dev = self.device = _gpu(device)
        self.head_dim, self.axes, self.eps = head_dim, max(axis) + 1, float(eps)
        f = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim) if freqs is None else torch.as_tensor(freqs).double().cpu()
        if tuple(f.shape) != (head_dim // 2,) or not bool(torch.isfinite(f).all()):
            raise ValueError(f"freqs needs {head_dim // 2} finite numbers")
        self._turns = (f / (2 * math.pi)).to(dev)
        self._axis = torch.tensor(axis, dtype=torch.int32, device=dev)
        self._turns_ptr, self._axis_ptr = self._turns.data_ptr(), self._axis.data_ptr()
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None and tuple(w.shape) != (head_dim,):
                raise ValueError(f"{name} must be [{head_dim}]")
        require_device(dev, q_norm=q_norm, k_norm=k_norm)
        self._norms = {}  # of each tokens' type: its flag, the weights
        given = [w.dtype for w in (q_norm, k_norm) if w is not None]
        for dt in _DTYPES:
            as_is = all(t == dt for t in given)
            self._norms[dt] = (0 if as_is else ROPE_NORM32, *(None if w is None else w.detach().to(dt if as_is else torch.float32, copy=True).contiguous()
                                                              for w in (q_norm, k_norm)))

    @staticmethod
    def sections(sizes, interleaved: bool = False) -> list:
        """axis_of_pair of ``sizes[a]`` pairs for axis a: one section after the other, or (interleaved) the axes in turn, each as
        long as it has pairs left."""
        if not interleaved:
            return [a for a, n in enumerate(sizes) for _ in range(n)]
        left, out = list(sizes), []
        while any(left):
            for a in range(len(left)):
                if left[a]:
                    out.append(a)
                    left[a] -= 1
        return out

    def _call(self, q, k, v, pos, q_out, k_out, k_pages, v_pages, slots):
        hd, dev = self.head_dim, self.device
        if q is None and k is None:
            raise ValueError("nothing to turn: q or k is needed")
        index = dev.index
        for t in (q, k, v, pos, q_out, k_out, k_pages, v_pages, slots):
            if t is not None and (t.get_device() != index or t.requires_grad):  # -1 on the host
                _require(dev, q=q, k=k, v=v, pos=pos, q_out=q_out, k_out=k_out, k_pages=k_pages, v_pages=v_pages, slots=slots)
        NQ = NK = qs = qh = ks = kh = vs = vh = os = oh = us = uh = qp = kp = vp = qo = ko = pages_k = pages_v = ps = pr = ph = n_pages = rows = sl = 0
        dt = T = None
        if q is not None:
            dt = q.dtype
            q, shape, qs, qh, qp = _heads(q, "q", hd)
            T, NQ, _ = shape
            q_out, os, oh, qo = _result(q_out, q, shape, "q_out", "q")
        if k is not None:
            k, shape, ks, kh, kp = _heads(k, "k", hd, dt)
            if T is not None and shape[0] != T:
                raise ValueError(f"k has {shape[0]} tokens, q has {T}")
            dt = k.dtype
            T, NK, _ = shape
            if slots is None:
                k_out, us, uh, ko = _result(k_out, k, shape, "k_out", "k")
            else:
                v, v_shape, vs, vh, vp = _heads(v, "v", hd, dt)
                pages_k, pages_v, ps, pr, ph, (n_pages, rows, pk, pd) = _pages(k_pages, v_pages, dt)
                if v_shape != shape or pk != NK or pd != hd:
                    raise ValueError(f"v {tuple(v_shape)} and the pages' heads {(pk, pd)} must match k {tuple(shape)}")
                n = slots.shape
                if len(n) != 1 or n[0] < T or slots.dtype != torch.int64 or (T > 1 and slots.stride(0) != 1):
                    raise ValueError(f"slots must be a contiguous int64 tensor of at least {T} entries")
                sl = slots.data_ptr()
        if pos.dim() == 1:
            pos = pos[None]
        n, pt = pos.shape, pos.dtype
        if len(n) != 2 or n[0] != self.axes or n[1] != T or pt not in (torch.int32, torch.int64):
            raise ValueError(f"pos must be [{self.axes}, {T}] int32 or int64, got {tuple(n)} {pt}")
        pa, one = pos.stride()
        if one != 1 or pa < T:
            pos = pos.contiguous()
            pa = T
        if T:
            kind, wq, wk = self._norms[dt]
            kind |= _DTYPES[dt] | (ROPE_POS64 if pt == torch.int64 else 0)
            a = _rope_args(T, NQ, NK, hd, self.axes, kind, self.eps, qp, kp, vp, qs, qh, ks, kh, vs, vh, qo, ko, os, oh, us, uh,
                           pos.data_ptr(), pa, self._axis_ptr, self._turns_ptr, 0 if wq is None else wq.data_ptr(),
                           0 if wk is None else wk.data_ptr(), sl, pages_k, pages_v, ps, pr, ph, n_pages, rows)
            _launch(lib().mkx_rope_axes, ctypes.byref(a), dev, "mkx_rope_axes")
        return q_out, k_out

    def __call__(self, q: torch.Tensor | None, k: torch.Tensor | None, pos: torch.Tensor, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None):
        """(q, k) [T, heads, head_dim] normed and turned by pos [axes, T] ([T] for one axis; int32 or int64); either may be None. ``q_out`` /
        ``k_out``: where the results go: q and k themselves, or memory that no input or other result has."""
        return self._call(q, k, None, pos, q_out, k_out, None, None, None)

    def store(self, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, k_pages: torch.Tensor,
              v_pages: torch.Tensor, slots: torch.Tensor, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """q normed and turned; k, normed and turned, and v go to their rows ``slots`` (``PageMap.slots``: page * page_rows + row;
        -1 stores nothing) of the pages [n_pages, page_rows, heads, head_dim]. Slots are distinct."""
        if k is None or v is None or slots is None:
            raise ValueError("k, v and slots are needed")
        return self._call(q, k, v, pos, q_out, None, k_pages, v_pages, slots)[0]


def page_attend(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, cu: torch.Tensor,
                kv_len: torch.Tensor, *, max_q: int | None = None, scale: float | None = None, causal: bool = True, window: int = 0,
                sinks: int = 0, out: torch.Tensor | None = None, granted: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens over the paged cache: q [T, NQ, head_dim], slot b's tokens at cu[b] .. cu[b + 1] - 1 and at the
    end of its kv_len[b] cached tokens (their own k and v stored before). causal with ``window`` > 0: a token sees the last
    ``window`` tokens up to itself and the request's first ``sinks``. ``max_q``: a bound of the chunks' lengths that the
    caller knows (1 for answered tokens); it and q's rows shape the launch only, but many more rows than the step can have
    keep the keys of a few tokens from being split. ``out``: where the result goes, not an input's memory; rows behind the
    last slot's tokens are left as they are there (and unset without it). ``granted`` (``PageMap.granted``): slots with 0 were
    refused their tokens, which are not in the cache; their rows are zeros."""
    shape = q.shape
    hd = shape[2] if len(shape) == 3 else 0
    if hd not in (64, 128):
        raise ValueError(f"q must be [T, heads, 64 or 128], got {tuple(shape)}")
    index = q.get_device()
    if index < 0:
        raise ValueError(f"q is on {q.device}: the paged cache sits on a GPU")
    for t in (q, k_pages, v_pages, table, cu, kv_len, out, granted):
        if t is not None and (t.get_device() != index or t.requires_grad):
            _require(q.device, q=q, k_pages=k_pages, v_pages=v_pages, table=table, cu=cu, kv_len=kv_len, out=out, granted=granted)
    dt = q.dtype
    q, shape, qs, qh, qp = _heads(q, "q", hd)
    T, NQ, _ = shape
    kp, vp, ps, pr, ph, (NP, P, NK, khd) = _pages(k_pages, v_pages, dt)
    if khd != hd or NK < 1 or NQ % NK:
        raise ValueError(f"the pages' heads {NK} x {khd} do not serve q's {NQ} x {hd}")
    n = kv_len.shape
    if len(n) != 1 or not 1 <= n[0] <= MAX_SLOTS:
        raise ValueError(f"kv_len must be [slots] with 1 .. {MAX_SLOTS} slots")
    B = n[0]
    _ints(kv_len, (B,), "kv_len")
    _ints(cu, (B + 1,), "cu")
    has = 0 if granted is None else _ints(granted, (B,), "granted").data_ptr()
    n, strides = table.shape, table.stride()
    if len(n) != 2 or n[0] != B or n[1] < 1 or table.dtype != torch.int32 or strides[1] != 1 or strides[0] < n[1]:
        raise ValueError(f"table must be [{B}, pages] int32 with contiguous rows, got {tuple(n)} {table.dtype}")
    cols, rows = n[1], strides[0]
    if window < 0 or sinks < 0 or (window and not causal) or (sinks and not window) or max(window, sinks) >= 1 << 31:
        raise ValueError("window needs causal, sinks need a window, and both are 0 .. 2^31 - 1")
    scale = hd ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    if max_q is None:
        max_q = T
    elif max_q < 0:
        raise ValueError("max_q must not be negative")
    out, os, oh, op = _result(out, q, shape, "out", "q")
    if T:
        a = _attend_args(T, B, NQ, NK, hd, cols, NP, P, _DTYPES[dt], 1 if causal else 0, window, sinks, min(max_q, T), scale, qp, op, qs, qh, os, oh,
                         kp, vp, ps, pr, ph, table.data_ptr(), rows, cu.data_ptr(), kv_len.data_ptr(), 0, 0)
        if _device() == index:
            _attend(a, has, index)
        else:
            with torch.cuda.device(index):
                _attend(a, has, index)
    return out


def _attend(a: MkxAttendArgs, granted: int, index: int) -> None:
    L, ref = lib(), ctypes.byref(a)
    n = L.mkx_page_attend_workspace(ref)
    if n < 0:
        check(EINVAL, "mkx_page_attend_workspace")
    ws = torch.empty(n, dtype=torch.uint8, device=index)  # of this call and its stream alone
    a.ws, a.ws_bytes = ws.data_ptr(), n
    rc = L.mkx_page_attend_granted(ref, granted, _stream(index)) if granted else L.mkx_page_attend(ref, _stream(index))
    if rc != OK:
        check(rc, "mkx_page_attend")


class PagedCache:
    """The pages of every layer and their pool: ``k[l]`` and ``v[l]`` are [n_pages, page_rows, n_kv_heads, head_dim]."""

    def __init__(self, layers: int, n_kv_heads: int, head_dim: int, n_pages: int, *, slots: int, table_cols: int, max_tokens: int,
                 page_rows: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if layers < 1 or n_kv_heads < 1 or head_dim not in (64, 128):
            raise ValueError("need layers >= 1, n_kv_heads >= 1 and a head_dim of 64 or 128")
        if dtype not in _DTYPES:
            raise ValueError("dtype must be bf16 or fp16")
        self.pool = PagePool(slots, n_pages, page_rows, table_cols, max_tokens, device)
        shape = (n_pages, page_rows, n_kv_heads, head_dim)
        self.k = [torch.empty(shape, dtype=dtype, device=self.pool.device) for _ in range(layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=self.pool.device) for _ in range(layers)]

    def append(self, add: torch.Tensor, done: torch.Tensor | None = None) -> PageMap:
        return self.pool.append(add, done)

    def store(self, layer: int, rope: AxesRotary, q, k, v, pos, m: PageMap, q_out=None):
        return rope.store(q, k, v, pos, self.k[layer], self.v[layer], m.slots, q_out=q_out)

    def attend(self, layer: int, q: torch.Tensor, m: PageMap, **how) -> torch.Tensor:
        """``page_attend`` of the step; rows of requests that it did not grant are zeros."""
        return page_attend(q, self.k[layer], self.v[layer], m.table, m.cu, m.kv_len, granted=m.granted, **how)
