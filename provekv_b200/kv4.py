"""A KV cache that stays in 4 bits while a model decodes from it.

The codecs of this package store a cache and give it back in f32 or 16 bits; between the two, a server that keeps many
contexts resident wants the cache small while it is read at every step.  `Kv4Cache` is one layer's keys and values
in pages of 4-bit codes (4.5 bits a value with the scales): `append` writes a step's vectors (or vectors the
codecs decoded), `attend` is attention straight from the pages (shared kv heads, one query token or many, a sliding
window with sinks), `evict` cuts a cache down to a budget by the attention weight its tokens received, and `read` gives
values back.  The format and the exact meaning of each call are in include/provekv_b200.h (``pkv_kv4_*``).

The lengths belong to the step, not to the layer: raise ``lens`` and ``ends`` once, then call the layers::

    lens += 1                                   # int32 [n_seqs], on the device, shared by all layers
    ends += 1                                   # (caches made without ends have as many tokens as they hold)
    for layer, cache in enumerate(caches):
        cache.append(k, v)                      # [n_seqs, 1, n_kv_heads, dim]
        out, lse = cache.attend(q)              # [n_seqs, 1, n_q_heads, dim]

Calls only enqueue work on the current torch stream of the cache's device and allocate through torch, so they can be captured into a
CUDA graph.  What a kernel finds wrong (a page number out of range, a value that is not finite) goes to the
cache's error word: `check` reads it.
"""
from __future__ import annotations

import ctypes as C
from operator import index

from . import _lib as L
from .patch import dst_dtype_of

__all__ = ["Kv4Cache", "atom_bytes", "ATOM_TOKENS"]

ATOM_TOKENS = 16


def atom_bytes(dim: int) -> int:
    """Bytes of 16 tokens of one kv head, keys and values."""
    return 18 * dim


def _int32(name: str, x: int) -> int:
    """A count as the library takes it (ctypes would cut off what is above 32 bits), as a plain number: what is kept by it
    must not change when the caller's object does."""
    x = index(x)
    if not 0 <= x < 1 << 31:
        raise ValueError(f"{name} must be at least 0 and below 2**31, not {x}")
    return x


def _raw_queries(torch):
    """(current device, current stream of a device) as plain numbers: torch's own accessors without the Python objects around
    them where this torch has them (a decode step's call is a few microseconds long)."""
    device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    return device, stream


class Kv4Cache:
    """One layer's cache over tensors the caller owns.

    pages       uint8 [n_pages][n_kv_heads][page_tokens / 16][18 * dim], contiguous
    page_table  int32 [n_seqs][max_pages]: the pages of each sequence
    lens        int32 [n_seqs]: slots in use, a step's new tokens included
    ends        int32 [n_seqs]: tokens the sequence has had (None: as many as it holds)
    positions   int32 [n_seqs][n_kv_heads][max_pages * page_tokens]: position of the token in a slot (None: the slot's number)
    mass        f32, the same shape: attention weight received

    They are attributes under these names; one that is assigned another tensor of the same kind uses it from the next call on.
    """
    pages, page_table, lens, ends, positions, mass = (
        property(lambda self, name=name: getattr(self, "_" + name), lambda self, t, name=name: self._rebind(name, t))
        for name in ("pages", "page_table", "lens", "ends", "positions", "mass"))
    error = property(lambda self: self._error, doc="The error word that the kernels report to (see `check`).")

    def __init__(self, pages, page_table, lens, *, ends=None, positions=None, mass=None):
        import torch
        if pages.dim() != 4 or pages.dtype != torch.uint8:
            raise ValueError("pages must be uint8 [n_pages][n_kv_heads][page_tokens / 16][18 * dim]")
        _, self.n_kv_heads, atoms, width = pages.shape
        self.dim, self.page_tokens, self.device = width // 18, atoms * ATOM_TOKENS, pages.device
        if width not in (atom_bytes(64), atom_bytes(128)):
            raise ValueError(f"an atom has 18 * 64 or 18 * 128 bytes, not {width}")
        if page_table.dim() != 2:
            raise ValueError("page_table must be [n_seqs][max_pages]")
        self.n_seqs, max_pages = page_table.shape
        self.capacity = max_pages * self.page_tokens
        stats = (self.n_seqs, self.n_kv_heads, self.capacity)
        self._like = {"pages": (torch.uint8, pages.shape[1:]), "page_table": (torch.int32, page_table.shape),
                      "lens": (torch.int32, (self.n_seqs,)), "ends": (torch.int32, (self.n_seqs,)),
                      "positions": (torch.int32, stats), "mass": (torch.float32, stats)}
        tensors = dict(pages=pages, page_table=page_table, lens=lens, ends=ends, positions=positions, mass=mass)
        for name, t in tensors.items():
            self._check_tensor(name, t)
        if self.device.type != "cuda":
            raise ValueError("a Kv4Cache lives on a CUDA device")
        self._c = L.Kv4CacheC(dim=self.dim, n_kv_heads=self.n_kv_heads, page_tokens=self.page_tokens, n_seqs=self.n_seqs,
                              max_pages=max_pages)
        self._rows_of, self._attend_of, self._evict_of = {}, {}, {}
        for name, t in tensors.items():
            self._bind(name, t)
        self._error = torch.full((1,), -1, dtype=torch.int64, device=self.device)
        # what a call needs besides its tensors' addresses, prepared once: a decode step makes few microseconds' calls
        self._ref, self._err, self._index = C.byref(self._c), self._error.data_ptr(), self.device.index
        self._lib, self._torch = L.lib(), torch
        self._current_device, self._current_stream = _raw_queries(torch)

    def _check_tensor(self, name: str, t) -> None:
        dtype, shape = self._like[name]
        if t is None:
            if name in ("pages", "page_table", "lens"):
                raise ValueError(f"{name} must be a tensor")
            return
        if t.dtype != dtype or tuple(t.shape[1:] if name == "pages" else t.shape) != tuple(shape):
            raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)}, not {t.dtype} of {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the pages on {self.device}")

    def _bind(self, name: str, t) -> None:
        """Makes a checked tensor the one that later calls use."""
        setattr(self, "_" + name, t)
        setattr(self._c, name, None if t is None else t.data_ptr())
        if name == "pages":
            self._c.n_pages = t.shape[0]
        self._attend_of.clear()  # workspaces go by which statistics there are
        self._evict_of.clear()

    def _rebind(self, name: str, t) -> None:
        if t is not getattr(self, "_" + name):  # (`cache.lens += 1` assigns the tensor that it changed)
            self._check_tensor(name, t)
            self._bind(name, t)

    @classmethod
    def allocate(cls, n_layers: int, n_seqs: int, n_kv_heads: int, dim: int, max_tokens: int, *, page_tokens: int = 64,
                 evictable: bool = False, device="cuda") -> list["Kv4Cache"]:
        """Empty caches for `n_layers` layers that share page table, `lens` and `ends`; each sequence owns the pages of
        `max_tokens` tokens.  `evictable`: with positions and mass."""
        import torch
        if page_tokens < 1 or page_tokens % ATOM_TOKENS:
            raise ValueError(f"page_tokens must be a multiple of {ATOM_TOKENS}, not {page_tokens}")
        max_pages = -(-max_tokens // page_tokens)
        table = torch.arange(n_seqs * max_pages, dtype=torch.int32, device=device).view(n_seqs, max_pages)
        lens, ends = (torch.zeros(n_seqs, dtype=torch.int32, device=device) for _ in range(2))
        out = []
        for _ in range(n_layers):
            pages = torch.zeros((n_seqs * max_pages, n_kv_heads, page_tokens // ATOM_TOKENS, atom_bytes(dim)), dtype=torch.uint8,
                                device=device)
            stats = (n_seqs, n_kv_heads, max_pages * page_tokens)
            out.append(cls(pages, table, lens, ends=ends,
                           positions=torch.zeros(stats, dtype=torch.int32, device=device) if evictable else None,
                           mass=torch.zeros(stats, dtype=torch.float32, device=device) if evictable else None))
        return out

    # -- calls -----------------------------------------------------------------------------------------------------------
    def _rows(self, t, name: str, heads: int | None = None, written: bool = False):
        """A reference to the pkv_kv4_rows of a tensor's shape, strides and type (kept: they depend on nothing else)."""
        key = (t.shape, t.stride(), t.dtype, written)
        r = self._rows_of.get(key)
        if r is None:
            shape, stride = t.shape, t.stride()
            if len(shape) != 4 or shape[0] != self.n_seqs or shape[3] != self.dim:
                raise ValueError(f"{name} must be [{self.n_seqs}][tokens][heads][{self.dim}], not {tuple(shape)}")
            if stride[3] != 1 and t.numel():
                raise ValueError(f"the values of a vector of {name} must be contiguous")
            steps = [st for n, st in zip(shape[:3], stride) if n > 1]
            if written and (any(st < self.dim for st in steps) or len(set(steps)) < len(steps)):
                raise ValueError(f"{name} is written: its vectors must not lie over one another")
            if len(self._rows_of) >= 256:
                self._rows_of.clear()
            # (the stride of a dimension of one says nothing)
            r = self._rows_of[key] = C.byref(L.Kv4RowsC(*(stride[i] if shape[i] > 1 else 0 for i in range(3)), _int32(f"the tokens of {name}", shape[1]),
                                                       dst_dtype_of(t)))
        if heads is not None and t.shape[2] != heads:
            raise ValueError(f"{name} has {t.shape[2]} heads, the cache {heads}")
        if t.get_device() != self._index:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        return r

    def _per_seq(self, t, name: str):
        if t is None:
            return None
        if t.dtype != self._torch.int32 or tuple(t.shape) != (self.n_seqs,) or not t.is_contiguous() or t.get_device() != self._index:
            raise ValueError(f"{name} must be a contiguous int32 [{self.n_seqs}] tensor on {self.device}")
        return t.data_ptr()

    def _on_device(self, fn, *args):
        """fn(*args) with the cache's device current (plans go by its size)."""
        if self._current_device() == self._index:
            return fn(*args)
        with self._torch.cuda.device(self._index):
            return fn(*args)

    def _call(self, fn, *args) -> int:
        """The status of fn(cache, *args, error word, stream) with the cache's device current."""
        if self._current_device() == self._index:
            return fn(self._ref, *args, self._err, self._current_stream(self._index))
        with self._torch.cuda.device(self._index):
            return fn(self._ref, *args, self._err, self._current_stream(self._index))

    def append(self, k, v, new_lens=None) -> None:
        """Writes the newest tokens of each sequence: row i of ``k`` and ``v`` [n_seqs][n][n_kv_heads][dim] goes to slot
        lens - n + i (with ``new_lens`` int32 [n_seqs]: the first new_lens[s] rows to lens - new_lens + i)."""
        kr, vr = self._rows(k, "k", self.n_kv_heads), self._rows(v, "v", self.n_kv_heads)
        if k.shape != v.shape:
            raise ValueError("k and v must have the same shape")
        if k.numel() == 0:
            return
        status = self._call(self._lib.pkv_kv4_append_dev, k.data_ptr(), kr, v.data_ptr(), vr, self._per_seq(new_lens, "new_lens"))
        if status:
            L.check(status)

    def read(self, n: int, dtype=None, new_lens=None, out=None):
        """(k, v) [n_seqs][n][n_kv_heads][dim]: the values the newest tokens stand for, at the rows `append` would take
        them from.  Rows from new_lens[s] on are zeros, or as they were in ``out`` = (k, v)."""
        torch = self._torch
        fresh = out is None
        if fresh:
            shape, dtype = (self.n_seqs, n, self.n_kv_heads, self.dim), dtype or torch.float32
            k = self._pages.new_empty(shape, dtype=dtype)
            v = torch.empty_like(k)
        else:
            k, v = out
            if k.shape[1] != n or (dtype is not None and k.dtype != dtype):
                raise ValueError("out does not have the rows or the type asked for")
            if k.shape != v.shape:
                raise ValueError("k and v must have the same shape")
        kr = self._rows(k, "k", self.n_kv_heads, True)
        vr = kr if fresh else self._rows(v, "v", self.n_kv_heads, True)
        if k.numel():
            status = self._call(self._lib.pkv_kv4_read_dev, k.data_ptr(), kr, v.data_ptr(), vr, self._per_seq(new_lens, "new_lens"), int(fresh))
            if status:
                L.check(status)
        return k, v

    def attend(self, q, *, scale: float | None = None, window: int = 0, sinks: int = 0, q_lens=None, accumulate: bool = False,
               max_len: int = 0, out=None, lse=None):
        """(out, lse): attention of the newest tokens' queries ``q`` [n_seqs][n][n_q_heads][dim] over what their
        sequences hold, each up to its own position.  Not differentiable.

        scale       of the products; None: dim ** -0.5
        window      > 0: only the `window` newest positions, and those below `sinks`
        q_lens      int32 [n_seqs]: the first q_lens[s] rows are sequence s's newest tokens, the others padding (zeros in a new
                    ``out``, untouched in a given one; the same for ``lse``)
        accumulate  adds the weights of these queries to ``mass``
        max_len     a bound on the lengths that the host knows (sizes the split of the work; any value is correct)
        out         where to write, of q's shape and type; may be q, or lie over it
        lse         f32 [n_seqs][n][n_q_heads], natural logarithm; -inf where a query sees nothing (its out is zeros)
        """
        torch = self._torch
        if q.requires_grad and torch.is_grad_enabled():
            raise ValueError("attend has no gradient: detach q, or call it under torch.no_grad()")
        qr = self._rows(q, "q")
        shape = q.shape
        if out is None:
            out = (torch.empty_like if q_lens is None else torch.zeros_like)(q, memory_format=torch.contiguous_format)
        elif out.shape != shape or out.dtype != q.dtype:
            raise ValueError("out must have the shape and type of q")
        outr = self._rows(out, "out", written=True)
        if lse is None:
            lse = (q.new_empty if q_lens is None else q.new_zeros)(shape[:3], dtype=torch.float32)
        elif lse.shape != shape[:3] or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.get_device() != self._index:
            raise ValueError("lse must be contiguous f32 [n_seqs][tokens][heads] on the cache's device")
        if scale is not None and type(scale) is not float:
            scale = float(scale)
        if not type(window) is type(sinks) is type(max_len) is int:
            window, sinks, max_len = _int32("window", window), _int32("sinks", sinks), _int32("max_len", max_len)
        accumulate = bool(accumulate)
        key = (shape, q.dtype, scale, window, sinks, accumulate, max_len)
        plan = self._attend_of.get(key)
        if plan is None:
            if accumulate and self._mass is None:
                raise ValueError("accumulate needs a cache with mass")
            args = L.Kv4AttendC(self.dim ** -0.5 if scale is None else scale, shape[2], _int32("window", window), _int32("sinks", sinks),
                                int(accumulate), _int32("max_len", max_len))
            if len(self._attend_of) >= 256:
                self._attend_of.clear()
            plan = self._attend_of[key] = (C.byref(args), self._on_device(self._lib.pkv_kv4_attend_workspace_bytes, self._ref, qr, C.byref(args)),
                                           q.numel() == 0)
        args, need, empty = plan
        if empty:
            return out, lse
        work = self._pages.new_empty(need) if need else None
        to = (out.data_ptr(), outr, lse.data_ptr(), self._per_seq(q_lens, "q_lens"), args, work.data_ptr() if need else None, need)
        status = self._call(self._lib.pkv_kv4_attend_dev, q.data_ptr(), qr, *to)
        if status:
            if status == L.ERR_INVALID_ARGUMENT and out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr():
                q = q.clone()  # out lies over queries that are still to be read
                status = self._call(self._lib.pkv_kv4_attend_dev, q.data_ptr(), self._rows(q, "q"), *to)
            L.check(status)
        return out, lse

    def evict(self, budget: int, *, sinks: int = 0, recent: int = 0) -> None:
        """Cuts every sequence longer than `budget` down to it, per kv head: positions below `sinks`, the `recent` newest
        positions, and the heaviest of the others stay (ties: the lowest slot).  Then ``lens.clamp_(max=budget)``, once
        all layers are done."""
        if self._positions is None or self._mass is None:
            raise ValueError("evict needs a cache with positions and mass")
        budget, sinks, recent = _int32("budget", budget), _int32("sinks", sinks), _int32("recent", recent)
        if self.n_seqs == 0:
            return
        need = self._evict_of.get(budget)
        if need is None:
            if len(self._evict_of) >= 256:
                self._evict_of.clear()
            need = self._evict_of[budget] = self._lib.pkv_kv4_evict_workspace_bytes(self._ref, budget)
        work = self._pages.new_empty(need) if need else None
        status = self._call(self._lib.pkv_kv4_evict_dev, budget, sinks, recent, work.data_ptr() if need else None, need)
        if status:
            L.check(status)

    def check(self) -> None:
        """Waits for the stream, raises PkvError for the first thing a kernel reported since the last check, and clears it."""
        code, index = C.c_int32(0), C.c_int64(-1)
        with self._torch.cuda.device(self._index):
            s = self._current_stream(self._index)
            st = self._lib.pkv_error_word_read(self._err, s, C.byref(code), C.byref(index))
            if st != L.OK:
                L.check(self._lib.pkv_error_word_reset(self._err, s))
                raise L.PkvError(st, L.status_string(st), index.value)
