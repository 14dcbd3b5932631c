"""A paged key/value cache on the GPU and the attention that reads it
(include/aero_cuda_pages.h).

`PagedCache` holds the K and V pages of every layer and the books that say which
pages hold which sequence. A serving step over a batch:

    cache.extend(seqs, counts)                      # room for the new tokens
    cache.append(layer, k, v, seqs, positions)      # their K and V rows, each layer
    out = cache.attend(layer, q, seqs)              # one new token per sequence
    out = cache.attend(layer, q, seqs, q_start)     # or several (prompts, drafts)

and between steps `fork`, `free`, `copy` and `compact`. Arrays are CUDA torch tensors,
sequence numbers, counts and positions int32. Calls run on torch's current stream
(or the one given to `set_stream`), enqueue their work and return; they do not
synchronise and can be captured in a CUDA graph. What only the device knows (lengths,
free pages) is checked there: `status()` returns the first code recorded, `check()`
raises it. A cache's calls share its books and workspace: whoever replays graphs that hold them
orders the replays, among one another and with calls, and a cache is not for two threads at once.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

from . import native_cuda as nc

STATUS = {
    1: "a sequence number outside the cache, or listed twice",
    2: "more pages asked for than are free",
    3: "a sequence would pass its row of the table, or a negative count",
    4: "a fork into a sequence that is not empty",
    5: "a page number outside the pool, or a position without a page",
    6: "q_start does not ascend from 0 to the tokens' number within the sequences' lengths",
    7: "a bounded device wait gave up",
    8: "an append into a page that several sequences hold",
}


class _Memory:
    """Device memory of the library, for torch.as_tensor (which keeps this object, and
    with it the cache, alive)."""

    def __init__(self, owner, ptr: int, shape, typestr: str) -> None:
        self._owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (ptr, False), "version": 3}


def _dtypes():
    import torch
    return {torch.float16: nc.TYPE_F16, torch.bfloat16: nc.TYPE_BF16}


def plan_bytes(n_layer: int, n_page: int, page_size: int, n_head_kv: int, head_dim: int, n_seq: int, max_pages: int,
               device: int = 0) -> dict:
    """Device bytes a cache of this shape allocates, as the memory guard charges them."""
    d = nc.PagesDesc(n_layer, n_page, page_size, n_head_kv, head_dim, n_seq, max_pages, nc.TYPE_F16, device, 0)
    by = (ctypes.c_int64 * 2)()
    if nc.lib().aero_cuda_pages_plan_bytes(ctypes.byref(d), by) < 0:
        raise ValueError("invalid cache description")
    return {"kv_cache": int(by[0]), "scratch": int(by[1]), "total": int(by[0]) + int(by[1])}


class PagedCache:
    def __init__(self, n_layer: int, n_page: int, page_size: int, n_head_kv: int, head_dim: int, n_seq: int,
                 max_pages: int, dtype=None, device: int = 0) -> None:
        """n_page pages of page_size positions in each of n_layer layers, for n_seq sequences of at
        most max_pages pages; dtype torch.float16 (default) or torch.bfloat16."""
        import torch
        self.handle = None
        self._lib = nc.lib()
        nc.require_gpu()
        dtype = torch.float16 if dtype is None else dtype
        if dtype not in _dtypes():
            raise ValueError(f"dtype must be torch.float16 or torch.bfloat16, got {dtype}")
        d = nc.PagesDesc(int(n_layer), int(n_page), int(page_size), int(n_head_kv), int(head_dim), int(n_seq),
                         int(max_pages), _dtypes()[dtype], int(device), 0)
        err = ctypes.create_string_buffer(512)
        h = self._lib.aero_cuda_pages_open(ctypes.byref(d), err, 512)
        if not h:
            raise RuntimeError(f"paged cache open: {err.value.decode()}")
        self.handle = h
        self.n_layer, self.n_page, self.page_size = int(n_layer), int(n_page), int(page_size)
        self.n_head_kv, self.head_dim, self.n_seq, self.max_pages = int(n_head_kv), int(head_dim), int(n_seq), int(max_pages)
        self.dtype, self.device = dtype, torch.device("cuda", int(device))
        self._torch = torch
        self._index = int(device)
        self._follow, self._stream = True, None
        self._current_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream builds an object each call
        self._i32_type, self._scale = torch.int32, 1.0 / math.sqrt(self.head_dim)
        p = [ctypes.c_void_p() for _ in range(5)]
        self._lib.aero_cuda_pages_buffers(h, *(ctypes.byref(x) for x in p))
        self._ptr = [x.value for x in p]

    # ---- memory
    def _view(self, ptr, shape, typestr):
        return self._torch.as_tensor(_Memory(self, ptr, shape, typestr), device=self.device)

    def _pool(self, ptr, layer):
        t = self._view(ptr, (self.n_layer, self.n_page, self.n_head_kv, self.page_size, self.head_dim), "<i2").view(self.dtype)
        return t if layer is None else t[layer]

    def k(self, layer: Optional[int] = None):
        """The K pages as a tensor over the cache's own memory: (n_layer, n_page, n_head_kv,
        page_size, head_dim), or one layer's."""
        return self._pool(self._ptr[0], layer)

    def v(self, layer: Optional[int] = None):
        return self._pool(self._ptr[1], layer)

    def tables(self):
        """(table, length, refs): the books as tensors over the cache's own memory, to be read; they
        are changed by the calls below (set_tables for books kept elsewhere)."""
        return (self._view(self._ptr[2], (self.n_seq, self.max_pages), "<i4"),
                self._view(self._ptr[3], (self.n_seq,), "<i4"), self._view(self._ptr[4], (self.n_page,), "<i4"))

    # ---- streams and errors
    def set_stream(self, stream) -> None:
        """Run on a cudaStream_t (int) or torch.cuda.Stream, whatever torch's current one is (the
        caller then orders tensors made or used on others); None: on torch's current stream
        at each call (the default)."""
        self._follow = stream is None
        if stream is not None:
            self._use(getattr(stream, "cuda_stream", stream))

    def _use(self, raw: int) -> None:
        if raw != self._stream:
            # (the legacy default stream is 0 in torch; to the library 0 is the handle's own)
            if self._lib.aero_cuda_pages_set_stream(self.handle, raw or 1) != 0:
                self._refused("set_stream")
            self._stream = raw

    def _on(self) -> None:
        if self.handle is None:
            raise RuntimeError("the cache is closed")
        if self._follow:
            raw = self._current_stream(self._index)
            if raw != self._stream:
                self._use(raw)

    def _refused(self, what: str):
        raise ValueError(f"{what} refused: {self.last_error()}")

    def last_error(self) -> str:
        r = self._lib.aero_cuda_pages_last_error(self.handle)
        return r.decode() if r else ""

    def status(self) -> int:
        """The first code recorded on the device since the last read (0: none); synchronises."""
        self._on()
        return int(self._lib.aero_cuda_pages_status(self.handle))

    def check(self) -> None:
        code = self.status()
        if code:
            raise RuntimeError(f"paged cache: {STATUS.get(code, f'status {code}')}")

    # ---- arguments
    def _i32(self, t, name: str, n: Optional[int] = None) -> int:
        if t.dtype is not self._i32_type or t.get_device() != self._index or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor on {self.device}")
        if n is not None and t.numel() != n:
            raise ValueError(f"{name} has {t.numel()} entries, expected {n}")
        return t.data_ptr()

    def _rows(self, t, name: str, heads: Optional[int]):
        """(address, token stride, head stride) of rows (tokens, heads, head_dim)."""
        if t.dtype is not self.dtype or t.get_device() != self._index:
            raise ValueError(f"{name} must be {self.dtype} on {self.device}, got {t.dtype} on {t.device}")
        shape = t.shape
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be (tokens, {heads or 'heads'}, {self.head_dim}), got {tuple(shape)}")
        token, head, one = t.stride()
        if one != 1:
            raise ValueError(f"{name} must be contiguous along head_dim")
        return t.data_ptr(), token, head

    # ---- books
    def set_tables(self, table, length, refs) -> None:
        """Adopt books kept elsewhere: table (n_seq, max_pages), length (n_seq), refs (n_page)."""
        self._on()
        if self._lib.aero_cuda_pages_set_tables(self.handle, self._i32(table, "table", self.n_seq * self.max_pages),
                                                self._i32(length, "length", self.n_seq),
                                                self._i32(refs, "refs", self.n_page)) != 0:
            self._refused("set_tables")

    def extend(self, seqs, counts) -> None:
        """Room for counts[i] more positions at the end of sequence seqs[i] (each listed once)."""
        self._on()
        n = seqs.numel()
        if self._lib.aero_cuda_pages_extend(self.handle, self._i32(seqs, "seqs"), self._i32(counts, "counts", n), n) != 0:
            self._refused("extend")

    def append(self, layer: int, k, v, seqs, positions) -> None:
        """K and V rows (T, n_head_kv, head_dim) of T tokens into a layer: token t to position
        positions[t] of sequence seqs[t], in a page that no other sequence holds."""
        self._on()
        T = k.shape[0]
        if v.shape != k.shape:
            raise ValueError(f"k and v differ in shape: {tuple(k.shape)}, {tuple(v.shape)}")
        if self._lib.aero_cuda_pages_append(self.handle, layer, *self._rows(k, "k", self.n_head_kv),
                                            *self._rows(v, "v", self.n_head_kv), self._i32(seqs, "seqs", T),
                                            self._i32(positions, "positions", T), T) != 0:
            self._refused("append")

    def fork(self, parents, children) -> None:
        """Sequence children[i] (empty) becomes a copy of parents[i]; full pages are shared."""
        self._on()
        n = parents.numel()
        if self._lib.aero_cuda_pages_fork(self.handle, self._i32(parents, "parents"),
                                          self._i32(children, "children", n), n) != 0:
            self._refused("fork")

    def free(self, seqs) -> None:
        """The sequences (each listed once) give up their pages and become empty."""
        self._on()
        if self._lib.aero_cuda_pages_free(self.handle, self._i32(seqs, "seqs"), seqs.numel()) != 0:
            self._refused("free")

    def copy(self, src, dst) -> None:
        """Pages dst[i] = src[i] in every layer."""
        self._on()
        n = src.numel()
        if self._lib.aero_cuda_pages_copy(self.handle, self._i32(src, "src"), self._i32(dst, "dst", n), n) != 0:
            self._refused("copy")

    def compact(self) -> None:
        """Moves the live pages to the pool's front (their order there: see the header)."""
        self._on()
        if self._lib.aero_cuda_pages_compact(self.handle) != 0:
            self._refused("compact")

    # ---- attention
    def attend(self, layer: int, q, seqs, q_start=None, *, window: int = 0, sinks: int = 0,
               scale: Optional[float] = None, out=None):
        """Attention of new tokens q (T, n_head, head_dim) over a layer's pages, causal; with a
        window a token sees the last `window` positions (its own among them) and the first
        `sinks`. q_start None: one token for each of seqs, its last position; else tokens
        [q_start[i], q_start[i + 1]) are the last positions of seqs[i]. scale: 1 /
        sqrt(head_dim) by default. Returns out (T, n_head, head_dim)."""
        self._on()
        qp, q_token, q_head = self._rows(q, "q", None)
        T, H, _ = q.shape
        if out is None:
            if q.is_contiguous():
                out, o_token, o_head = self._torch.empty_like(q), q_token, q_head
            else:
                out, o_token, o_head = q.new_empty(q.shape), H * self.head_dim, self.head_dim
            op = out.data_ptr()
        else:
            if out.shape != q.shape:
                raise ValueError(f"out has shape {tuple(out.shape)}, expected {tuple(q.shape)}")
            op, o_token, o_head = self._rows(out, "out", H)
        n = seqs.numel()
        if self._lib.aero_cuda_pages_attend(
                self.handle, layer, qp, q_token, q_head, T, H, self._i32(seqs, "seqs"),
                None if q_start is None else self._i32(q_start, "q_start", n + 1), n,
                self._scale if scale is None else scale, window, sinks, op, o_token, o_head) != 0:
            self._refused("attend")
        return out

    # ---- end
    def close(self) -> None:
        """Frees the cache's memory (tensors over it must not be used any more)."""
        h, self.handle = self.handle, None
        if h:
            self._lib.aero_cuda_pages_close(h)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
