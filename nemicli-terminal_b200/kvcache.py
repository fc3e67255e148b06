"""The quantised key / value cache of a decoder and attention over it (kernels: csrc/qmv_kv.cu, csrc/qmv_attn.cu;
layout and contracts: include/nemicli_qmv.h, qmv_kv_cache).

* `KVCache` — a paged cache of K and V, each held as Q4_0 (4.5 bits a value) or Q8_0 (8.5 bits).
* `KVCache.write` — new tokens' K and V rotated (RoPE), quantised and written to their slots, the queries
  rotated with them, in one launch.
* `KVCache.read` — the values that slots hold.
* `KVCache.attend` — causal attention of new tokens over the cache: one token a sequence (decode), a few
  (drafted tokens), or whole prompts, with grouped heads, a sliding window and sequences of unequal lengths.
* `KVCache.summarise`, `choose`, `attend_chosen` — attention of a few tokens over the pages that matter to them: boxes around each
  page's keys, the pages whose boxes reach furthest along a query, attention over those (csrc/qmv_sparse.cu).
* `KVCache.copy` — pages copied, for beams that part (pages.py).

The reference's own cache for this step is bf16 (ggufengine/mmvq.py:139-330, rope_kv and attention1).  Everything
runs on torch's current stream and is CUDA-graph safe: lengths, page tables, slots and positions are read on the
device.  Nothing falls back to another implementation.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .formats import TYPE_ID

FORMATE = ("Q4_0", "Q8_0")                  # what K and V can be held in
DIMS = (64, 96, 128, 256)                   # values a head
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Cache(ctypes.Structure):             # qmv_kv_cache
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("n_pages", ctypes.c_int64),
                ("n_kv", ctypes.c_int), ("dim", ctypes.c_int), ("page", ctypes.c_int), ("k_type", ctypes.c_int),
                ("v_type", ctypes.c_int)]


def _bytes(fmt: str) -> int:
    return 4 if fmt == "Q4_0" else 8         # of eight values


def _rows(t: torch.Tensor, heads: int, dim: int):
    """t (rows, heads, dim) as the kernels read it (the values of a row side by side, rows any multiple of 4
    values apart, a start on four values) and the values between rows."""
    row = heads * dim
    rows_apart, heads_apart, apart = t.stride()
    if apart != 1 or heads_apart != dim and heads > 1 or t.shape[0] > 1 and (rows_apart < row or rows_apart % 4) \
            or t.data_ptr() % (4 * t.element_size()):
        t = t.contiguous()
        if t.data_ptr() % (4 * t.element_size()):
            t = t.clone()
        rows_apart = row
    return t, (rows_apart if t.shape[0] > 1 else row)


def rope_axes(sections, mixed: bool = False) -> tuple:
    """The axis of each frequency, for KVCache.write: sections[a] frequencies of axis a, one section behind the other, or `mixed`
    in turns (0, 1, 2, 0, 1, 2, ...) as long as each lasts."""
    sections = [int(n) for n in sections]
    if not sections or min(sections) < 0 or sum(sections) == 0:
        raise RuntimeError(f"rope_axes: sections {sections}")
    if not mixed:
        return tuple(a for a, n in enumerate(sections) for _ in range(n))
    return tuple(a for i in range(max(sections)) for a, n in enumerate(sections) if i < n)


class KVCache:
    """n_pages pages of `page` tokens (a power of two, 16 to 1024) for n_kv heads of `dim` values (DIMS); the slot
    of a token is page index * page + its place.  k_fmt, v_fmt: FORMATE.  buffers: existing (k, v, scales) tensors of
    the shapes below instead of new zeroed ones (shared, not copied).
        k_codes uint8 (n_pages, n_kv, page, dim * b / 8), v_codes uint8 (n_pages, n_kv, page / 2, dim * b / 4),
        scales float16 (n_pages, n_kv, page, 2, dim / 32);  b = 4 for Q4_0, 8 for Q8_0 (bytes of 8 values)
    The object keeps no state between calls but the tensors, so calls on several streams only need the order
    that their slots need."""

    def __init__(self, n_pages: int, n_kv: int, dim: int, page: int = 64, k_fmt: str = "Q4_0", v_fmt: str = "Q4_0",
                 device=None, buffers=None):
        if k_fmt not in FORMATE or v_fmt not in FORMATE:
            raise RuntimeError(f"KVCache: formats {FORMATE} (got {k_fmt}, {v_fmt})")
        if dim not in DIMS:
            raise RuntimeError(f"KVCache: heads of {DIMS} values (got {dim})")
        if page not in (16, 32, 64, 128, 256, 512, 1024) or n_pages <= 0 or not 0 < n_kv <= 65535:
            raise RuntimeError("KVCache: pages of 16 to 1024 tokens (a power of two), n_pages and n_kv positive")
        self.n_pages, self.n_kv, self.dim, self.page, self.k_fmt, self.v_fmt = n_pages, n_kv, dim, page, k_fmt, v_fmt
        shapes = ((n_pages, n_kv, page, dim * _bytes(k_fmt) // 8), (n_pages, n_kv, page // 2, dim * _bytes(v_fmt) // 4),
                  (n_pages, n_kv, page, 2, dim // 32))
        types = (torch.uint8, torch.uint8, torch.float16)
        if buffers is None:
            device = torch.device("cuda" if device is None else device)
            if not _lib.on_gpu(device):
                raise RuntimeError(f"KVCache: device {device}; the cache lives on a CUDA device")
            buffers = [torch.zeros(s, dtype=t, device=device) for s, t in zip(shapes, types)]
        for t, s, ty in zip(buffers, shapes, types):
            if t.shape != s or t.dtype != ty or not t.is_contiguous() or not _lib.on_gpu(t) or t.device != buffers[0].device:
                raise RuntimeError(f"KVCache: buffers must be contiguous CUDA tensors of shapes {shapes} and types {types}")
        self.k_codes, self.v_codes, self.scales = buffers
        self.device = self.k_codes.device
        self._where = self.k_codes.get_device()
        self._c = _Cache(self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.scales.data_ptr(), n_pages, n_kv, dim, page,
                         TYPE_ID[k_fmt], TYPE_ID[v_fmt])
        self._ref = ctypes.byref(self._c)
        self._at = ctypes.addressof(self._c)
        self._need = {}                     # workspace bytes of the calls so far, by their sizes
        self._none = None                   # stands for the workspace of calls that use none

    def _tokens(self, t: torch.Tensor, what: str, heads: Optional[int] = None, like: Optional[torch.Tensor] = None):
        shape = t.shape
        if t.get_device() != self._where:
            raise RuntimeError(f"{what}: tensor on {t.device}, the cache on {self.device}")
        if len(shape) != 3 or shape[2] != self.dim or t.dtype not in _DTYPES or heads is not None and shape[1] != heads \
                or shape[1] == 0:
            raise RuntimeError(f"{what}: (rows, {heads or 'heads'}, {self.dim}) of float32, bfloat16 or float16 expected, "
                               f"got {tuple(shape)} {t.dtype}")
        if like is not None and (t.dtype != like.dtype or shape[0] != like.shape[0]):
            raise RuntimeError(f"{what}: {like.shape[0]} rows of {like.dtype} expected")

    def _index(self, t: torch.Tensor, what: str, dtype, *shape):
        got = t.shape
        ok = t.dtype is dtype and t.get_device() == self._where and t.is_contiguous()
        if ok and got != shape:
            ok = len(got) == len(shape)
            if ok:
                for n, want in zip(got, shape):
                    if want is not None and n != want:
                        ok = False
        if not ok:
            raise RuntimeError(f"{what}: contiguous {dtype} {shape} on {self.device} expected, got {t.dtype} {tuple(got)}")

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, q: Optional[torch.Tensor] = None, rope=None,
              paired: bool = False, axes=None) -> Optional[torch.Tensor]:
        """k, v: (rows, n_kv, dim) -> quantised into slots (rows,) int64, which are distinct; a negative slot is a
        padding row.  rope = (cos, sin, positions): k is rotated first, by tables float32 (n_positions, rot / 2),
        positions (rows,) int64; value i < rot / 2 of a head pairs with i + rot / 2, with `paired` 2 i with 2 i + 1; rot
        is a multiple of 8.  q: (rows, heads, dim) of k's type -> the rotated queries (without rope a copy), else
        None.  Values beyond float16's range are clamped, NaN counts as 0.  One launch.  Slots past the cache and
        positions outside the tables leave the row unwritten (its queries 0) and set the device status.
        axes: rot / 2 numbers, the axis of each frequency (rope_axes), for tokens with a position on each of up to four axes
        (time, height and width of pictures): positions is then (axes, rows)."""
        cos, sin, positions = (None, None, None) if rope is None else rope
        if axes is not None:
            try:
                axes = bytes(tuple(axes))
            except (TypeError, ValueError):
                raise RuntimeError(f"KVCache.write: axes {axes} (numbers from 0 on)") from None
        return _lib.host().write(self._at, self._where, k, v, slots, q, cos, sin, positions, paired, axes)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        """The values at slots (rows,) int64 -> k, v (rows, n_kv, dim) of dtype; negative slots give zeros."""
        if dtype not in _DTYPES:
            raise RuntimeError(f"KVCache.read: dtype {dtype} (float32, bfloat16 or float16)")
        return _lib.host().read(self._at, self._where, slots, _DTYPES[dtype])

    def attend(self, q: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, starts: Optional[torch.Tensor] = None,
               max_new: Optional[int] = None, scale: Optional[float] = None, window: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the newest tokens over the cache.  q: (rows, heads, dim), heads a multiple of n_kv (head h
        reads key head h // (heads // n_kv)); tables int32 (sequences, width): the pages of each sequence in order;
        lens int32 (sequences,): its tokens in the cache, the new ones among them (write comes first).  One row a
        sequence, or with starts int32 (sequences + 1,) rows starts[b] .. starts[b + 1] for sequence b, its last tokens;
        max_new: at least the most new tokens of a sequence (default: all rows; it chooses between two kernels, so a
        tight bound is the faster one).  scale: default dim ** -0.5.  window: a
        query sees that many keys up to its own (0: all).  -> like q, rows side by side; in `out` (contiguous; q itself if
        that is) if given; rows that no sequence covers keep what out held (without `out` they are undefined).  Queries that
        see no key give zeros.  16-bit queries: weights (few rows: times V's scales) are held in float16,
        to 2^-11 of themselves or 2^-34 of the largest in the row, many rows' keys and values too; float32 queries: two float16
        parts, 2^-21 or 2^-35 of the largest."""
        self._tokens(q, "KVCache.attend q")
        rows, heads, _ = q.shape
        if heads % self.n_kv:
            raise RuntimeError(f"KVCache.attend: {heads} heads are not a multiple of {self.n_kv} key heads")
        self._index(tables, "KVCache.attend tables", torch.int32, None, None)
        n_seq, width = tables.shape
        self._index(lens, "KVCache.attend lens", torch.int32, n_seq)
        if starts is not None:
            self._index(starts, "KVCache.attend starts", torch.int32, n_seq + 1)
        elif rows < n_seq:
            raise RuntimeError(f"KVCache.attend: {rows} query rows for {n_seq} sequences")
        most = 1 if starts is None else (rows if max_new is None else int(max_new))
        if scale is not None and not abs(scale) < 3.5e38:          # float32's end, and NaN
            raise RuntimeError(f"KVCache.attend: scale {scale} is not finite")
        if window < 0 or most < 0:
            raise RuntimeError("KVCache.attend: window and max_new must not be negative")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous() \
                or out.data_ptr() % 16:
            raise RuntimeError(f"KVCache.attend: out must be a contiguous, 16-byte aligned {tuple(q.shape)} tensor of {q.dtype}")
        if rows == 0 or n_seq == 0 or most == 0:
            return out
        if width == 0:
            raise RuntimeError("KVCache.attend: tables without a page")
        q, qs = _rows(q, heads, self.dim)
        lib = _lib.load()
        most, window, dtype = min(most, rows), min(int(window), 2 ** 31 - 1), _DTYPES[q.dtype]
        with _lib.on_device(self.device):
            sizes = (heads, n_seq, most, dtype, width, window)
            nbytes = self._need.get(sizes)
            if nbytes is None:
                nbytes = lib.qmv_kv_attend_workspace_bytes(self._ref, *sizes)
                if nbytes <= 0:
                    raise RuntimeError(f"KVCache.attend: {heads} heads, {n_seq} sequences of {most} new tokens not supported")
                if len(self._need) >= 4096:           # sizes that never come back
                    self._need.clear()
                self._need[sizes] = nbytes
            if nbytes > 256:
                ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            else:                                     # used by nothing
                if self._none is None:
                    self._none = torch.empty(256, dtype=torch.uint8, device=self.device)
                ws = self._none
            st = lib.qmv_kv_attend(self._ref, q.data_ptr(), dtype, qs, heads, tables.data_ptr(), width, lens.data_ptr(),
                                   _lib.addr(starts), n_seq, rows, most, self.dim ** -0.5 if scale is None else float(scale), window,
                                   out.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_of(self.device))
        if st:
            _lib.check(st, "qmv_kv_attend")
        return out

    def copy(self, src: torch.Tensor, dst: torch.Tensor, used: Optional[torch.Tensor] = None) -> None:
        """Page src[i] copied to page dst[i] (int32, any shape; -1: nothing), its first used[i] tokens or all; for beams that part
        (pages.reorder).  No page is the target of two copies, nor target and source."""
        _lib.host().copy(self._at, self._where, src, dst, used)

    def bounds(self) -> torch.Tensor:
        """A new, zeroed float16 (n_pages, n_kv, 2, dim) for summarise and choose: the least and largest key of each page, key
        head and channel."""
        return torch.zeros((self.n_pages, self.n_kv, 2, self.dim), dtype=torch.float16, device=self.device)

    def summarise(self, bounds: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, starts: Optional[torch.Tensor] = None,
                  max_new: Optional[int] = None) -> None:
        """Writes into bounds (KVCache.bounds) the boxes of the pages that the newest tokens completed, behind their write; tables,
        lens, starts as for attend (one new token a sequence, or starts[b + 1] - starts[b]).  max_new: at least the most new tokens
        of a sequence (default: a whole table of them).  One launch."""
        _lib.host().summarise(self._at, self._where, tables, lens, starts, bounds, max_new)

    def choose(self, q: torch.Tensor, bounds: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, keep: int,
               starts: Optional[torch.Tensor] = None, first: int = 1, last: int = 1):
        """The pages each query looks at -> chosen int32 (rows, n_kv, keep), -1 behind the last one, and held int32 (rows,), the
        tokens in them, for attend_chosen.  q, tables, lens, starts as for attend (a positive scale is meant).  Of a query's pages the
        `first` first and the `last` last ones (1 at least: its own) are always chosen, of the others those whose box reaches
        furthest along some query head of the key head; all of them where there are no more than keep.  Rows that no sequence covers
        get none.  Boxes of all pages but the query's own must have been written (summarise).  Both are parts of one allocation: clone what is
        kept for long, resize none.  Two launches."""
        return _lib.host().choose(self._at, self._where, tables, lens, starts, bounds, q, keep, first, last)

    def attend_chosen(self, q: torch.Tensor, chosen: torch.Tensor, held: torch.Tensor, scale: Optional[float] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of each row of q over the pages chosen for it (choose): row r's heads of key head h see the first held[r] tokens
        of the pages chosen[r, h].  Rounding, scale and out as for attend; rows with held 0 give zeros."""
        return _lib.host().attend_chosen(self._at, self._where, q, chosen, held, scale, out)
