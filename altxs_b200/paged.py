"""Paged key/value cache: rotary positions, append and attention of new tokens.

A cache of fixed-size pages for streams of different lengths.  ``PagedKV``
holds (or wraps) the page pools of one layer, ``Chunks`` says which new tokens
a call brings to which sequences, ``PageAllocator`` hands out pages and builds
the ``Chunks`` of a batch of streams:

    alloc = PageAllocator(n_seqs, n_pages, page_size, max_kv, device)
    chunks = alloc.extend([64, 64, 1])            # new tokens of each stream
    q = cache.append(chunks, k, v, rotary=rot, q=q)
    y = cache.attend(chunks, q)

The attention covers a sequence's new tokens, one or thousands, over everything
it has cached (causal, optionally a sliding window): the role of the
reference's static cache and its encoder's multi-symbol windows
(``StaticACEngine``, altxs ``src/xsa_ttt/incremental.py:203-1218``,
``run_window`` ``:1268-1290``).  All tensors of a call share one type (fp32,
bf16 or fp16); work is enqueued on the current stream.  No call records a
gradient (inputs that require one raise; ``rope_backward`` is ``rope``'s).
Errors of the arguments raise; errors of the device data (a position beyond the
tables, a page out of range, lengths beyond their bounds) set bits that
``check_status`` raises on.
"""

from __future__ import annotations

import ctypes as C
import math
import weakref
from typing import Sequence

import numpy as np
import torch

from . import _lib

# the workspaces of the caches that are alive, by device and stream
_shared: weakref.WeakValueDictionary[tuple[torch.device, int], torch.Tensor] = weakref.WeakValueDictionary()
_GROWTH = 64 << 20  # bytes that a workspace grows by at most beyond what a call needs
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _stream_handle(device: torch.device) -> int:
    """The current stream of a device as the driver's handle (a torch Stream object costs 2 us a call)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


# the index of the current device: kernels launch there, whatever device their arguments are on
_current_device = torch._C._cuda_getDevice


def rope_table(positions: int, dims: int, base: float = 1e4, *, scaling: str | None = None, factor: float = 1.0,
               trained: int | None = None, device: torch.device | str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """cos/sin ``[positions][dims/2]`` (fp32, rounded once from 64 bits).

    Frequencies ``w_j = base^(-2j/dims)``; for contexts ``factor`` times longer
    than the ``trained`` length:

    - ``scaling="linear"``: every frequency divided by ``factor``;
    - ``scaling="base"``: the base raised to ``base * factor^(dims/(dims-2))``,
      which keeps the fastest frequency and divides the slowest by ``factor``;
    - ``scaling="parts"``: by the turns ``r_j = trained * w_j / 2 pi`` a pair makes
      over the trained length: pairs with ``r > 32`` keep their frequency, pairs
      with ``r < 1`` are divided by ``factor``, a linear ramp between, and the
      tables carry the amplitude ``0.1 ln(factor) + 1`` (scores grow by its square).
    """
    if positions < 0 or dims < 0 or dims % 2:
        raise ValueError("positions must be >= 0 and dims even")
    if factor < 1.0:
        raise ValueError("factor must be >= 1")
    j = torch.arange(0, dims, 2, dtype=torch.float64)
    amplitude = 1.0
    if scaling == "base" and dims > 2:
        base = base * factor ** (dims / (dims - 2))
    w = base ** (-j / max(dims, 1))
    if scaling == "linear":
        w = w / factor
    elif scaling == "parts":
        if trained is None:
            raise ValueError("scaling='parts' needs the trained length")
        keep = ((trained * w / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        w = w * (keep + (1.0 - keep) / factor)
        amplitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"unknown scaling {scaling!r}")
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * w.to(device)
    return (a.cos() * amplitude).float(), (a.sin() * amplitude).float()


def _raise_status(word: torch.Tensor, what: str) -> None:
    v = int(word.item())
    if v:
        word.zero_()
        why = "a device wait gave up" if v & _lib.ST_TIMEOUT else "position, page or length out of range"
        raise RuntimeError(f"{what}: device status {v:#x} ({why})")


class Rotary:
    """Rotary tables (``rope_table``, or ``DeviceModel.rope_cos`` / ``rope_sin``) and their pairing."""

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False):
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or cos.shape != sin.shape:
            raise ValueError("cos and sin must be fp32 [positions][dims/2] of one shape")
        if not (cos.is_contiguous() and sin.is_contiguous()) or cos.device != sin.device or not cos.is_cuda:
            raise ValueError("cos and sin must be contiguous on one GPU")
        self.cos, self.sin, self.device = cos, sin, cos.device
        self.status = torch.zeros(1, dtype=torch.int32, device=cos.device)
        self.struct = _lib.RotaryTables(cos=cos.data_ptr(), sin=sin.data_ptr(), positions=cos.shape[0],
                                        dims=2 * cos.shape[1], interleaved=int(interleaved))
        self._ref = C.byref(self.struct)

    def check_status(self) -> None:
        """Waits for the current stream; raises if a position of ``rope`` was outside the tables."""
        _raise_status(self.status, "rope")


def _heads(x: torch.Tensor, what: str, dtype: torch.dtype, device: torch.device) -> int:
    """Row stride of ``[tokens][heads][head_dim]`` whose heads lie side by side."""
    if x.dim() != 3 or x.dtype != dtype or x.device != device:
        raise ValueError(f"{what} must be [tokens][heads][head_dim] {dtype} on {device}")
    st = x.stride()
    n, h, d = x.shape
    if (d > 1 and st[2] != 1) or (h > 1 and st[1] != d):
        raise ValueError(f"{what}: the heads of a token must lie side by side")
    return st[0] if n > 1 else h * d  # the stride over one token is never taken


def _no_history(what: str) -> None:
    """For an input that a gradient is asked for: raises, since what these calls return has no history."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} records no gradient: detach its inputs or call it under torch.no_grad() "
                           "(rope_backward is rope's gradient)")


def _positions(pos: torch.Tensor, n: int, device: torch.device) -> int:
    if pos.dtype != torch.int64 or pos.shape != (n,) or pos.device != device or not pos.is_contiguous():
        raise ValueError(f"positions must be a contiguous int64 [{n}] tensor on {device}")
    return pos.data_ptr()


def _rope(x: torch.Tensor, rotary: Rotary, pos: torch.Tensor, out: torch.Tensor | None, backward: int) -> torch.Tensor:
    if _current_device() != rotary.device.index:
        with torch.cuda.device(rotary.device):
            return _rope(x, rotary, pos, out, backward)
    if x.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {x.dtype}")
    if x.requires_grad:
        _no_history("rope")
    ldx = _heads(x, "x", x.dtype, rotary.device)
    n, h, d = x.shape
    p = _positions(pos, n, rotary.device)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        ldy = h * d
    else:
        ldy = _heads(out, "out", x.dtype, rotary.device)
        if out.shape != x.shape:
            raise ValueError("out must have x's shape")
    rc = _lib.lib().altxs_rope(_DTYPES[x.dtype], n, h, d, rotary._ref, p, backward, x.data_ptr(), ldx, out.data_ptr(),
                               ldy, rotary.status.data_ptr(), _stream_handle(rotary.device))
    _lib.check(rc, "altxs_rope")
    return out


def rope(x: torch.Tensor, rotary: Rotary, pos: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x`` ``[tokens][heads][head_dim]`` rotated to its positions (``out=x`` in place)."""
    return _rope(x, rotary, pos, out, 0)


def rope_backward(dy: torch.Tensor, rotary: Rotary, pos: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of ``rope``: the transposed rotation of ``dy``."""
    return _rope(dy, rotary, pos, out, 1)


def _workspace(need: int, device: torch.device) -> torch.Tensor:
    """A new workspace of the attention: its counters are zero, the rest needs no value."""
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
    ws[:_lib.PAGED_COUNTER_BYTES].zero_()
    return ws


class Chunks:
    """The new tokens of a batch of sequences (``altxs_chunks``).

    ``q_start`` int32 ``[n_seqs + 1]``: sequence s owns rows ``q_start[s] ..
    q_start[s+1]`` of the token tensors; ``kv_len`` int32 ``[n_seqs]``: its
    positions in the cache, the new tokens (the last ones) included;
    ``page_table`` int32 ``[n_seqs][blocks]``.  ``max_new`` and ``max_kv`` bound
    the device lengths, ``total_kv`` their sum where it is known.
    """

    def __init__(self, q_start: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor, *, max_new: int,
                 max_kv: int, total_kv: int = 0):
        n = kv_len.shape[0] if kv_len.dim() == 1 else -1
        for t, shape in ((q_start, (n + 1,)), (kv_len, (n,)), (page_table, (n, page_table.shape[-1]))):
            if t.dtype != torch.int32 or t.shape != shape or t.device != q_start.device:
                raise ValueError("q_start [n+1], kv_len [n] and page_table [n][blocks] must be int32 on one device")
        if not (q_start.is_contiguous() and kv_len.is_contiguous()) or (page_table.shape[1] > 1 and
                                                                       page_table.stride(1) != 1):
            raise ValueError("q_start, kv_len and the rows of page_table must be contiguous")
        if page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
            raise ValueError("the rows of page_table must not overlap")
        if not (0 <= max_new < 1 << 31 and 0 <= max_kv < 1 << 31 and 0 <= total_kv < 1 << 63):
            raise ValueError("max_new, max_kv and total_kv must be counts (of 31, 31 and 63 bits)")
        self.q_start, self.kv_len, self.page_table = q_start, kv_len, page_table
        self.device, self.max_kv = q_start.device, int(max_kv)
        self.struct = _lib.Chunks(q_start=q_start.data_ptr(), kv_len=kv_len.data_ptr(),
                                  page_table=page_table.data_ptr(),
                                  table_stride=page_table.stride(0) if n > 1 else page_table.shape[1], n_seqs=n,
                                  n_tokens=0, max_new=int(max_new), max_kv=int(max_kv), total_kv=int(total_kv))
        self._ref = C.byref(self.struct)


class PagedKV:
    """Page pools of one layer's keys and values: ``[pages][page_size][kv_heads][head_dim]``
    tensors of equal strides (any view with contiguous channels; a
    ``[pages][kv_heads][page_size][head_dim]`` pool is passed as its
    ``transpose(1, 2)``).  ``PagedKV.empty`` allocates them."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        # a stride over one element is never taken: whatever it is, it stands for the channels of a head
        strides = [[s if m > 1 else x.shape[-1] for m, s in zip(x.shape, x.stride())] for x in (k, v)]
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or strides[0] != strides[1]:
            raise ValueError("k and v must be [pages][page_size][kv_heads][head_dim] of equal shape, type and strides")
        if k.dtype not in _DTYPES or not k.is_cuda or k.device != v.device:
            raise ValueError("k and v must be fp32, bf16 or fp16 on one GPU")
        if k.stride(3) != 1:
            raise ValueError("the channels of k and v must be contiguous")
        self.k, self.v, self.device, self.dtype = k, v, k.device, k.dtype
        self.page_size, self.kv_heads, self.head_dim = k.shape[1:]
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        ps, ts, hs, _ = strides[0]
        self.struct = _lib.PagedKv(k=k.data_ptr(), v=v.data_ptr(), page_stride=ps, token_stride=ts,
                                   head_stride=hs, dtype=_DTYPES[k.dtype], page_size=self.page_size,
                                   n_pages=k.shape[0], n_kv_heads=self.kv_heads, head_dim=self.head_dim)
        self._ref = C.byref(self.struct)
        self._ws: dict[int, torch.Tensor] = {}  # by stream: calls on different streams do not share

    @classmethod
    def empty(cls, n_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.float32,
              device: torch.device | str = "cuda") -> PagedKV:
        shape = (n_pages, page_size, kv_heads, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))

    def _chunks(self, c: Chunks, n: int):
        if c.device != self.device:
            raise ValueError(f"chunks must be on {self.device}")
        if c.page_table.shape[1] * self.page_size < c.max_kv:
            raise ValueError("the page table does not cover max_kv positions")
        c.struct.n_tokens = n
        c.struct.status = self.status.data_ptr()
        return c._ref

    def _workspace_for(self, need: int, stream: int) -> torch.Tensor:
        """One workspace per stream, shared by the caches whose calls follow one another there and freed with the
        last of them (a call that gives up spoils it for all of them: each then reports that).  A call that is
        captured has its own, from the graph's memory and cleared in the graph: it lives as long as the graph does,
        and no other call, captured or not, meets its counters."""
        if torch.cuda.is_current_stream_capturing():
            return _workspace(need, self.device)
        ws = self._ws.get(stream)
        if ws is None or ws.numel() < need:
            ws = _shared.get((self.device, stream))
            if ws is None or ws.numel() < need:  # with room for the next steps of growing streams
                more = 0 if ws is None else ws.numel() + min(ws.numel() // 2, _GROWTH)
                ws = _shared[self.device, stream] = _workspace(max(need, more), self.device)
            self._ws[stream] = ws
        return ws

    def append(self, chunks: Chunks, k: torch.Tensor, v: torch.Tensor, *, rotary: Rotary | None = None,
               q: torch.Tensor | None = None, positions: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Writes the new tokens' keys (rotated) and values to their pages; returns
        the rotated queries when ``q`` is given.  ``positions``: rotary positions
        where they are not the cache's own."""
        if _current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self.append(chunks, k, v, rotary=rotary, q=q, positions=positions, q_out=q_out)
        if k.requires_grad or v.requires_grad or (q is not None and q.requires_grad):
            _no_history("append")
        ldk, ldv = _heads(k, "k", self.dtype, self.device), _heads(v, "v", self.dtype, self.device)
        n = k.shape[0]
        if k.shape != v.shape or k.shape[1:] != (self.kv_heads, self.head_dim):
            raise ValueError("k and v must be [tokens][kv_heads][head_dim]")
        if rotary is not None and rotary.device != self.device:
            raise ValueError(f"the rotary tables must be on {self.device}")
        qp = qo = None
        ldq = ldqo = H = 0
        if q is not None:
            ldq, H = _heads(q, "q", self.dtype, self.device), q.shape[1]
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            ldqo = _heads(q_out, "q_out", self.dtype, self.device)
            if q.shape != (n, H, self.head_dim) or q_out.shape != q.shape:
                raise ValueError("q and q_out must be [tokens][heads][head_dim]")
            qp, qo = q.data_ptr(), q_out.data_ptr()
        rc = _lib.lib().altxs_paged_append(
            self._ref, self._chunks(chunks, n), None if rotary is None else rotary._ref,
            None if positions is None else _positions(positions, n, self.device), k.data_ptr(), ldk, v.data_ptr(), ldv,
            H, qp, ldq, qo, ldqo, _stream_handle(self.device))
        _lib.check(rc, "altxs_paged_append")
        return q_out

    def attend(self, chunks: Chunks, q: torch.Tensor, *, scale: float | None = None, window: int = 0,
               out: torch.Tensor | None = None, return_lse: bool = False):
        """Attention of the new tokens over the cache: ``[tokens][heads][head_dim]``, and
        with ``return_lse`` each row's log2 sum ``[heads][tokens]`` (fp32).
        ``scale`` defaults to ``head_dim ** -0.5``; ``window`` 0 sees everything.  Rows of no
        sequence are not written."""
        if _current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self.attend(chunks, q, scale=scale, window=window, out=out, return_lse=return_lse)
        if q.requires_grad:
            _no_history("attend")
        ldq = _heads(q, "q", self.dtype, self.device)
        n, H, d = q.shape
        if d != self.head_dim or H % self.kv_heads:
            raise ValueError("q must be [tokens][heads][head_dim] with heads a multiple of kv_heads")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            ldo = H * d
        else:
            ldo = _heads(out, "out", self.dtype, self.device)
            if out.shape != q.shape:
                raise ValueError("out must have q's shape")
        lse = torch.empty((H, n), dtype=torch.float32, device=self.device) if return_lse else None
        window = max(-1, min(window, (1 << 31) - 1))  # (beyond 32 bits it would arrive as another)
        L = _lib.lib()
        cref, st = self._chunks(chunks, n), _stream_handle(self.device)
        need = L.altxs_paged_attention_workspace_bytes(self._ref, cref, H, window)
        if need < 0:
            _lib.check(_lib.ALTXS_EINVAL, "altxs_paged_attention_workspace_bytes")
        ws = self._workspace_for(need, st) if need else None
        rc = L.altxs_paged_attention(self._ref, cref, H, self.head_dim ** -0.5 if scale is None else scale, window,
                                     q.data_ptr(), ldq, out.data_ptr(), ldo, lse.data_ptr() if return_lse else None,
                                     ws.data_ptr() if need else None, ws.numel() if need else 0, st)
        _lib.check(rc, "altxs_paged_attention")
        return (out, lse) if return_lse else out

    def check_status(self) -> None:
        """Waits for the current stream (the calls' own, or one that follows it); raises if a call met a position,
        page or length out of range, or gave up waiting."""
        try:
            _raise_status(self.status, "paged cache")
        except RuntimeError:
            # A call that gave up may leave its counters counting: later calls start from zeroed ones, on this
            # stream in the same workspace, elsewhere in another.
            here = _stream_handle(self.device) if self._ws else 0
            for stream, ws in list(self._ws.items()):
                if stream == here:
                    ws[:_lib.PAGED_COUNTER_BYTES].zero_()
                else:
                    del self._ws[stream]
                    if _shared.get((self.device, stream)) is ws:
                        del _shared[self.device, stream]
            raise


class PageAllocator:
    """Pages of a batch of streams (host side): grants pages as streams grow,
    takes them back, and builds the ``Chunks`` of a step.  One allocator serves
    the caches of all layers, since they share lengths and page tables."""

    def __init__(self, n_seqs: int, n_pages: int, page_size: int, max_kv: int, device: torch.device | str = "cuda"):
        if n_seqs < 1 or n_pages < 0 or page_size < 1 or max_kv < 1:
            raise ValueError("n_seqs, page_size and max_kv must be positive")
        self.page_size, self.max_kv, self.device = page_size, int(max_kv), torch.device(device)
        self.free = list(range(n_pages - 1, -1, -1))
        self.table = np.full((n_seqs, -(-self.max_kv // page_size)), -1, dtype=np.int32)
        self.len = np.zeros(n_seqs, dtype=np.int32)

    def extend(self, new: Sequence[int]) -> Chunks:
        """Grants the pages of ``new[s]`` more tokens of every stream s; raises
        (granting nothing) when a stream would pass ``max_kv`` or the pages run out."""
        new = np.asarray(new, dtype=np.int32)
        if new.shape != self.len.shape or (new < 0).any():
            raise ValueError(f"new must be {self.len.shape[0]} counts")
        grown = self.len.astype(np.int64) + new
        if (grown > self.max_kv).any():
            raise ValueError("a stream would pass max_kv")
        have, want = -(-self.len // self.page_size), -(-grown // self.page_size)
        if int((want - have).sum()) > len(self.free):
            raise RuntimeError("out of pages")
        for s in np.nonzero(want > have)[0]:
            for b in range(have[s], want[s]):
                self.table[s, b] = self.free.pop()
        self.len = grown.astype(np.int32)
        start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        up = lambda a: torch.from_numpy(a.copy()).to(self.device)  # noqa: E731
        return Chunks(up(start), up(self.len), up(self.table), max_new=int(new.max()), max_kv=max(1, int(self.len.max())),
                      total_kv=int(self.len.sum()))

    def trim(self, seq: int, window: int) -> int:
        """Takes back the pages that no later token of a ``window``-wide attention
        sees (``window`` 0 sees everything); returns how many."""
        if window < 0:
            raise ValueError("window must be >= 0")
        if window == 0:
            return 0
        first = max(0, int(self.len[seq]) + 1 - window) // self.page_size  # block of the next token's first position
        behind = self.table[seq, :first]
        back = behind[behind >= 0].tolist()
        self.free += back
        behind[:] = -1
        return len(back)

    def release(self, seq: int) -> None:
        """Ends a stream: its pages are free again and its length is 0."""
        self.free += [int(p) for p in self.table[seq] if p >= 0]
        self.table[seq] = -1
        self.len[seq] = 0
