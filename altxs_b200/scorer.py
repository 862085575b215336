"""Teacher-forced scoring of many streams in chunks over paged caches.

``PagedScorer`` runs the plain model over streams of different lengths, some
symbols of each at a time, keeping what every stream has cached in pages: the
bits a stream would cost under the model, without coding it (ranking candidate
inputs, checking a codec's weights on held-out data, choosing a segment
length).  It is the chunked form of the engine's step: a chunk of W symbols per
stream is one forward, as in the reference's windowed encoder (``run_window``,
altxs ``src/xsa_ttt/incremental.py:1268-1290``), over each stream's own sliding
window of ``cfg.ctx`` symbols at absolute positions.  Pages that have left a
stream's window are taken back as it goes, so memory follows the windows and not
the stream lengths.

The linears run on the library's mixed-bit kernels, keys and values are rotated
and stored by ``PagedKV.append`` and read by ``PagedKV.attend`` in fp32.
Adapters are not applied; models with motifs, or whose context is rebuilt at every
segment (``context_mode="reset"``), are refused.
"""

from __future__ import annotations

import ctypes as C
import math
from typing import Sequence

import numpy as np
import torch
import torch.nn.functional as F

from . import _lib
from .engine import DeviceModel, _stream_handle
from .paged import PageAllocator, PagedKV, Rotary


class PagedScorer:
    """``dm``: the model; ``max_len``: the longest stream; ``page_size``: positions per page;
    ``n_pages``: pages per layer (default: enough for every stream's window and a chunk)."""

    def __init__(self, dm: DeviceModel, n_streams: int, max_len: int, *, chunk: int = 64, page_size: int = 64,
                 n_pages: int | None = None):
        cfg = dm.cfg
        if (cfg.smear_gate_enabled or cfg.xsa_last_n or cfg.sparse_attn_gate_enabled or cfg.asym_logit_rescale
                or cfg.num_loops or cfg.parallel_start_layer):
            raise ValueError("PagedScorer runs plain models only (no motifs)")
        if cfg.context_mode != "sliding":
            raise ValueError(f"PagedScorer scores with a sliding window, not context_mode={cfg.context_mode!r}")
        if cfg.head_dim not in (32, 64, 128):
            raise ValueError(f"the paged cache has heads of 32, 64 or 128 channels, not {cfg.head_dim}")
        if chunk < 1 or max_len < 1 or n_streams < 1:
            raise ValueError("chunk, max_len and n_streams must be positive")
        self.dm, self.cfg, self.n, self.chunk, self.window = dm, cfg, int(n_streams), int(chunk), int(cfg.ctx)
        dm.ensure_rope(max_len + 1)
        self.rotary = Rotary(dm.rope_cos, dm.rope_sin)
        if n_pages is None:
            held = min(max_len, self.window + chunk)
            n_pages = self.n * (-(-held // page_size) + 2)
        self.pages = PageAllocator(self.n, n_pages, page_size, max_len, dm.device)
        self.caches = [PagedKV.empty(n_pages, page_size, cfg.num_kv_heads, cfg.head_dim, device=dm.device)
                       for _ in range(cfg.num_layers)]
        emb = dm.q["emb"]
        if dm.full_params:  # the arena's own: an update between calls changes it
            self.emb = dm.arena("emb").view(emb.rows, emb.cols)
        else:
            self.emb = torch.empty((emb.rows, emb.cols), dtype=torch.float32, device=dm.device)
            _lib.check(_lib.lib().altxs_dequant(C.byref(emb), self.emb.data_ptr(), emb.cols, _stream_handle(dm.device)),
                       "altxs_dequant")
        layers, d = cfg.num_layers, cfg.model_dim
        shapes = {"q_gain": (layers, cfg.num_heads), "attn_scale": (layers, d), "mlp_scale": (layers, d),
                  "resid_mix": (layers, 2, d), "ln_scale": (layers,), "skip_weights": (-1, d), "skip_gates": (-1, d)}
        self.small = {k: dm.small[k].view(shape) for k, shape in shapes.items()}  # (an arena's are flat)
        self._ws = torch.empty(0, dtype=torch.uint8, device=dm.device)

    def _linear(self, name: str, row0: int, rows: int, x: torch.Tensor) -> torch.Tensor:
        L, q, split = _lib.lib(), self.dm.q[name], self.dm._split
        y = torch.empty((x.shape[0], rows), dtype=torch.float32, device=x.device)
        need = int(L.altxs_linear_workspace_bytes(x.shape[0], q.cols))
        if self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        hi, lo = (getattr(split, f"{name}_{p}") for p in ("hi", "lo")) if split is not None else (None, None)
        _lib.check(L.altxs_linear(C.byref(q), hi, lo, row0, rows, x.data_ptr(), x.shape[0], y.data_ptr(),
                                  self._ws.data_ptr(), self._ws.numel(), _stream_handle(x.device)), "altxs_linear")
        return y

    def advance(self, new: Sequence[np.ndarray]) -> torch.Tensor:
        """Consumes ``new[s]`` (also none) of every stream and returns the logits after
        each: ``[sum of lengths][vocab]``, stream by stream.  The default ``n_pages``
        hold ``chunk`` symbols of every stream at a time; more may raise "out of pages"
        (nothing is consumed then)."""
        cfg, sm, dev = self.cfg, self.small, self.dm.device
        lens = [len(a) for a in new]
        tokens = torch.from_numpy(np.concatenate([np.asarray(a, dtype=np.int64) for a in new])).to(dev)
        if tokens.numel() and (int(tokens.min()) < 0 or int(tokens.max()) >= cfg.vocab_size):
            raise ValueError("symbol outside the vocabulary")
        chunks = self.pages.extend(lens)
        if not tokens.numel():
            return torch.empty((0, cfg.vocab_size), dtype=torch.float32, device=dev)
        d, H, Hkv, hd, kvd, mh = cfg.model_dim, cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.kv_dim, cfg.mlp_hidden
        rms = lambda t: F.rms_norm(t, (t.size(-1),))  # noqa: E731
        x = x0 = rms(self.emb[tokens])
        enc, dec = cfg.layer_schedule
        skips = []
        for slot, i in enumerate(enc + dec):
            if slot >= len(enc) and slot - len(enc) < cfg.num_skip_weights and skips:
                j = slot - len(enc)
                scaled = sm["skip_weights"][j] * skips.pop()
                x = torch.lerp(scaled, x, torch.sigmoid(sm["skip_gates"][j])) if cfg.skip_gates_enabled else x + scaled
            ln = sm["ln_scale"][i]
            x = sm["resid_mix"][i][0] * x + sm["resid_mix"][i][1] * x0
            qkv = self._linear("qkv", i * (d + 2 * kvd), d + 2 * kvd, rms(x) * ln)
            q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.split([d, kvd, kvd], 1))
            q = rms(q) * sm["q_gain"][i][:, None]
            q = self.caches[i].append(chunks, rms(k), v, rotary=self.rotary, q=q, q_out=q)
            y = self.caches[i].attend(chunks, q, window=self.window)
            x = x + sm["attn_scale"][i] * self._linear("o", i * d, d, y.flatten(1))
            h = F.leaky_relu(self._linear("up", i * mh, mh, rms(x) * ln), 0.5).square()
            x = x + sm["mlp_scale"][i] * self._linear("down", i * d, d, h)
            if slot < len(enc):
                skips.append(x)
        for s in range(self.n):
            self.pages.trim(s, self.window)
        logits = self._linear("emb", 0, cfg.vocab_size, rms(x))
        return cfg.logit_softcap * torch.tanh(logits / cfg.logit_softcap)

    def score(self, streams: Sequence[np.ndarray]) -> list[np.ndarray]:
        """Bits of every symbol of every stream (fp64); a stream's first symbol costs log2(vocab)."""
        if len(streams) != self.n:
            raise ValueError(f"expected {self.n} streams")
        for s in range(self.n):
            self.pages.release(s)
        bits = [np.zeros(len(a)) for a in streams]
        for b in bits:
            b[:1] = math.log2(self.cfg.vocab_size)
        for t0 in range(0, max(len(a) for a in streams), self.chunk):
            new = [a[t0:min(t0 + self.chunk, max(len(a) - 1, 0))] for a in streams]  # the last symbol predicts nothing
            target = np.concatenate([a[t0 + 1:t0 + 1 + len(p)] for a, p in zip(streams, new)]).astype(np.int64)
            if not target.size:
                break
            logits = self.advance(new).double()
            at = torch.from_numpy(target).to(logits.device)
            cost = ((torch.logsumexp(logits, 1) - logits.gather(1, at[:, None])[:, 0]) / math.log(2)).cpu().numpy()
            at = 0
            for b, p in zip(bits, new):
                b[t0 + 1:t0 + 1 + len(p)] = cost[at:at + len(p)]
                at += len(p)
        for c in self.caches:
            c.check_status()
        return bits
