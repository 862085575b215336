"""Paged cache on the GPU: rotary positions, append and attention of new tokens
against plain restatements in 64 bits.

Tolerances, from the arithmetic: a value rounded once to b significand bits is
within 2^-b of it relatively.  The rotation is two fp32 products and a sum of
values of size |x|, then one rounding: 2^-22 |x|max (fp32), 2^-8 (bf16), 2^-11
(fp16) of |x|max sqrt(2).  The attention's output is a mean of V rows: fp32
scores of up to ~40 (log2 units) carry 40 x 2^-21 from products kept to 22 bits
and the exponential's 2^-22, so 4e-5 |V|max covers p's relative error; in 16
bits p is rounded once (2^-9, 2^-12) and the result once more, and q, k, v are
the inputs' own: 2^-8 and 2^-11 of |V|max with half as much again for the
scores.  The row sums' log2 is fp32: 4e-5 absolute.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from altxs_b200 import _lib, paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROT_TOL = {"f32": 2.0 ** -22, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
ATT_TOL = {"f32": 4e-5, "bf16": 1.5 * 2.0 ** -8, "f16": 1.5 * 2.0 ** -11}
LSE_TOL = 4e-5


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rot_ref(x, cos, sin, pos, il, backward=False):
    """The rotation pair by pair in 64 bits, as matrices [[c, s], [-s, c]] (transposed backward)."""
    x = x.double().clone()
    d = 2 * cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    if backward:
        s = -s
    j = torch.arange(d // 2, device=x.device)
    ia, ib = (2 * j, 2 * j + 1) if il else (j, j + d // 2)
    a, b = x[..., ia].clone(), x[..., ib].clone()
    x[..., ia], x[..., ib] = c * a + s * b, c * b - s * a
    return x


def _table(n, dims):
    return paged.rope_table(n, dims, device=DEV)


# ---- rotary positions ----------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("T,H,hd,dims,lead", [(1, 1, 2, 2, 0), (1, 3, 32, 8, 0), (7, 5, 64, 16, 64), (130, 8, 128, 128, 3),
                                               (33, 2, 96, 48, 0), (5, 1, 512, 512, 8), (300, 1, 64, 0, 0), (3, 7, 30, 14, 1)])
def test_rope_forward_and_backward(dtype, il, T, H, hd, dims, lead):
    g = _gen(T * 31 + hd)
    cos, sin = _table(5000, dims)
    rot = paged.Rotary(cos, sin, il)
    wide = _rand(g, T, lead + H * hd + 5).to(DT[dtype])
    x = wide[:, lead:lead + H * hd].unflatten(1, (H, hd))
    pos = torch.randint(0, 5000, (T,), generator=g, device=DEV)
    for back, f in ((False, paged.rope), (True, paged.rope_backward)):
        want = _rot_ref(x, cos, sin, pos, il, back)
        y = f(x, rot, pos)
        err = (y.double() - want).abs().max().item()
        assert err <= ROT_TOL[dtype] * math.sqrt(2) * x.abs().max().item()
    assert torch.equal(y[..., dims:], x[..., dims:])
    # in place through the same strided view: same bits, and nothing outside the view changes
    keep, y = wide.clone(), paged.rope(x, rot, pos)
    paged.rope(x, rot, pos, out=x)
    assert torch.equal(x, y)
    assert torch.equal(wide[:, :lead], keep[:, :lead]) and torch.equal(wide[:, lead + H * hd:], keep[:, lead + H * hd:])
    rot.check_status()


@pytest.mark.parametrize("il", [False, True])
def test_rope_backward_is_the_gradient(il):
    """Against differences: the loss sum(c * rope(x)) changes by <rope_backward(c), e> along every e
    (the map is linear, so the quotient is exact up to rounding)."""
    g = _gen(3)
    cos, sin = _table(100, 12)
    rot = paged.Rotary(cos, sin, il)
    x, c = _rand(g, 2, 1, 16), _rand(g, 2, 1, 16)
    pos = torch.tensor([17, 99], device=DEV)
    grad = paged.rope_backward(c, rot, pos)
    base = (c * paged.rope(x, rot, pos)).double().sum()
    for i in range(x.numel()):
        e = torch.zeros_like(x)
        e.view(-1)[i] = 1.0
        diff = (c * paged.rope(x + e, rot, pos)).double().sum() - base
        assert abs(diff.item() - grad.reshape(-1)[i].item()) < 32 * 2.0 ** -21
    xg = x.double().requires_grad_()
    (_autograd_rot(xg, cos, sin, pos, il) * c).sum().backward()
    assert (xg.grad - grad).abs().max().item() < 2.0 ** -20


def _autograd_rot(x, cos, sin, pos, il):
    d = 2 * cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = (x[..., 0:d:2], x[..., 1:d:2]) if il else (x[..., :d // 2], x[..., d // 2:d])
    u, v = a * c + b * s, b * c - a * s
    r = torch.stack((u, v), -1).flatten(-2) if il else torch.cat((u, v), -1)
    return torch.cat((r, x[..., d:]), -1)


def test_rope_position_outside_the_table():
    cos, sin = _table(10, 16)
    rot = paged.Rotary(cos, sin)
    x = _rand(_gen(1), 4, 2, 32)
    y = paged.rope(x, rot, torch.tensor([0, 10, -1, 9], device=DEV))
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[[0, 3]]).all()
    with pytest.raises(RuntimeError, match="status 0x20"):
        rot.check_status()
    rot.check_status()


def test_rope_matches_the_engine_tables():
    """The engine's own tables and sense: the step's rotation of a head."""
    from altxs_b200.config import c3_config
    from altxs_b200.lora import rope_tables

    cfg = c3_config()
    cos, sin = (torch.from_numpy(a).to(DEV) for a in rope_tables(cfg, 64))
    x = _rand(_gen(2), 3, cfg.num_heads, cfg.head_dim)
    pos = torch.tensor([0, 5, 63], device=DEV)
    y = paged.rope(x, paged.Rotary(cos, sin), pos)
    h = cfg.rope_dims // 2
    x1, x2, c, s = x[..., :h], x[..., h:2 * h], cos[pos][:, None], sin[pos][:, None]
    want = torch.cat((x1 * c + x2 * s, x1 * -s + x2 * c, x[..., 2 * h:]), -1)
    assert (y - want).abs().max().item() < 1e-6


# ---- a batch of sequences over a paged cache --------------------------------------


class Batch:
    """Random sequences in a random page order; unheld pages and slots past a
    sequence's length hold NaN."""

    def __init__(self, dtype, hd, Hkv, P, news, kvs, seed=0, layout="nhd", spare=2):
        g = _gen(seed)
        blocks = [-(-max(k, 0) // P) for k in kvs]
        n_pages = sum(blocks) + spare
        perm = torch.randperm(n_pages, generator=g, device=DEV).tolist()
        cols = max(1, max(blocks))
        table = np.full((len(kvs), cols), 0x7ffffff0, dtype=np.int32)
        at = 0
        for s, b in enumerate(blocks):
            table[s, :b] = perm[at:at + b]
            at += b
        shape = (n_pages, P, Hkv, hd) if layout == "nhd" else (n_pages, Hkv, P, hd)
        if layout == "pair":  # keys and values of a page side by side
            both = torch.full((n_pages, 2, P, Hkv, hd), float("nan"), dtype=DT[dtype], device=DEV)
            k, v = both[:, 0], both[:, 1]
        else:
            k, v = (torch.full(shape, float("nan"), dtype=DT[dtype], device=DEV) for _ in range(2))
            if layout == "hnd":
                k, v = k.transpose(1, 2), v.transpose(1, 2)
        self.K = [_rand(g, max(L, 0), Hkv, hd).to(DT[dtype]) for L in kvs]
        self.V = [_rand(g, max(L, 0), Hkv, hd).to(DT[dtype]) for L in kvs]
        self.table, self.P, self.news, self.kvs, self.dtype, self.hd, self.Hkv = table, P, news, kvs, dtype, hd, Hkv
        self.cache = paged.PagedKV(k, v)
        for s in range(len(kvs)):
            self.fill(s, 0, kvs[s])
        self.q_start = torch.tensor(np.concatenate(([0], np.cumsum(news))), dtype=torch.int32, device=DEV)
        self.kv_len = torch.tensor(kvs, dtype=torch.int32, device=DEV)
        self.tab = torch.from_numpy(table).to(DEV)
        self.chunks = self.make_chunks()

    def slots(self, s, p0, p1):
        pos = torch.arange(p0, p1, device=DEV)
        return self.tab_of(s)[pos // self.P].long(), pos % self.P

    def tab_of(self, s):
        return torch.from_numpy(self.table[s]).to(DEV)

    def fill(self, s, p0, p1):
        if p1 > p0:
            page, slot = self.slots(s, p0, p1)
            self.cache.k[page, slot], self.cache.v[page, slot] = self.K[s][p0:p1], self.V[s][p0:p1]

    def make_chunks(self, **kw):
        kw = {"max_new": max(self.news), "max_kv": max(1, max(self.kvs)), **kw}
        return paged.Chunks(self.q_start, self.kv_len, self.tab, **kw)

    def ref(self, q, scale, window):
        """Row by row over the keys a row sees, 64 bits; (out, lse in log2 units)."""
        T, H, hd = q.shape
        out = torch.zeros(T, H, hd, dtype=torch.float64, device=DEV)
        lse = torch.full((H, T), -math.inf, dtype=torch.float64, device=DEV)
        t = 0
        for s, (n, L) in enumerate(zip(self.news, self.kvs)):
            K, V = (x[s].double().repeat_interleave(H // self.Hkv, 1) for x in (self.K, self.V))
            for i in range(n):
                p = L - n + i
                if p >= 0:
                    lo = max(0, p - window + 1) if window else 0
                    x = torch.einsum("hd,jhd->hj", q[t].double(), K[lo:p + 1]) * scale
                    lse[:, t] = torch.logsumexp(x, 1) / math.log(2)
                    out[t] = torch.einsum("hj,jhd->hd", torch.softmax(x, 1), V[lo:p + 1])
                t += 1
        return out, lse


def _check(b, q, window=0, scale=None, cache=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, lse = b.cache.attend(b.chunks, q, scale=scale, window=window, return_lse=True)
    want, wl = b.ref(q, scale, window)
    vmax = max([v.abs().max().item() for v in b.V if v.numel()] + [1.0])
    assert torch.isfinite(out).all()
    assert (out.double() - want).abs().max().item() <= ATT_TOL[b.dtype] * vmax
    seen = torch.isfinite(wl)
    assert torch.equal(torch.isneginf(lse), ~seen)
    if seen.any():
        assert (lse.double() - wl)[seen].abs().max().item() <= LSE_TOL
    b.cache.check_status()
    return out, lse


# every head size and type against group sizes, page sizes, lengths around tiles and splits
ONE = [([1], [1]), ([1, 1, 1], [2, 17, 33]), ([1] * 5, [255, 256, 257, 640, 1]), ([1, 1], [4097, 511]),
       ([1, 0, 1], [100, 37, 0])]
FEW = [([2], [2]), ([3, 5], [3, 300]), ([4, 1, 7], [259, 1, 1030]), ([5], [2])]
MANY = [([17], [17]), ([64, 33], [64, 500]), ([130, 1, 129], [130, 77, 1000]), ([300], [1300]), ([40], [10]),
        ([257, 2, 128], [257, 2, 385])]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kind", ["one", "few", "many"])
def test_attention_matches_float64(dtype, hd, kind):
    cases = {"one": ONE, "few": FEW, "many": MANY}[kind]
    for i, (news, kvs) in enumerate(cases):
        Hkv, G = [(1, 1), (2, 4), (3, 3), (1, 16), (4, 1), (2, 8)][i]
        P = [16, 1, 24, 64, 7, 128][(i + hd // 32) % 6]
        for window in (0, [1, 5, 64, 300][i % 4]):
            b = Batch(dtype, hd, Hkv, P, news, kvs, seed=i, layout=["nhd", "hnd", "pair"][i % 3])
            q = (2.0 * _rand(_gen(9 + i), sum(news), Hkv * G, hd)).to(DT[dtype])
            _check(b, q, window=window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_peaked_and_growing_scores(dtype):
    """Scores that rise along the keys (the running maximum moves at every tile) and rows
    dominated by one key."""
    b = Batch(dtype, 64, 2, 32, [1, 40], [700, 700], seed=4)
    for s in range(2):
        ramp = torch.linspace(-3, 3, b.kvs[s], device=DEV)[:, None, None]
        b.K[s] = (torch.ones(b.kvs[s], 2, 64, device=DEV) * ramp).to(DT[dtype])
        b.fill(s, 0, b.kvs[s])
    q = torch.full((41, 4, 64), 1.0, device=DEV).to(DT[dtype])
    _check(b, q, scale=0.25)
    _check(b, q, scale=-0.25)
    _check(b, q, scale=0.0)


def test_attention_rows_do_not_depend_on_the_batch():
    """Every sequence alone gives the bits it has in the batch (16- and 32-bit types,
    one, few and many new tokens)."""
    for dtype in ("f32", "bf16"):
        news, kvs = [1, 3, 70, 1, 200], [900, 40, 333, 2500, 1000]
        b = Batch(dtype, 64, 2, 16, news, kvs, seed=5)
        q = (2.0 * _rand(_gen(6), sum(news), 8, 64)).to(DT[dtype])
        out, lse = b.cache.attend(b.chunks, q, return_lse=True, window=0)
        again = b.cache.attend(b.chunks, q)
        assert torch.equal(out, again)
        t = 0
        for s, n in enumerate(news):
            c = paged.Chunks(torch.tensor([0, n], dtype=torch.int32, device=DEV), b.kv_len[s:s + 1], b.tab[s:s + 1],
                             max_new=n, max_kv=kvs[s])
            o, l1 = b.cache.attend(c, q[t:t + n], return_lse=True)
            assert torch.equal(o, out[t:t + n]) and torch.equal(l1, lse[:, t:t + n])
            t += n


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_ignores_what_its_mask_hides(dtype):
    """NaN and infinities in keys and values that a row does not see (later tokens of its own
    chunk, keys before its window) do not reach it."""
    for n, G in ((1, 2), (4, 2), (64, 2)):
        L, w = 300, 100
        b = Batch(dtype, 64, 2, 16, [n], [L], seed=7)
        q = (2.0 * _rand(_gen(8), n, 2 * G, 64)).to(DT[dtype])
        want, _ = b.ref(q, 0.125, w)
        bad_k, bad_v = float("nan"), float("inf")
        page, slot = b.slots(0, 0, L - n + 1 - w)  # before every window
        b.cache.k[page, slot], b.cache.v[page, slot] = bad_k, bad_v
        if n > 1:  # the last token's key and value: only the last row sees them
            page, slot = b.slots(0, L - 1, L)
            b.cache.k[page, slot], b.cache.v[page, slot] = bad_v, bad_k
        out = b.cache.attend(b.chunks, q, window=w)
        rows = slice(0, max(1, n - 1))
        assert torch.isfinite(out[rows]).all()
        vmax = b.V[0].abs().max().item()
        assert (out[rows].double() - want[rows]).abs().max().item() <= ATT_TOL[dtype] * vmax
        if n > 1:
            assert torch.isnan(out[-1]).any()


def test_attention_table_entries_before_the_window_are_not_read():
    b = Batch("bf16", 64, 2, 16, [1, 20], [400, 400], seed=11)
    q = _rand(_gen(12), 21, 4, 64).bfloat16()
    want = b.cache.attend(b.chunks, q, window=50)
    b.tab[0, : (400 - 50) // 16] = -1
    b.tab[1, : (400 - 20 - 50) // 16] = 1 << 30
    assert torch.equal(b.cache.attend(b.chunks, q, window=50), want)
    b.cache.check_status()


@pytest.mark.parametrize("n", [1, 30])
def test_attention_page_out_of_range_is_unseen_and_reported(n):
    b = Batch("f32", 64, 1, 16, [n], [200], seed=13)
    q = _rand(_gen(14), n, 2, 64)
    b.tab[0, 3] = 1 << 28  # positions 48 .. 63
    out = b.cache.attend(b.chunks, q)
    keep = torch.cat((torch.arange(48), torch.arange(64, 200))).to(DEV)
    for i in range(n):
        k = keep[keep <= 200 - n + i]
        for h in range(2):
            p = torch.softmax(b.K[0][k, 0].double() @ q[i, h].double() / 8, 0)
            assert ((p @ b.V[0][k, 0].double()) - out[i, h]).abs().max().item() < 1e-4
    with pytest.raises(RuntimeError, match="status 0x20"):
        b.cache.check_status()


def test_attention_lengths_outside_their_bounds_are_left_out():
    b = Batch("f32", 32, 1, 16, [1, 1, 1], [50, 60, 70], seed=15)
    q = _rand(_gen(16), 3, 1, 32)
    want, _ = b.ref(q, 32 ** -0.5, 0)
    out = torch.full_like(q, 7.0)
    b.cache.attend(b.make_chunks(max_kv=60), q, out=out)  # the third is longer than its bound
    assert (out[:2].double() - want[:2]).abs().max().item() < 1e-4 and (out[2] == 7.0).all()
    with pytest.raises(RuntimeError, match="status"):
        b.cache.check_status()


def test_attention_far_offsets():
    """Pages whose element offset passes 2^32."""
    P, Hkv, hd = 64, 8, 128
    per = P * Hkv * hd
    n_pages = (1 << 32) // per + 20
    k = torch.empty(n_pages, P, Hkv, hd, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    b = Batch("bf16", hd, Hkv, P, [1, 40], [300, 200], seed=17)
    tab = torch.full_like(b.tab, -1)
    at = n_pages - 12
    for s in range(2):
        for blk in range(-(-b.kvs[s] // P)):
            src = int(b.table[s, blk])
            k[at], v[at] = b.cache.k[src], b.cache.v[src]
            tab[s, blk] = at
            at += 1
    q = (2.0 * _rand(_gen(18), 41, 16, hd)).bfloat16()
    want, wl = b.cache.attend(b.chunks, q, return_lse=True)
    far = paged.PagedKV(k, v)
    c = paged.Chunks(b.q_start, b.kv_len, tab, max_new=40, max_kv=300)
    out, lse = far.attend(c, q, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    # and the append reaches them
    kn, vn = _rand(_gen(1), 41, Hkv, hd).bfloat16(), _rand(_gen(2), 41, Hkv, hd).bfloat16()
    far.append(c, kn, vn)
    pos = torch.arange(160, 200, device=DEV)
    assert torch.equal(k[tab[1][pos // P].long(), pos % P], kn[1:])
    far.check_status()


def test_attention_on_a_side_stream_and_strided_rows():
    b = Batch("f32", 64, 2, 16, [1, 30], [600, 90], seed=19)
    wide = _rand(_gen(20), 31, 5 * 64 + 4)
    q = wide[:, 4:4 + 4 * 64].unflatten(1, (4, 64))
    want, _ = b.ref(q, 0.125, 0)
    buf = torch.zeros(31, 6 * 64, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.cache.attend(b.chunks, q, out=buf[:, 64:320].unflatten(1, (4, 64)))
    s.synchronize()
    assert (buf[:, 64:320].unflatten(1, (4, 64)).double() - want).abs().max().item() < 1e-4
    assert (buf[:, :64] == 0).all() and (buf[:, 320:] == 0).all()


def test_attention_in_a_cuda_graph():
    b = Batch("bf16", 64, 2, 16, [1, 1], [600, 90], seed=21)
    q = _rand(_gen(22), 2, 4, 64).bfloat16()
    want = b.cache.attend(b.chunks, q)
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.cache.attend(b.chunks, q, out=out)
        s.synchronize()
        out.zero_()
        with torch.cuda.graph(g, stream=s):
            b.cache.attend(b.chunks, q, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---- append -------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,dims,il,P,layout", [(32, 8, False, 16, "nhd"), (64, 16, False, 7, "hnd"), (128, 128, True, 64, "nhd"),
                                                  (64, 64, True, 1, "pair"), (128, 6, False, 24, "hnd")])
def test_append_writes_pages_and_rotates(dtype, hd, dims, il, P, layout):
    news, kvs = [1, 0, 5, 90, 33], [40, 12, 5, 300, 64]
    b = Batch(dtype, hd, 2, P, news, kvs, seed=hd + dims, layout=layout)
    g, T, H = _gen(5), sum(news), 6
    cos, sin = _table(512, dims)
    rot = paged.Rotary(cos, sin, il)
    rows = _rand(g, T, (H + 4) * hd).to(DT[dtype])
    q, k, v = (x.unflatten(1, (-1, hd)) for x in rows.split([H * hd, 2 * hd, 2 * hd], 1))
    k0, v0 = b.cache.k.clone(), b.cache.v.clone()
    qr = b.cache.append(b.chunks, k, v, rotary=rot, q=q)
    pos = torch.cat([torch.arange(L - n, L) for n, L in zip(news, kvs)]).to(DEV)
    assert torch.equal(qr, paged.rope(q, rot, pos))
    assert (qr.double() - _rot_ref(q, cos, sin, pos, il)).abs().max().item() <= \
        ROT_TOL[dtype] * math.sqrt(2) * q.abs().max().item()
    kr, t = paged.rope(k, rot, pos), 0
    for s, (n, L) in enumerate(zip(news, kvs)):
        if n:
            page, slot = b.slots(s, L - n, L)
            k0[page, slot], v0[page, slot] = kr[t:t + n], v[t:t + n]
        t += n
    bits = lambda x: x.contiguous().view(torch.int32 if dtype == "f32" else torch.int16)  # noqa: E731
    assert torch.equal(bits(b.cache.k), bits(k0)) and torch.equal(bits(b.cache.v), bits(v0))  # and nothing else
    # given positions, queries in place, and no rotation at all
    other = torch.randint(0, 512, (T,), generator=g, device=DEV)
    want = paged.rope(q, rot, other)
    b.cache.append(b.chunks, k, v, rotary=rot, q=q, positions=other, q_out=q)
    assert torch.equal(q, want)
    b.cache.append(b.chunks, k, v)
    page, slot = b.slots(3, 210, 300)
    assert torch.equal(b.cache.k[page, slot], k[6:96])
    b.cache.check_status()


def test_append_skips_and_reports_what_has_no_place():
    b = Batch("f32", 32, 1, 16, [2, 3, 1], [30, 2, 20], seed=2)  # the second has one token too many
    cos, sin = _table(25, 16)
    rot = paged.Rotary(cos, sin)
    b.tab[2, 1] = b.cache.k.shape[0]  # position 19's page does not exist
    k, v, q = (_rand(_gen(i), 6, 1, 32) for i in (1, 2, 3))
    before = b.cache.k.clone()
    qr = b.cache.append(b.chunks, k, v, rotary=rot, q=q)
    assert torch.isnan(qr[:2]).all()   # positions 28, 29 are outside the table
    assert torch.isnan(qr[2]).all()    # position -1
    assert torch.isfinite(qr[3:]).all()
    page, slot = b.slots(1, 0, 2)
    before[page, slot] = paged.rope(k[3:5], rot, torch.tensor([0, 1], device=DEV))
    assert torch.equal(torch.nan_to_num(b.cache.k, 9.0), torch.nan_to_num(before, 9.0))
    with pytest.raises(RuntimeError, match="status 0x20"):
        b.cache.check_status()


def test_chunked_appends_and_attention_equal_one_pass():
    """A sequence fed in pieces of 1, 7, 64 and 28 tokens gives what one piece of 100 gives
    (each against the 64-bit reference)."""
    g, hd, H, Hkv = _gen(31), 64, 4, 2
    k, v, q = _rand(g, 100, Hkv, hd), _rand(g, 100, Hkv, hd), 2 * _rand(g, 100, H, hd)
    cos, sin = _table(128, 16)
    rot = paged.Rotary(cos, sin)
    outs = []
    for pieces in ([100], [1, 7, 64, 28]):
        cache = paged.PagedKV.empty(12, 16, Hkv, hd)
        alloc = paged.PageAllocator(1, 12, 16, 128, DEV)
        t, ys = 0, []
        for n in pieces:
            c = alloc.extend([n])
            qr = cache.append(c, k[t:t + n], v[t:t + n], rotary=rot, q=q[t:t + n])
            ys.append(cache.attend(c, qr))
            t += n
        outs.append(torch.cat(ys))
        cache.check_status()
    pos = torch.arange(100, device=DEV)
    kr, qr = _rot_ref(k, cos, sin, pos, False), _rot_ref(q, cos, sin, pos, False)
    x = torch.einsum("ihd,jhd->hij", qr, kr.repeat_interleave(2, 1)) / 8
    x.masked_fill_(torch.ones(100, 100, dtype=torch.bool, device=DEV).triu(1), -math.inf)
    want = torch.einsum("hij,jhd->ihd", torch.softmax(x, 2), v.double().repeat_interleave(2, 1))
    for o in outs:
        assert (o.double() - want).abs().max().item() <= ATT_TOL["f32"] * v.abs().max().item()


# ---- refusals ------------------------------------------------------------------


def test_refusals():
    b = Batch("f32", 64, 2, 16, [1], [40], seed=1)
    q = _rand(_gen(1), 1, 4, 64)
    cos, sin = _table(64, 16)
    rot = paged.Rotary(cos, sin)
    with pytest.raises(ValueError):
        b.cache.attend(b.chunks, q.double())
    with pytest.raises(ValueError):
        b.cache.attend(b.chunks, q[:, :3])            # heads not a multiple
    with pytest.raises(ValueError):
        b.cache.attend(b.chunks, q.cpu())
    with pytest.raises(ValueError):
        b.cache.attend(b.chunks, _rand(_gen(1), 4, 1, 64).transpose(0, 1)[:, ::2])  # heads apart
    with pytest.raises(RuntimeError):
        b.cache.attend(b.chunks, q, window=-1)
    with pytest.raises(RuntimeError):                  # rows not on 16 bytes
        b.cache.attend(b.chunks, _rand(_gen(1), 260)[1:257].view(1, 4, 64))
    with pytest.raises(ValueError):
        b.cache.append(b.chunks, q, q)                 # wrong head count
    with pytest.raises(ValueError):
        paged.PagedKV(b.cache.k, b.cache.v.half())
    with pytest.raises(ValueError):
        paged.Rotary(cos.half(), sin.half())
    with pytest.raises(RuntimeError):
        paged.rope(_rand(_gen(1), 1, 1, 8), rot, torch.zeros(1, dtype=torch.int64, device=DEV))  # dims > head
    with pytest.raises(ValueError):
        paged.rope(q, rot, torch.zeros(1, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError):                  # head size without a kernel
        p = paged.PagedKV.empty(2, 16, 1, 96)
        p.attend(b.chunks, _rand(_gen(1), 1, 1, 96))
    with pytest.raises(ValueError):
        b.cache.attend(b.make_chunks(max_kv=500), q)   # the table is shorter
    # nothing to do is not an error
    c0 = paged.Chunks(torch.zeros(2, dtype=torch.int32, device=DEV), b.kv_len, b.tab, max_new=0, max_kv=40)
    assert b.cache.attend(c0, q[:0]).shape == (0, 4, 64)
    assert b.cache.append(c0, q[:0, :2], q[:0, :2]) is None
    assert paged.rope(q[:0], rot, torch.zeros(0, dtype=torch.int64, device=DEV)).shape == (0, 4, 64)
    b.cache.check_status()


def test_short_workspace_is_refused():
    import ctypes

    b = Batch("f32", 64, 2, 16, [1], [4000], seed=1)
    q = _rand(_gen(1), 1, 4, 64)
    L = _lib.lib()
    b.cache._chunks(b.chunks, 1)
    need = L.altxs_paged_attention_workspace_bytes(b.cache._ref, b.chunks._ref, 4, 0)
    rc = L.altxs_paged_attention(b.cache._ref, b.chunks._ref, 4, ctypes.c_float(0.1), 0, q.data_ptr(), 256, q.data_ptr(), 256,
                                 None, None, need - 1, None)
    assert rc == _lib.ALTXS_ENOSPC


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_attention_ignores_huge_values_that_its_mask_hides(dtype, hd):
    """Finite values near the type's end in keys and values that only some rows see (later tokens
    of the chunk, keys before the later rows' windows) leave the other rows as they are."""
    big = torch.finfo(DT[dtype]).max
    for n, G in ((1, 2), (4, 2), (64, 2), (150, 2)):
        L, w = 400, 180
        b = Batch(dtype, hd, 2, 16, [n], [L], seed=21)
        q = (2.0 * _rand(_gen(22), n, 2 * G, hd)).to(DT[dtype])
        want, _ = b.ref(q, hd ** -0.5, w)
        first, half = L - n - w + 1, n // 2  # row i sees [first + i, L - n + i]
        for p0, p1 in ((0, first + half), (L - n + half + 1, L)):
            page, slot = b.slots(0, max(p0, 0), p1)
            b.cache.k[page, slot], b.cache.v[page, slot] = big, -big
        out = b.cache.attend(b.chunks, q, window=w)
        vmax = b.V[0].abs().max().item()
        assert (out[half].double() - want[half]).abs().max().item() <= ATT_TOL[dtype] * vmax
        b.cache.check_status()


@pytest.mark.parametrize("n", [1, 4, 64])
def test_attention_scales_of_keys_and_values(n):
    """fp32 keys 2^40 below and queries 2^40 above 1, values near the type's end: as if none were scaled."""
    b = Batch("f32", 64, 2, 16, [n], [300], seed=23)
    q = 2.0 * _rand(_gen(24), n, 4, 64)
    want, wl = b.ref(q, 0.125, 0)
    b.cache.k.mul_(2.0 ** -40)
    b.cache.v.mul_(2.0 ** 120)
    out, lse = b.cache.attend(b.chunks, q * 2.0 ** 40, return_lse=True)
    vmax = b.V[0].abs().max().item()
    assert (out.double() * 2.0 ** -120 - want).abs().max().item() <= ATT_TOL["f32"] * vmax
    assert (lse.double() - wl).abs().max().item() <= LSE_TOL


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 4, 64, 300])
def test_attention_of_a_nan_query(dtype, n):
    """A query of NaN makes its own row NaN, output and sum, and no other."""
    b = Batch(dtype, 64, 2, 16, [n], [4000], seed=25)
    q = (2.0 * _rand(_gen(26), n, 4, 64)).to(DT[dtype])
    want, wl = b.cache.attend(b.chunks, q, return_lse=True)
    q[n // 2, 1] = float("nan")
    out, lse = b.cache.attend(b.chunks, q, return_lse=True)
    assert torch.isnan(out[n // 2, 1]).all() and torch.isnan(lse[1, n // 2])
    out[n // 2, 1], lse[1, n // 2] = want[n // 2, 1], wl[1, n // 2]
    assert torch.equal(out, want) and torch.equal(lse, wl)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_windows_beyond_the_cache_see_everything(dtype):
    news, kvs = [1, 20, 8, 300], [700, 500, 3, 1300]
    b = Batch(dtype, 64, 2, 16, news, kvs, seed=27)
    q = _rand(_gen(28), sum(news), 4, 64).to(DT[dtype])
    want = b.cache.attend(b.chunks, q)
    for w in (1300, 2000, 2 ** 31 - 1):
        assert torch.equal(b.cache.attend(b.chunks, q, window=w), want)
    b.cache.check_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_a_pool_of_one_page(dtype):
    """The stride over a single page is never taken, whatever it is."""
    b = Batch(dtype, 64, 2, 64, [40], [50], seed=29, spare=0)
    q = _rand(_gen(30), 40, 4, 64).to(DT[dtype])
    want = b.cache.attend(b.chunks, q)
    k, v = (torch.as_strided(x, x.shape, (0, *x.stride()[1:])) for x in (b.cache.k, b.cache.v))
    assert torch.equal(paged.PagedKV(k, v).attend(b.chunks, q), want)


@pytest.mark.parametrize("heads", [2, 40])
def test_sequences_above_a_bound_of_no_new_tokens_are_reported(heads):
    b = Batch("bf16", 64, 1, 16, [3], [50], seed=31)
    q = _rand(_gen(32), 3, heads, 64).bfloat16()
    b.cache.attend(b.make_chunks(max_new=0), q)
    with pytest.raises(RuntimeError):
        b.cache.check_status()


def test_lengths_beyond_the_limits_are_refused():
    """max_kv and max_new above 2^30 (the pools' pages would cover them): no kernel runs."""
    k, v = (torch.empty((1, 1 << 16, 1, 32), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cache = paged.PagedKV(k, v)
    table = torch.zeros(1, 1 << 15, dtype=torch.int32, device=DEV)
    one = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    q = torch.zeros((1, 1, 32), dtype=torch.bfloat16, device=DEV)
    for max_new, max_kv in ((1, 2 ** 30 + 1), (2 ** 30 + 1, 64)):
        c = paged.Chunks(one, one[1:], table, max_new=max_new, max_kv=max_kv)
        with pytest.raises(RuntimeError):
            cache.attend(c, q)
        with pytest.raises(RuntimeError):
            cache.append(c, q, q)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_many_rows_that_see_nothing(dtype):
    """Far more new tokens than positions: thousands of blocks of rows without a key between a few that have some."""
    n, L = 40000, 300
    b = Batch(dtype, 32, 4, 16, [n], [L], seed=35)
    q = torch.zeros(n, 16, 32, dtype=DT[dtype], device=DEV)
    q[n - L:] = (2.0 * _rand(_gen(36), L, 16, 32)).to(DT[dtype])
    out, lse = b.cache.attend(b.chunks, q, return_lse=True)
    b.cache.check_status()
    assert not out[:n - L].any() and torch.isneginf(lse[:, :n - L]).all()
    c = paged.Chunks(torch.tensor([0, L], dtype=torch.int32, device=DEV), b.kv_len, b.tab, max_new=L, max_kv=L)
    tail, tl = b.cache.attend(c, q[n - L:], return_lse=True)
    want, wl = Batch(dtype, 32, 4, 16, [L], [L], seed=35).ref(q[n - L:], 32 ** -0.5, 0)
    vmax = b.V[0].abs().max().item()
    for o, l1 in ((out[n - L:], lse[:, n - L:]), (tail, tl)):
        assert (o.double() - want).abs().max().item() <= ATT_TOL[dtype] * vmax
        assert (l1.double() - wl).abs().max().item() <= LSE_TOL


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kv", [20, 150])
def test_attention_of_many_short_sequences(dtype, kv):
    """Hundreds of chunks of one or two key tiles each: several in a row for every block."""
    n = 450
    b = Batch(dtype, 64, 2, 16, [20 - (s % 3) for s in range(n)], [kv + (s % 7) for s in range(n)], seed=37)
    q = (2.0 * _rand(_gen(38), sum(b.news), 4, 64)).to(DT[dtype])
    _check(b, q)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("G", [1, 4, 16])
def test_attention_of_a_padded_token_buffer(dtype, G):
    """A buffer of n_seqs x max_new rows of which the sequences own fewer: every sequence is computed, short ones
    included, and the rows of no sequence stay as they are."""
    news, kvs, pad = [32, 1, 1, 0, 2, 32], [300, 70, 5, 9, 900, 600], 6 * 32
    b = Batch(dtype, 64, 2, 16, news, kvs, seed=41)
    q = (2.0 * _rand(_gen(42), pad, 2 * G, 64)).to(DT[dtype])
    T = sum(news)
    out = torch.full_like(q, 7.0)
    b.cache.attend(b.chunks, q, out=out)
    _, lse = b.cache.attend(b.chunks, q, return_lse=True)
    want, wl = b.ref(q, 0.125, 0)
    vmax = max(v.abs().max().item() for v in b.V if v.numel())
    assert (out[:T].double() - want[:T]).abs().max().item() <= ATT_TOL[dtype] * vmax
    assert (lse[:, :T].double() - wl[:, :T]).abs().max().item() <= LSE_TOL
    assert (out[T:] == 7.0).all()
    b.cache.check_status()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("n", [2, 4, 7, 8])
def test_attention_keeps_what_every_row_sees(dtype, hd, n):
    """A NaN and an infinity among the values that all rows see, next to positions that only some see, reach
    every row; one in the last token's value reaches the last row alone."""
    L = 300
    b = Batch(dtype, hd, 2, 16, [n], [L], seed=43)
    q = (0.1 * _rand(_gen(44), n, 4, hd)).to(DT[dtype])  # even weights: none of them is 0
    for window in (0, 150):
        want, _ = b.ref(q, hd ** -0.5, window)
        first = L - window if window else 0  # what the last row, so every row, sees begins here
        for p, c, x in ((L - n - 1, 3, float("nan")), (L - n, 5, float("inf")), (first + 1, 7, -float("inf")),
                        (L - 1, 9, float("inf"))):
            page, slot = b.slots(0, p, p + 1)
            b.cache.v[page, slot, :, c] = x
        out = b.cache.attend(b.chunks, q, window=window).double()
        assert torch.isnan(out[:, :, 3]).all()
        assert (out[:, :, 5] == math.inf).all() and (out[:, :, 7] == -math.inf).all()
        assert torch.isfinite(out[:-1, :, 9]).all() and (out[-1, :, 9] == math.inf).all()
        rest = [c for c in range(hd) if c not in (3, 5, 7, 9)]
        vmax = b.V[0].abs().max().item()
        assert (out - want)[:, :, rest].abs().max().item() <= ATT_TOL[dtype] * vmax
        b.fill(0, 0, L)
    b.cache.check_status()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,G", [(1, 2), (4, 4), (20, 1), (20, 16)])
def test_attention_of_a_long_context_behind_one_key(dtype, n, G):
    """One key takes all but 2^-25.5 of each of 60000 others: those weigh 0.13 % together.  Relative error of their
    part: p rounded once (2^-11, and 2^-10.5 where fp16 has left its normal range; 2^-8 for bf16), the result once."""
    L = 60000
    b = Batch(dtype, 64, 1, 64, [n], [L], seed=45)
    b.K[0].zero_()
    b.V[0].fill_(1.0)
    b.K[0][0, 0, 0], b.V[0][0] = 1131 / 256 if dtype == "f16" else 4.40625, 0.0
    b.fill(0, 0, L)
    q = torch.zeros(n, G, 64, device=DEV).to(DT[dtype])
    q[:, :, 0] = 4.0
    want, wl = b.ref(q, 1.0, 0)
    out, lse = b.cache.attend(b.chunks, q, scale=1.0, return_lse=True)
    assert 1e-3 < want.min().item() and want.max().item() < 2e-3
    assert ((out.double() - want) / want).abs().max().item() <= {"f16": 2.0 ** -9, "bf16": 2.0 ** -7}[dtype]
    assert (lse.double() - wl).abs().max().item() <= LSE_TOL


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_needs_zeros_in_its_counters_alone(dtype):
    """The rest of a workspace may hold anything: splits of few and of many rows, and more counters than the
    caller zeroes."""
    b = Batch(dtype, 64, 4, 64, [1, 40], [4000, 6000], seed=47)
    n = _lib.PAGED_COUNTER_BYTES // 32 + 1  # sequences, on the same pages, of four heads: counters beyond the bound
    one = Batch(dtype, 64, 4, 64, [1], [513], seed=48)
    many = paged.Chunks(torch.arange(n + 1, dtype=torch.int32, device=DEV), one.kv_len.repeat(n), one.tab.repeat(n, 1),
                        max_new=1, max_kv=513)
    for cache, chunks, rows in ((b.cache, b.chunks, 41), (one.cache, many, n)):
        q = (2.0 * _rand(_gen(49), rows, 8, 64)).to(DT[dtype])
        want = cache.attend(chunks, q)
        (ws,) = cache._ws.values()
        assert ws.numel() > _lib.PAGED_COUNTER_BYTES
        ws.fill_(0xff)
        ws[:_lib.PAGED_COUNTER_BYTES].zero_()
        for _ in range(2):
            assert torch.equal(cache.attend(chunks, q), want)
        assert torch.isfinite(want).all()
        cache.check_status()


def test_graphs_keep_their_workspaces():
    """Two graphs from one stream whose first call is the first's capture; then larger calls on that stream, other
    tensors in what memory is free, and replays in both orders and on another stream."""
    b = Batch("bf16", 64, 2, 16, [1, 40, 1], [3000, 5000, 90], seed=51)
    q = [(2.0 * _rand(_gen(52 + i), 42, 4, 64)).bfloat16() for i in range(2)]
    want = [b.cache.attend(b.chunks, x) for x in q]
    big = Batch("bf16", 64, 2, 16, [1] * 8 + [300], [9000] * 9, seed=53)
    bq = _rand(_gen(54), 308, 4, 64).bfloat16()
    bw = big.cache.attend(big.chunks, bq)
    cache = paged.PagedKV(b.cache.k, b.cache.v)
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, outs = [], [torch.zeros_like(x) for x in want]
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for x, o in zip(q, outs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                cache.attend(b.chunks, x, out=o)
            graphs.append(g)
        assert torch.equal(cache.attend(b.chunks, q[0]), want[0])  # before any replay
        far = paged.PagedKV(big.cache.k, big.cache.v)
        far._ws = cache._ws  # (the same stream's)
        assert torch.equal(far.attend(big.chunks, bq), bw)
        junk = [torch.full((1 << 20,), 0xff, dtype=torch.uint8, device=DEV) for _ in range(32)]
        s.synchronize()
    for order in ((1, 0), (0, 1), (1, 1), (0, 0)):
        for i in order:
            outs[i].zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(other):
                graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])
    assert all((j == 0xff).all() for j in junk)
    cache.check_status()


def test_inputs_with_a_history_are_refused():
    """No call records a gradient: rather than lose one in silence it raises, unless gradients are off."""
    b = Batch("f32", 64, 2, 16, [1], [40], seed=55)
    q, kv = _rand(_gen(56), 1, 4, 64), _rand(_gen(57), 1, 2, 64)
    rot, pos = paged.Rotary(*_table(64, 16)), torch.tensor([39], device=DEV)
    g = lambda x: x.clone().requires_grad_()  # noqa: E731
    for call in (lambda f: paged.rope(f(q), rot, pos), lambda f: paged.rope_backward(f(q), rot, pos),
                 lambda f: b.cache.append(b.chunks, f(kv), kv), lambda f: b.cache.append(b.chunks, kv, f(kv)),
                 lambda f: b.cache.append(b.chunks, kv, kv, q=f(q)), lambda f: b.cache.attend(b.chunks, f(q))):
        with pytest.raises(RuntimeError, match="gradient"):
            call(g)
        with torch.no_grad():
            call(g)
        call(torch.clone)
    b.cache.check_status()


@pytest.mark.parametrize("given", [False, True])
def test_append_without_rotation_copies_every_query(given):
    """Whatever a token's position, its cache's or a given one: queries of sequences are copied, rows of no sequence
    are left."""
    b = Batch("f32", 32, 1, 16, [5], [2], seed=59)  # cache positions -3 .. 1
    k, v, q = _rand(_gen(1), 7, 1, 32), _rand(_gen(2), 7, 1, 32), _rand(_gen(3), 7, 2, 32)
    pos = torch.tensor([-3, -2, -1, 0, -2, -2, 7], device=DEV) if given else None
    out = torch.full_like(q, 7.0)
    b.cache.append(b.chunks, k, v, q=q, q_out=out, positions=pos)
    assert torch.equal(out[:5], q[:5]) and (out[5:] == 7.0).all()
    page, slot = b.slots(0, 0, 2)
    assert torch.equal(b.cache.k[page, slot], k[3:5]) and torch.equal(b.cache.v[page, slot], v[3:5])
    with pytest.raises(RuntimeError, match="status 0x20"):  # three of them have no place
        b.cache.check_status()


def test_windows_beyond_32_bits_see_everything():
    b = Batch("bf16", 64, 2, 16, [1, 20], [70, 50], seed=61)
    q = _rand(_gen(62), 21, 4, 64).bfloat16()
    want = b.cache.attend(b.chunks, q)
    for w in (2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1):
        assert torch.equal(b.cache.attend(b.chunks, q, window=w), want)
    with pytest.raises(RuntimeError):
        b.cache.attend(b.chunks, q, window=-2 ** 32 + 5)
    b.cache.check_status()


@pytest.mark.parametrize("n", [1, 40])
def test_strides_over_one_page_slot_or_head_do_not_count(n):
    """They are never taken: any value will do, also one that is no multiple of 16 bytes, or another in v than in k."""
    q = _rand(_gen(64), n, 4, 64).bfloat16()
    for P, kv, Hkv in ((64, 50, 2), (1, 45, 2), (16, 60, 1)):  # one page, one slot a page, one head
        b = Batch("bf16", 64, Hkv, P, [n], [kv], seed=63, spare=0)
        want = b.cache.attend(b.chunks, q)
        pools = []
        for x, odd in ((b.cache.k, 77), (b.cache.v, 99)):
            pools.append(torch.as_strided(x, x.shape, [odd if m == 1 else s for m, s in zip(x.shape, x.stride())]))
        cache = paged.PagedKV(*pools)
        assert torch.equal(cache.attend(b.chunks, q), want)
        kn, vn = _rand(_gen(65), n, Hkv, 64).bfloat16(), _rand(_gen(66), n, Hkv, 64).bfloat16()
        cache.append(b.chunks, kn, vn)
        page, slot = b.slots(0, kv - n, kv)
        assert torch.equal(b.cache.k[page, slot], kn) and torch.equal(b.cache.v[page, slot], vn)
        cache.check_status()
    with pytest.raises(ValueError):
        paged.PagedKV(b.cache.k, b.cache.v.transpose(0, 1))
