"""What the paged-cache operators are measured on: rotary positions, the append of
new keys and values to a paged cache, and the attention of new tokens over it.

Three operators, by the case's "op":

rope    y = R(position) x on the first ``dims`` channels of every head, for x
        [tokens][heads][hd]; "backward" is the product with the transpose.
append  the new tokens' keys, rotated, and values go to their pages, and the
        queries are rotated in the same pass; returns the pools and the queries.
attend  softmax attention of each sequence's new tokens (the last ``new`` of its
        ``kv`` positions) over the cache, causal, optionally within a window.

Lengths are functions of the case alone; the values, and which page holds what,
come from the seed.  ``own`` False: the plain forms, in torch's elementary
operations and 32 bits; ``own`` True: altxs_b200.paged.
"""

from __future__ import annotations

import math
import random

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ES = {"f32": 4, "bf16": 2, "f16": 2}
_TABLE = 1 << 17     # positions of the rotary tables
_GAIN = 3.0          # the queries' gain after their RMS norm (the models here start at 5)
_MAX_SCORES = 1.45e9  # entries of the plain form's largest score matrix


def _case(name, op, dtype, hd, heads, kv_heads, **more):
    return {"name": name, "op": op, "dtype": dtype, "hd": hd, "heads": heads, "kv_heads": kv_heads, **more}


def listed():
    return [
        # one symbol of 8 streams of the 33M model: its q and k heads side by side, 16 of 64 channels
        _case("rope step f32", "rope", "f32", 64, 16, 0, tokens=8, dims=16, interleaved=False, backward=False, ld_pad=512),
        # the gradient of a training window's rotated q and k heads of the same model
        _case("rope window backward", "rope", "f32", 64, 16, 0, tokens=2047, dims=16, interleaved=False, backward=True, ld_pad=512),
        # a long prefill of a wider model, whole heads, neighbouring channels paired
        _case("rope prefill bf16", "rope", "bf16", 128, 40, 0, tokens=32768, dims=128, interleaved=True, backward=False, ld_pad=1024),
        # one symbol of 256 streams of the 33M model (the share of one GPU of eight)
        _case("append step f32", "append", "f32", 64, 8, 8, seqs=256, new="1", kv="1..2048", mix=1, page=16, dims=16, interleaved=False),
        # prompts of very different lengths, grouped heads, whole heads rotated
        _case("append prompts bf16", "append", "bf16", 128, 32, 8, seqs=13, new="1..8192", kv="new", mix=2, page=64, dims=128, interleaved=True),
        # one symbol of one stream with its window full: latency
        _case("decode 1 stream f32", "attend", "f32", 64, 8, 8, seqs=1, new="1", kv="2049", mix=3, page=64, window=2048, lse=False),
        # one symbol of 256 streams, windows filling
        _case("decode 256 streams f32", "attend", "f32", 64, 8, 8, seqs=256, new="1", kv="1..2048", mix=4, page=64, window=0, lse=False),
        # three very long contexts, grouped heads
        _case("decode long bf16", "attend", "bf16", 128, 32, 8, seqs=3, new="1", kv="60000..100001", mix=5, page=64, window=0, lse=False),
        # five proposed tokens checked at once in each of 48 streams, sliding window, small pages
        _case("check 5 tokens f16", "attend", "f16", 64, 16, 4, seqs=48, new="5", kv="100..6000", mix=6, page=16, window=1024, lse=True),
        # the encoder's 64-symbol windows of 16 streams over a full context, in the engine's precision
        _case("encode windows f32", "attend", "f32", 64, 8, 8, seqs=16, new="64", kv="2112", mix=7, page=64, window=2048, lse=False),
        # prompts continued in pieces next to streams that decode: ragged, grouped heads
        _case("mixed prompts bf16", "attend", "bf16", 128, 16, 4, seqs=9, new="1|1..1999", kv="new..4500", mix=8, page=32, window=0, lse=True),
        # a long piece of one long prompt
        _case("long piece f16", "attend", "f16", 128, 16, 8, seqs=1, new="4096", kv="20000", mix=9, page=128, window=0, lse=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "append", "attend", "attend", "attend"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    hd = rng.choice((32, 64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
    dims = rng.choice((hd // 4, hd // 2, hd))
    mix = rng.randrange(1, 1 << 20)
    page = rng.choice((16, 24, 32, 64, 128, 256))
    half = rng.random() < 0.5
    if op == "rope":
        most = 160_000_000 // (heads * hd)
        return {"op": op, "dtype": dtype, "hd": hd, "heads": heads, "kv_heads": 0, "tokens": _log_int(rng, 1, min(32768, most)),
                "dims": dims, "interleaved": half, "backward": rng.random() < 0.5, "ld_pad": rng.choice((0, 64, 1024))}
    if op == "append":
        seqs = _log_int(rng, 1, 256)
        new = _log_int(rng, 1, max(1, 16384 // seqs))
        kv = new + _log_int(rng, 1, 2048)
        return {"op": op, "dtype": dtype, "hd": hd, "heads": heads, "kv_heads": kv_heads, "seqs": seqs, "new": "1..%d" % new,
                "kv": "new..%d" % kv, "mix": mix, "page": page, "dims": dims, "interleaved": half}
    kind = rng.choice(("one", "few", "many"))
    new = 1 if kind == "one" else _log_int(rng, 2, 16) if kind == "few" else _log_int(rng, 17, 4096)
    kv = max(new, _log_int(rng, 16, 20000 if kind == "many" else 100000))
    row = kv_heads * hd * 2 * _ES[dtype]
    most = min(256, int(1.6e9 / (kv * row)), int(_MAX_SCORES / (heads * new * kv)),
               int(1.5e11 / (heads * new * kv * hd * (4 if dtype == "f32" else 1))))
    seqs = _log_int(rng, 1, max(1, most))
    if heads * new * kv > _MAX_SCORES:
        kv = max(new, int(_MAX_SCORES / (heads * new)))
    return {"op": op, "dtype": dtype, "hd": hd, "heads": heads, "kv_heads": kv_heads, "seqs": seqs,
            "new": str(new) if rng.random() < 0.5 else "1..%d" % new, "kv": "new..%d" % kv, "mix": mix, "page": page,
            "window": 0 if rng.random() < 0.6 else _log_int(rng, 16, kv), "lse": rng.random() < 0.3}


def _lengths(case):
    """(new, kv) of every sequence; the first sequence has the largest of both."""
    rng = random.Random(case["mix"])
    news, kvs = [], []
    for s in range(case["seqs"]):
        spec = case["new"]
        one, _, spec2 = spec.partition("|")
        if spec2:  # "1|a..b": every other sequence has one token
            spec = one if s % 2 else spec2
        lo, _, hi = spec.partition("..")
        n = int(hi or lo) if s == 0 else rng.randint(int(lo), int(hi or lo))
        lo, _, hi = case["kv"].partition("..")
        hi = hi or lo
        lo = n if lo == "new" else max(n, int(lo))
        hi = n if hi == "new" else max(lo, int(hi))
        news.append(n)
        kvs.append(hi if s == 0 else rng.randint(lo, hi))
    return news, kvs


def _rms(x):
    return x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)


def _tables(dims, device):
    inv = 1.0 / 1e4 ** (torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    a = torch.arange(_TABLE, dtype=torch.float64, device=device)[:, None] * inv.to(device)
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt, hd, H, Hkv = _DT[case["dtype"]], case["hd"], case["heads"], case["kv_heads"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    st = {"case": case}
    if case["op"] == "rope":
        T, wide = case["tokens"], H * hd + case["ld_pad"]
        rows = randn(T, wide).to(dt)  # a row of a fused projection: the heads, then what is not rotated
        st["x"] = rows[:, :H * hd].unflatten(1, (H, hd))
        st["pos"] = torch.randint(0, _TABLE, (T,), generator=gen, device=dev)
        st["cos"], st["sin"] = _tables(case["dims"], dev)
        if own:
            from altxs_b200 import paged

            st["rotary"] = paged.Rotary(st["cos"], st["sin"], case["interleaved"])
        return st
    news, kvs = _lengths(case)
    P, n = case["page"], case["seqs"]
    blocks = [-(-k // P) for k in kvs]
    n_pages = sum(blocks) + 3
    perm = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    # sequence s's blocks are the next blocks[s] entries of the permutation; entries past them name no page
    first = torch.tensor([0] + blocks, device=dev).cumsum(0)[:n, None]
    at = torch.arange(max(blocks), device=dev)[None, :]
    held = at < torch.tensor(blocks, device=dev)[:, None]
    st["table"] = torch.where(held, perm[(first + at).clamp_(max=n_pages - 1)], -1).to(torch.int32)
    st["q_start"] = torch.tensor([0] + news, device=dev).cumsum(0).to(torch.int32)
    st["kv_len"] = torch.tensor(kvs, dtype=torch.int32, device=dev)
    T = sum(news)
    st["k_pool"] = randn(n_pages, P, Hkv, hd).to(dt)  # roughly what a per-head norm leaves
    st["v_pool"] = randn(n_pages, P, Hkv, hd).to(dt)
    st["q"] = (_rms(randn(T, H, hd)) * _GAIN).to(dt)
    st["new"], st["kv"] = max(news), max(kvs)
    if case["op"] == "append":
        qkv = torch.cat((st["q"], _rms(randn(T, Hkv, hd)).to(dt), randn(T, Hkv, hd).to(dt)), 1)
        st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        st["cos"], st["sin"] = _tables(case["dims"], dev)
    if own:
        from altxs_b200 import paged

        st["cache"] = paged.PagedKV(st["k_pool"], st["v_pool"])
        st["chunks"] = paged.Chunks(st["q_start"], st["kv_len"], st["table"], max_new=st["new"], max_kv=st["kv"])
        if case["op"] == "append":
            st["rotary"] = paged.Rotary(st["cos"], st["sin"], case["interleaved"])
    return st


# ---- plain forms -------------------------------------------------------------


def _rotate(x, cos, sin, interleaved, backward=False):
    """x [T][heads][hd] in 32 bits; cos, sin [T][1][dims / 2]."""
    dims = 2 * cos.shape[-1]
    r, rest = x[..., :dims], x[..., dims:]
    if backward:
        sin = -sin
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos + b * sin, b * cos - a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :dims // 2], r[..., dims // 2:]
        r = torch.cat((a * cos + b * sin, b * cos - a * sin), -1)
    return torch.cat((r, rest), -1)


def _rows_of(st):
    """(sequence, position) of every new token."""
    t = torch.arange(st["q"].shape[0], device=st["q"].device)
    seq = torch.bucketize(t, st["q_start"][1:].long(), right=True)
    return seq, st["kv_len"][seq].long() - st["q_start"][seq + 1].long() + t


def _plain_append(st):
    c = st["case"]
    seq, pos = _rows_of(st)
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    page, slot = st["table"][seq, pos // c["page"]].long(), pos % c["page"]
    k = _rotate(st["k"].float(), cos, sin, c["interleaved"])
    st["k_pool"][page, slot] = k.to(st["k_pool"].dtype)
    st["v_pool"][page, slot] = st["v"]
    q = _rotate(st["q"].float(), cos, sin, c["interleaved"]).to(st["q"].dtype)
    return {"k": st["k_pool"], "v": st["v_pool"], "q": q}


def _plain_attend(st):
    c, q = st["case"], st["q"]
    H, Hkv, hd, n = c["heads"], c["kv_heads"], c["hd"], c["seqs"]
    G, Q = H // Hkv, st["new"]
    seq, pos = _rows_of(st)
    off = torch.arange(q.shape[0], device=q.device) - st["q_start"][seq].long()
    qp = torch.zeros(n, Q, H, hd, device=q.device)
    qp[seq, off] = q.float()
    qpos = torch.full((n, Q), -1, device=q.device)
    qpos[seq, off] = pos
    table = st["table"].clamp(min=0).long()
    k = st["k_pool"][table].flatten(1, 2).float().permute(0, 2, 3, 1)  # [n][Hkv][hd][keys]
    v = st["v_pool"][table].flatten(1, 2).float().transpose(1, 2)      # [n][Hkv][keys][hd]
    qp = qp.unflatten(2, (Hkv, G)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [n][Hkv][G * Q][hd]
    s = torch.matmul(qp, k).mul_(1.0 / math.sqrt(hd)).unflatten(2, (G, Q))
    at = torch.arange(s.shape[-1], device=q.device)
    seen = at <= qpos[..., None]
    if c["window"]:
        seen &= at > qpos[..., None] - c["window"]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (G, Q)) / total.clamp(min=1e-30)
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, off].to(q.dtype)
    if not c["lse"]:
        return {"out": out}
    lse = (m + total.log())[..., 0].permute(0, 3, 1, 2).flatten(2, 3)[seq, off] * math.log2(math.e)
    return {"out": out, "lse": lse.T.contiguous()}


def run(st):
    c = st["case"]
    if own:
        from altxs_b200 import paged

        if c["op"] == "rope":
            f = paged.rope_backward if c["backward"] else paged.rope
            return {"y": f(st["x"], st["rotary"], st["pos"])}
        if c["op"] == "append":
            q = st["cache"].append(st["chunks"], st["k"], st["v"], rotary=st["rotary"], q=st["q"])
            return {"k": st["k_pool"], "v": st["v_pool"], "q": q}
        if c["lse"]:
            out, lse = st["cache"].attend(st["chunks"], st["q"], window=c["window"], return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": st["cache"].attend(st["chunks"], st["q"], window=c["window"])}
    if c["op"] == "rope":
        cos, sin = st["cos"][st["pos"]][:, None], st["sin"][st["pos"]][:, None]
        return {"y": _rotate(st["x"].float(), cos, sin, c["interleaved"], c["backward"]).to(st["x"].dtype)}
    return _plain_append(st) if c["op"] == "append" else _plain_attend(st)


# ---- the definition in 64 bits -----------------------------------------------


def _exact_rotation(x, cos, sin, pos, interleaved, backward):
    """Pairs as complex numbers: (a + ib) times e^(-i angle), or its conjugate."""
    dims = 2 * cos.shape[1]
    y = x.double().clone()
    w = torch.complex(cos.double()[pos], (1 if backward else -1) * sin.double()[pos])[:, None, :]
    r = y[..., :dims]
    z = (torch.complex(r[..., 0::2].contiguous(), r[..., 1::2].contiguous()) if interleaved else
         torch.complex(r[..., :dims // 2].contiguous(), r[..., dims // 2:].contiguous())) * w
    if interleaved:
        y[..., 0:dims:2], y[..., 1:dims:2] = z.real, z.imag
    else:
        y[..., :dims // 2], y[..., dims // 2:dims] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return {"y": _exact_rotation(st["x"], st["cos"], st["sin"], st["pos"], case["interleaved"], case["backward"])}
    news, kvs = _lengths(case)
    P, starts = case["page"], [sum(news[:s]) for s in range(len(news))]
    if case["op"] == "append":
        k, v = st["k_pool"].double(), st["v_pool"].double()
        q = torch.empty(st["q"].shape, dtype=torch.float64, device=k.device)
        for s, (n, t0, L) in enumerate(zip(news, starts, kvs)):
            pos = torch.arange(L - n, L, device=k.device)
            rows = slice(t0, t0 + n)
            flat = st["table"][s].long()[pos // P] * P + pos % P
            k.flatten(0, 1)[flat] = _exact_rotation(st["k"][rows], st["cos"], st["sin"], pos, case["interleaved"], False)
            v.flatten(0, 1)[flat] = st["v"][rows].double()
            q[rows] = _exact_rotation(st["q"][rows], st["cos"], st["sin"], pos, case["interleaved"], False)
        return {"k": k, "v": v, "q": q}
    H, Hkv, hd, w = case["heads"], case["kv_heads"], case["hd"], case["window"]
    out = torch.zeros(sum(news), H, hd, dtype=torch.float64, device="cuda")
    lse = torch.zeros(H, sum(news), dtype=torch.float64, device="cuda")
    for s, (n, t0, L) in enumerate(zip(news, starts, kvs)):
        first = max(0, L - n - w + 1) if w else 0  # nothing before it is seen by any row
        pos = torch.arange(first, L, device="cuda")
        page, slot = st["table"][s].long()[pos // P], pos % P
        ks, vs = st["k_pool"][page, slot].double(), st["v_pool"][page, slot].double()
        for r0 in range(0, n, 1024):
            rows = torch.arange(r0, min(n, r0 + 1024), device="cuda")
            age = (L - n + rows)[:, None] - pos[None, :]
            hide = (age < 0) | (age >= w) if w else age < 0
            for h in range(H):
                g = h * Hkv // H
                x = (st["q"][t0 + rows, h].double() @ ks[:, g].T) / math.sqrt(hd)
                x[hide] = -math.inf
                total = torch.logsumexp(x, 1)
                out[t0 + rows, h] = torch.exp(x - total[:, None]) @ vs[:, g]
                lse[h, t0 + rows] = total / math.log(2.0)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def work(case):
    hd, H, Hkv, es = case["hd"], case["heads"], case["kv_heads"], _ES[case["dtype"]]
    if case["op"] == "rope":
        T = case["tokens"]
        return {"bytes": 2 * T * H * hd * es + T * (8 + 4 * case["dims"]), "flops": 3 * T * H * case["dims"]}
    news, kvs = _lengths(case)
    T = sum(news)
    if case["op"] == "append":
        return {"bytes": 2 * T * (H + 2 * Hkv) * hd * es + 4 * T * case["dims"], "flops": 3 * T * (H + Hkv) * case["dims"]}
    w = case["window"] or max(kvs)
    keys = sum(min(L, w + n - 1) for n, L in zip(news, kvs))
    # row i of a sequence sees min(w, L - n + i + 1) keys
    pairs = sum(sum(min(w, L - n + i + 1) for i in range(n)) for n, L in zip(news, kvs))
    return {"bytes": 2 * keys * Hkv * hd * es + 2 * T * H * hd * es + (4 * T * H if case["lse"] else 0),
            "flops": 4 * pairs * H * hd}
