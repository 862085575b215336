"""CPU checks of the paged cache: argument validation runs before any CUDA call,
the page allocator is plain host code, and the rotary tables follow their rules."""

from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

from altxs_b200 import _lib, paged


def _kv(**kw):
    d = dict(k=4096, v=8192, page_stride=16 * 2 * 64, token_stride=2 * 64, head_stride=64, dtype=_lib.F32,
             page_size=16, n_pages=4, n_kv_heads=2, head_dim=64)
    return _lib.PagedKv(**{**d, **kw})


def _ch(**kw):
    d = dict(q_start=4096, kv_len=4096, page_table=4096, table_stride=4, n_seqs=1, n_tokens=1, max_new=1, max_kv=40)
    return _lib.Chunks(**{**d, **kw})


def _attend(kv, ch, H=4, window=0, ldq=256, ws=0, nbytes=0):
    return _lib.lib().altxs_paged_attention(C.byref(kv), C.byref(ch), H, 0.1, window, 4096, ldq, 4096, 256, None, ws,
                                            nbytes, None)


@pytest.mark.parametrize("kv,ch,kw,code", [
    (dict(head_dim=48), {}, {}, _lib.ALTXS_ENOTSUP), (dict(dtype=3), {}, {}, _lib.ALTXS_EINVAL),
    (dict(page_size=0), {}, {}, _lib.ALTXS_EINVAL), (dict(k=4097), {}, {}, _lib.ALTXS_EINVAL),
    (dict(token_stride=130), {}, {}, _lib.ALTXS_EINVAL), (dict(token_stride=32), {}, {}, _lib.ALTXS_EINVAL),
    (dict(dtype=_lib.F16, head_stride=68), {}, {}, _lib.ALTXS_EINVAL), (dict(n_kv_heads=0), {}, {}, _lib.ALTXS_EINVAL),
    ({}, dict(max_kv=65), {}, _lib.ALTXS_EINVAL), ({}, dict(n_seqs=-1), {}, _lib.ALTXS_EINVAL),
    ({}, dict(max_new=-1), {}, _lib.ALTXS_EINVAL), ({}, dict(q_start=None), {}, _lib.ALTXS_EINVAL),
    ({}, {}, dict(H=5), _lib.ALTXS_EINVAL), ({}, {}, dict(H=0), _lib.ALTXS_EINVAL),
    ({}, {}, dict(window=-1), _lib.ALTXS_EINVAL), ({}, {}, dict(ldq=255), _lib.ALTXS_EINVAL),
    ({}, {}, dict(ldq=258), _lib.ALTXS_EINVAL), ({}, dict(n_seqs=0), {}, 0), ({}, dict(n_tokens=0), {}, 0)])
def test_attention_refuses_before_touching_the_device(kv, ch, kw, code):
    assert _attend(_kv(**kv), _ch(**ch), **kw) == code


def test_workspace_sizes():
    L = _lib.lib()
    f = lambda kv, ch, H=4, w=0: L.altxs_paged_attention_workspace_bytes(C.byref(kv), C.byref(ch), H, w)  # noqa: E731
    assert f(_kv(head_dim=48), _ch()) == -1 and f(_kv(), _ch(), H=3) == -1 and f(_kv(), _ch(), w=-1) == -1
    long = _ch(n_seqs=64, n_tokens=64, max_kv=100000, table_stride=10000)
    assert f(_kv(), long) >= f(_kv(), _ch()) >= 0
    # a window and a known total bound it
    assert f(_kv(), long, w=512) <= f(_kv(), long)
    some = _ch(n_seqs=64, n_tokens=64, max_kv=100000, table_stride=10000, total_kv=200000)
    assert f(_kv(), some) <= f(_kv(), long)


def test_rope_and_append_refuse_before_touching_the_device():
    L = _lib.lib()
    r = _lib.RotaryTables(cos=4096, sin=4096, positions=10, dims=16, interleaved=0)

    def rope(dtype=0, T=1, H=2, hd=64, r=r, pos=4096, x=4096, ldx=128, y=8192, ldy=128):
        return L.altxs_rope(dtype, T, H, hd, C.byref(r), pos, 0, x, ldx, y, ldy, None, None)

    bad = lambda **kw: _lib.RotaryTables(**{**dict(cos=4096, sin=4096, positions=10, dims=16, interleaved=0), **kw})  # noqa: E731
    assert rope(dtype=7) == _lib.ALTXS_EINVAL and rope(hd=63) == _lib.ALTXS_EINVAL
    assert rope(hd=514, ldx=2000, ldy=2000) == _lib.ALTXS_ENOTSUP
    assert rope(ldx=127) == _lib.ALTXS_EINVAL and rope(pos=None) == _lib.ALTXS_EINVAL
    assert rope(x=4097) == _lib.ALTXS_EINVAL and rope(x=8192, ldx=256) == _lib.ALTXS_EINVAL
    assert rope(r=bad(dims=66)) == _lib.ALTXS_EINVAL and rope(r=bad(dims=15)) == _lib.ALTXS_EINVAL
    assert rope(r=bad(cos=4100)) == _lib.ALTXS_EINVAL and rope(r=bad(sin=None)) == _lib.ALTXS_EINVAL
    assert rope(T=0) == 0 and rope(H=0, ldx=0, ldy=0) == 0

    def append(kv=_kv(), ch=_ch(), ldk=128, H=4, q=4096, ldq=256, qo=8192, ldqo=256, r=r, k=4096):
        return L.altxs_paged_append(C.byref(kv), C.byref(ch), C.byref(r), None, k, ldk, 8192, 128, H, q, ldq, qo, ldqo,
                                    None)

    assert append(kv=_kv(head_dim=16)) == _lib.ALTXS_ENOTSUP and append(ldk=127) == _lib.ALTXS_EINVAL
    assert append(ldq=255) == _lib.ALTXS_EINVAL and append(qo=None) == _lib.ALTXS_EINVAL
    assert append(qo=4096, ldqo=512) == _lib.ALTXS_EINVAL and append(k=None) == _lib.ALTXS_EINVAL
    assert append(k=4098) == _lib.ALTXS_EINVAL and append(r=bad(dims=128)) == _lib.ALTXS_EINVAL
    assert append(ch=_ch(n_tokens=0)) == 0


def test_page_allocator():
    a = paged.PageAllocator(3, 6, 4, 20, "cpu")
    c = a.extend([5, 0, 1])
    assert c.q_start.tolist() == [0, 5, 5, 6] and c.kv_len.tolist() == [5, 0, 1]
    assert c.struct.max_new == 5 and c.struct.max_kv == 5 and c.struct.total_kv == 6
    held = [p for p in a.table.ravel() if p >= 0]
    assert len(set(held)) == 3 and len(a.free) == 3 and (a.table[1] == -1).all()
    a.extend([3, 0, 0])  # fills the second page: no new one
    assert len(a.free) == 3 and a.len.tolist() == [8, 0, 1]
    before = a.table.copy()
    with pytest.raises(RuntimeError, match="out of pages"):
        a.extend([4, 12, 0])
    with pytest.raises(ValueError, match="max_kv"):
        a.extend([13, 0, 0])
    with pytest.raises(ValueError):
        a.extend([1, 1])
    assert (a.table == before).all() and a.len.tolist() == [8, 0, 1]
    a.extend([9, 0, 0])  # 17 tokens: five pages
    # window 6: the next token (position 17) sees 12 ..: pages of 0-3, 4-7, 8-11 come back
    assert a.trim(0, 6) == 3 and a.trim(0, 6) == 0 and (a.table[0, :3] == -1).all() and (a.table[0, 3:5] >= 0).all()
    a.release(0)
    assert a.len[0] == 0 and len(a.free) == 5 and sorted(a.free + [int(a.table[2, 0])]) == list(range(6))


def test_rope_table_rules():
    n, d, base = 300, 32, 1e4
    p, j = np.arange(n)[:, None], np.arange(0, d, 2)
    w = base ** (-j / d)

    def close(t, w, amp=1.0):
        cos, sin = t
        return max(np.abs(cos.double().numpy() - amp * np.cos(p * w)).max(),
                   np.abs(sin.double().numpy() - amp * np.sin(p * w)).max()) < 2.0 ** -23

    assert close(paged.rope_table(n, d, base, device="cpu"), w)
    assert close(paged.rope_table(n, d, base, scaling="linear", factor=4.0, device="cpu"), w / 4)
    wb = (base * 4.0 ** (d / (d - 2))) ** (-j / d)
    assert wb[0] == 1.0 and abs(wb[-1] * 4 / w[-1] - 1) < 1e-12
    assert close(paged.rope_table(n, d, base, scaling="base", factor=4.0, device="cpu"), wb)
    t = 2048
    turns = t * w / (2 * math.pi)
    wp = np.where(turns > 32, w, np.where(turns < 1, w / 8, 0))
    ramp = (turns - 1) / 31
    mid = (turns <= 32) & (turns >= 1)
    wp[mid] = (w * (ramp + (1 - ramp) / 8))[mid]
    amp = 0.1 * math.log(8.0) + 1
    assert close(paged.rope_table(n, d, base, scaling="parts", factor=8.0, trained=t, device="cpu"), wp, amp)
    assert paged.rope_table(0, 16, device="cpu")[0].shape == (0, 8)
    assert torch.equal(paged.rope_table(5, 2, scaling="base", factor=2.0, device="cpu")[0],
                       paged.rope_table(5, 2, device="cpu")[0])
    for kw in (dict(scaling="parts", factor=2.0), dict(scaling="x"), dict(factor=0.5)):
        with pytest.raises(ValueError):
            paged.rope_table(4, 16, device="cpu", **kw)
    with pytest.raises(ValueError):
        paged.rope_table(4, 15, device="cpu")


@pytest.mark.parametrize("dtype", [_lib.F32, _lib.BF16, _lib.F16])
def test_workspace_covers_short_sequences_of_a_padded_buffer(dtype):
    """A token buffer of n_seqs x max_new rows may hold rows of no sequence, so it says nothing about the
    lengths: the plan for it holds what a buffer of one row less needs."""
    L = _lib.lib()
    size = lambda ch: L.altxs_paged_attention_workspace_bytes(C.byref(_kv(dtype=dtype)), C.byref(ch), 4, 0)  # noqa: E731
    for new in (16, 32):
        c = [_ch(n_seqs=4, n_tokens=4 * new - d, max_new=new, max_kv=100000, table_stride=10000) for d in (1, 0)]
        assert size(c[1]) >= size(c[0]) > 0


def test_a_new_workspace_has_zero_counters():
    for need in (0, 1000, _lib.PAGED_COUNTER_BYTES + 4096):
        ws = paged._workspace(need, torch.device("cpu"))
        assert ws.numel() == max(need, 16) and not ws[:_lib.PAGED_COUNTER_BYTES].any()


def test_a_captured_call_has_a_workspace_of_its_own(monkeypatch):
    """What a graph holds is neither kept for other calls nor replaced by them: a larger call, or a cache whose
    status raised, must not give away memory that a graph still writes."""
    cache = object.__new__(paged.PagedKV)
    cache.device, cache._ws = torch.device("cpu"), {}
    capturing = False
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    eager = cache._workspace_for(1000, 7)
    assert cache._workspace_for(900, 7) is eager and cache._workspace_for(900, 8) is not eager
    capturing = True
    first, second = cache._workspace_for(900, 7), cache._workspace_for(900, 7)
    assert first is not second and first is not eager and not first.any() and cache._ws[7] is eager
    assert cache._workspace_for(900, 9) is not None and 9 not in cache._ws
    capturing = False
    bigger = cache._workspace_for(5000, 7)
    assert cache._ws[7] is bigger and bigger.numel() >= 5000


def test_workspaces_of_growing_streams_are_not_replaced_at_every_step(monkeypatch):
    """256 streams of eight heads of 64, a token at a time from 600 positions on, sized by their total as the allocator
    gives it: the need grows at most steps, the workspace seldom."""
    cache = object.__new__(paged.PagedKV)
    cache.device, cache._ws = torch.device("cpu"), {}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    needs, sizes = [], []
    for step in range(0, 2000, 16):
        ch = _ch(n_seqs=256, n_tokens=256, max_kv=600 + step, table_stride=1000, total_kv=256 * (600 + step))
        needs.append(_lib.lib().altxs_paged_attention_workspace_bytes(C.byref(_kv(n_kv_heads=8)), C.byref(ch), 8, 0))
        sizes.append(cache._workspace_for(needs[-1], 0).numel())
        assert sizes[-1] >= needs[-1] > 0
    assert len(set(needs)) > 50 and len(set(sizes)) <= 5 and sizes[-1] <= 1.5 * needs[-1]
    huge = max(needs[-1] * 100, 1 << 30)
    cache._ws[0] = torch.empty(0, dtype=torch.uint8).new_empty(huge)
    assert cache._workspace_for(huge + 1, 0).numel() <= huge + (64 << 20)


def test_trim_of_a_window_that_sees_everything():
    """Window 0 sees everything, as in attend: nothing comes back; a negative one is refused."""
    a = paged.PageAllocator(1, 6, 4, 20, "cpu")
    a.extend([17])
    before = a.table.copy()
    assert a.trim(0, 0) == 0 and (a.table == before).all() and len(a.free) == 1
    with pytest.raises(ValueError, match="window"):
        a.trim(0, -1)
    assert (a.table == before).all() and a.trim(0, 1) == 4


def _plain_cfg(**kw):
    from altxs_b200.config import ModelConfig

    d = dict(vocab_size=512, num_layers=3, model_dim=128, num_heads=4, num_kv_heads=2, mlp_mult=4.0, rope_dims=16,
             block_size=48, online_retrain_every=64, seed=11, retrain_mode="none")
    return ModelConfig(**{**d, **kw})


def test_the_scorer_refuses_reset_contexts():
    """It scores with a sliding window: a model whose context is rebuilt at every segment costs other bits."""
    from types import SimpleNamespace

    from altxs_b200.scorer import PagedScorer

    with pytest.raises(ValueError, match="context_mode"):
        PagedScorer(SimpleNamespace(cfg=_plain_cfg(context_mode="reset")), 1, 64)


def test_the_scorer_refuses_head_sizes_without_a_kernel():
    """At construction, not in the first append after pages were granted."""
    from types import SimpleNamespace

    from altxs_b200.scorer import PagedScorer

    cfg = _plain_cfg(model_dim=192)  # heads of 48
    cfg.validate()
    with pytest.raises(ValueError, match="head"):
        PagedScorer(SimpleNamespace(cfg=cfg), 1, 64)


@pytest.mark.parametrize("current,entered", [(0, [1]), (1, [])])
def test_calls_run_on_the_tensors_device(monkeypatch, current, entered):
    """Kernels launch on the current device: where the tensors' is another one, it is made current for the call."""
    dev, seen = torch.device("cuda", 1), []

    class On:
        def __init__(self, d):
            seen.append(d.index)

        def __enter__(self):
            monkeypatch.setattr(paged, "_current_device", lambda: 1)

        def __exit__(self, *a):
            monkeypatch.setattr(paged, "_current_device", lambda: current)

    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(paged, "_current_device", lambda: current)
    cache, rot, x = object.__new__(paged.PagedKV), object.__new__(paged.Rotary), torch.zeros(1, 2, 64)
    cache.device = rot.device = dev
    cache.dtype = torch.float32
    for call in (lambda: cache.attend(None, x), lambda: cache.append(None, x, x), lambda: paged.rope(x, rot, None),
                 lambda: paged.rope_backward(x, rot, None)):
        seen.clear()
        with pytest.raises(ValueError, match="cuda:1"):  # x is not there: the call got as far as its checks
            call()
        assert seen == entered


def test_the_stride_over_a_single_token_does_not_count():
    """It is never taken: a row of an odd-sized buffer is as good as any."""
    dev = torch.device("cpu")
    wide = torch.zeros(3, 4 * 64 + 5)
    x = wide[:, :256].unflatten(1, (4, 64))[1:2]
    assert x.stride(0) == 261 and paged._heads(x, "q", torch.float32, dev) == 256
    assert paged._heads(wide[:, :256].unflatten(1, (4, 64)), "q", torch.float32, dev) == 261
    assert paged._heads(x[:0], "q", torch.float32, dev) == 256


def test_bounds_that_do_not_fit_are_refused():
    """Instead of reaching the library modulo 2^32."""
    z, one = torch.zeros(2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    for kw in (dict(max_new=2 ** 32 + 1, max_kv=4), dict(max_new=1, max_kv=2 ** 32 + 4), dict(max_new=2 ** 31, max_kv=4),
               dict(max_new=-1, max_kv=4), dict(max_new=1, max_kv=-1), dict(max_new=1, max_kv=4, total_kv=-1)):
        with pytest.raises(ValueError, match="max_new"):
            paged.Chunks(z, one, table, **kw)
    c = paged.Chunks(z, one, table, max_new=2 ** 31 - 1, max_kv=2 ** 31 - 1)
    assert c.struct.max_new == c.struct.max_kv == 2 ** 31 - 1


def test_caches_of_one_stream_share_a_workspace(monkeypatch):
    """Not those of different streams or devices; it goes with the last cache that has used it."""
    import gc

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(paged, "_shared", type(paged._shared)())

    def cache():
        c = object.__new__(paged.PagedKV)
        c.device, c._ws = torch.device("cpu"), {}
        return c

    a, b = cache(), cache()
    ws = a._workspace_for(1000, 7)
    assert b._workspace_for(900, 7) is ws and b._workspace_for(900, 8) is not ws
    bigger = b._workspace_for(3000, 7)
    assert bigger.numel() >= 3000 and a._workspace_for(1000, 7) is ws and a._workspace_for(2500, 7) is bigger
    del ws, bigger, a, b
    gc.collect()
    assert len(paged._shared) == 0


def _cut_items(pairs, nt):
    """Items of a sequence's last, partly filled wave over 148 SMs that are splits: the cheapest number of splits of at
    least 8 tiles, where a split costs 4.5 tiles' time besides its own and a whole item 1.5, and a twentieth is gained."""
    f = np.float32
    waves, rest = divmod(pairs, 148)
    cost, best = (f(nt) + f(1.5)) * (f(1) - f(0.05) * f(waves + 1)), 1
    for ns in range(2, min(16, nt // 8) + 1):
        c = f(-(-rest * ns // 148)) * (f(nt) * f(1 / ns) + f(4.5))
        if rest * ns <= 1184 and c < cost * f(1 - 1e-6):
            cost, best = c, ns
    return rest * best if best > 1 else 0


def test_workspace_holds_every_split_and_not_much_more():
    """bf16, 32 heads over 8 of 128 channels (64 tokens to a block of 256 rows)."""
    L = _lib.lib()
    kv = _kv(dtype=_lib.BF16, head_dim=128, n_kv_heads=8, page_size=128, token_stride=1024, head_stride=128,
             page_stride=1 << 17)

    def slots(n, new, max_kv, total=0):
        ch = _ch(n_seqs=n, n_tokens=n * new, max_new=new, max_kv=max_kv, table_stride=max_kv // 128 + 1, total_kv=total)
        ws = L.altxs_paged_attention_workspace_bytes(C.byref(kv), C.byref(ch), 32, 0)
        few = ((total or n * max_kv) // 512 + n) * 8 * 16 * 132 * 4
        return ws, (ws - _lib.PAGED_COUNTER_BYTES - few) // (256 * 130 * 4)

    for nt in (16, 26, 27, 40, 60, 61, 100, 111, 181, 276, 402, 566, 1300):
        for blocks in list(range(1, 20)) + [37, 55, 74]:
            got = slots(1, 64 * blocks, 128 * nt)[1]
            assert got >= max(_cut_items(8 * b, k) for b in range(1, blocks + 1) for k in {nt, nt - 1, (nt + 15) // 2, 16})
    cache = 2 * 8 * 128 * 2  # bytes of a position
    for n, new, max_kv, most in ((8, 2048, 4096, 400 << 20), (64, 4096, 8192, 2 * 64 * 8192 * cache),
                                 (256, 1024, 4096, 3 * 256 * 4096 * cache)):
        assert slots(n, new, max_kv)[0] <= most
    # sequences of fewer than 16 tiles are not split: a known total bounds the number of those that are
    assert slots(64, 4096, 8192, 10 * 15 * 128)[1] <= 10 * 3 * 148


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_attention_refuses_a_scale_that_is_not_finite(scale):
    """One of NaN gave every key the same weight where a sequence has many rows, and NaN where it has few."""
    rc = _lib.lib().altxs_paged_attention(C.byref(_kv()), C.byref(_ch()), 4, scale, 0, 4096, 256, 4096, 256, None, 0, 0, None)
    assert rc == _lib.ALTXS_EINVAL
    rc = _lib.lib().altxs_paged_attention(C.byref(_kv()), C.byref(_ch(n_tokens=0)), 4, scale, 0, 4096, 256, 4096, 256, None, 0,
                                          0, None)
    assert rc == _lib.ALTXS_EINVAL


def test_trim_of_long_streams():
    """Block by block in their order, and a step of a stream of a million positions takes no longer for those that
    have come back long ago (a table of 65536 blocks: a loop over them took 5 ms, this 20 us)."""
    import time

    a = paged.PageAllocator(2, 70000, 16, 1 << 20, "cpu")
    rng = np.random.default_rng(1)
    a.extend([1 << 19, 77])
    for w in (300000, 5000, 64):
        first = max(0, int(a.len[0]) + 1 - w) // 16
        want = [int(p) for p in a.table[0, :first] if p >= 0]
        free = list(a.free)
        assert a.trim(0, w) == len(want) and a.free == free + want and (a.table[0, :first] == -1).all()
        a.extend([int(rng.integers(1, 100)), 0])
    a.extend([(1 << 20) - int(a.len[0]), 0])
    a.trim(0, 64)
    t = time.perf_counter()
    for _ in range(50):
        assert a.trim(0, 64) == 0
    assert (time.perf_counter() - t) / 50 < 1e-3
