"""PagedScorer (chunked forward over paged caches: append with rotation, chunk
attention) against the oracle's one-symbol steps: logits within the step's own
bar of 2e-3, and the bits that follow from them."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from altxs_b200 import codec as C
from altxs_b200.config import ModelConfig
from altxs_b200.engine import DeviceModel
from altxs_b200.scorer import PagedScorer
from altxs_b200.synth import zipf_markov
from oracle.model import OracleModel, OracleWeights

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
TOL = 2e-3


def _cfg(**kw):
    d = dict(vocab_size=512, num_layers=3, model_dim=128, num_heads=4, num_kv_heads=2, mlp_mult=4.0, rope_dims=16,
             block_size=48, online_retrain_every=64, seed=11, retrain_mode="none")
    return ModelConfig(**{**d, **kw})


def _oracle_logits(w, syms):
    om = OracleModel(OracleWeights.from_model_weights(w))
    st = om.new_stream()
    return np.stack([om.step(st, int(t)).numpy() for t in syms])


@pytest.mark.parametrize("tensor_cores", [True, False])
def test_chunks_match_the_step_oracle(tensor_cores):
    """Uneven chunks (none, one, many symbols), past the sliding window, pages taken back on the way."""
    cfg = _cfg()
    w = C.synth_weights(cfg, seed=6)
    dm = DeviceModel(w, DEV, tensor_cores=tensor_cores)
    n, T = 3, 130
    data = zipf_markov(T, cfg.vocab_size, np.arange(n) + 4)
    want = [_oracle_logits(w, data[s]) for s in range(n)]
    sc = PagedScorer(dm, n, 200, chunk=64, page_size=16)
    done = [0] * n
    rng = np.random.default_rng(3)
    while min(done) < T:
        take = [min(int(rng.choice([0, 1, 2, 5, 17, 64])), T - d) for d in done]
        if not any(take):
            continue
        got = sc.advance([data[s][done[s]:done[s] + take[s]] for s in range(n)]).cpu().numpy()
        at = 0
        for s in range(n):
            if take[s]:
                assert np.abs(got[at:at + take[s]] - want[s][done[s]:done[s] + take[s]]).max() < TOL
            at += take[s]
            done[s] += take[s]
    held = (sc.pages.table >= 0).sum(1)
    assert (held <= -(-cfg.ctx // 16) + 1).all()  # what has left the window is free again


def test_scores_of_ragged_streams():
    cfg = _cfg(num_heads=2)  # head size 64
    w = C.synth_weights(cfg, seed=7)
    dm = DeviceModel(w, DEV)
    lens = [1, 100, 37, 2]
    data = zipf_markov(100, cfg.vocab_size, np.arange(4) + 1)
    streams = [data[s, :m] for s, m in enumerate(lens)]
    sc = PagedScorer(dm, 4, 128, chunk=33, page_size=16)
    bits = sc.score(streams)
    again = sc.score(streams)
    for s, m in enumerate(lens):
        assert np.array_equal(bits[s], again[s]) and bits[s].shape == (m,)
        want = [math.log2(cfg.vocab_size)]
        if m > 1:
            lg = torch.from_numpy(_oracle_logits(w, streams[s][:-1])).double()
            want += (-torch.log_softmax(lg, 1).gather(1, torch.from_numpy(streams[s][1:].astype(np.int64))[:, None])[:, 0]
                     / math.log(2)).tolist()
        assert np.abs(bits[s] - np.array(want)).max() < 2 * TOL / math.log(2)


def test_refusals():
    dm = DeviceModel(C.synth_weights(_cfg(), seed=1), DEV)
    with pytest.raises(ValueError):
        PagedScorer(dm, 0, 10)
    sc = PagedScorer(dm, 1, 64, page_size=16, n_pages=2)
    with pytest.raises(ValueError):
        sc.advance([np.array([512])])
    with pytest.raises(RuntimeError, match="out of pages"):
        sc.advance([np.zeros(40, dtype=np.int64)])
    with pytest.raises(ValueError):
        sc.score([np.zeros(3, dtype=np.int64)] * 2)
    motif = _cfg(xsa_last_n=1)
    with pytest.raises(ValueError, match="plain"):
        PagedScorer(DeviceModel(C.synth_weights(motif, seed=1), DEV), 1, 64)


@pytest.mark.parametrize("tensor_cores", [True, False])
def test_arena_models_score_with_their_live_parameters(tensor_cores):
    """A model whose parameters lie in one arena scores like the oracle; after an update (the embedding's rows in
    another order: symbol i is the old symbol perm[i], on both sides), input rows and head are the new ones."""
    cfg = _cfg()
    w = C.synth_weights(cfg, seed=8)
    dm = DeviceModel(w, DEV, tensor_cores=tensor_cores, full_params=True)
    T = 60
    data = zipf_markov(T, cfg.vocab_size, np.arange(1) + 9)
    sc = PagedScorer(dm, 1, 200, chunk=64, page_size=16)
    got = sc.advance([data[0]]).cpu().numpy()
    assert np.abs(got - _oracle_logits(w, data[0])).max() < TOL
    perm = np.random.default_rng(5).permutation(cfg.vocab_size)
    emb = dm.arena("emb").view(cfg.vocab_size, cfg.model_dim)
    emb.copy_(emb.clone()[torch.from_numpy(perm).to(DEV)])
    dm.refresh()
    new = np.argsort(perm)[data[0]]  # the new names of the same symbols
    for s in (sc, PagedScorer(dm, 1, 200, chunk=64, page_size=16)):
        s.pages.release(0)
        assert np.abs(s.advance([new]).cpu().numpy() - got[:, perm]).max() < 1e-5
