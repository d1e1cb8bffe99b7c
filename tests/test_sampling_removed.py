"""Tokens that rules removed (logits of G2_MASKED) are never drawn: the host
sampler on the CPU, the device sampler on an engine's slot.

The reference's own picks stay where nothing is removed (index 0 at u = 0, any
index where the sum falls short): test_abi_cpu.py and test_gpu_sampler.py hold
those.
"""
import ctypes as C
import os

import numpy as np
import pytest

import gpt2b200 as g2
from gpt2b200 import synth

STATE = -7


def draws(logits, n, **kw):
    libc = C.CDLL(None)
    libc.srand(11)
    return {g2.sample(logits, kw.pop("ctx", []), **kw) for _ in range(n)}


def masked(V, allowed, seed=0):
    rng = np.random.default_rng(seed)
    l = np.full(V, g2.MASKED, np.float32)
    l[allowed] = rng.standard_normal(len(allowed)).astype(np.float32)
    return l


@pytest.mark.parametrize("T", [0.05, 1.0, 9.0, 11.0, 1e4])
@pytest.mark.parametrize("k", [0, 1, 3, 40])
def test_host_draws_allowed_tokens(T, k):
    allowed = [3, 17, 300, 998]
    l = masked(1000, allowed)
    got = draws(l, 300, temperature=T, top_k=k, ctx=[3, 4, 5], rep_penalty=1.5)
    assert got <= set(allowed)
    if T >= 9 and k in (0, 40):
        assert got == set(allowed)


@pytest.mark.parametrize("T", [0.0, 0.7, 1.0, 20.0])
def test_host_nothing_left(T):
    for l in (masked(400, []), np.full(400, -np.inf, np.float32)):
        with pytest.raises(g2.G2Error) as e:
            g2.sample(l, [], temperature=T)
        assert e.value.code == STATE


def test_host_only_eos_left_and_forbidden():
    l = masked(50257, [g2.EOS])
    for T in (0.0, 1.0, 20.0):
        assert g2.sample(l, [], temperature=T) == g2.EOS
        with pytest.raises(g2.G2Error) as e:
            g2.sample(l, [], forbid_eos=True, temperature=T)
        assert e.value.code == STATE


@pytest.fixture(scope="module")
def engine():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from conftest import MODEL_CACHE
    with g2.Engine(synth.ensure_model(os.path.join(MODEL_CACHE, "tiny_s2"), synth.TINY, seed=2)) as eng:
        yield eng


US = [0.0, 1e-300, 1e-12, 0.3, 0.999, 1 - 2.0 ** -53]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0.05, 1.0, 9.0, 11.0, 1e4])
@pytest.mark.parametrize("k", [0, 1, 3, 300])
def test_device_draws_allowed_tokens(engine, T, k):
    """The first and the last token are among the removed ones."""
    V = engine.cfg.vocab_size
    allowed = [1, 77, 30000, V - 2]
    engine.prefill([5, 6, 7])
    engine.process_logits(allowed=allowed)
    got = {u: engine.sample_device([5, 77], temperature=T, top_k=k, rep_penalty=1.3, u=u) for u in US}
    assert set(got.values()) <= set(allowed)
    if k == 0 and T >= 1:
        assert got[0.0] == 1 and got[1 - 2.0 ** -53] == V - 2      # the first and the last with a weight
    # the host sampler picks from the same set
    assert draws(engine.logits()[:V], 20, temperature=T, top_k=k) <= set(allowed)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0.0, 0.7, 1.0, 20.0])
def test_device_nothing_left(engine, T):
    engine.prefill([5, 6, 7])
    engine.process_logits(allowed=[])
    for u in (0.0, 0.5):
        with pytest.raises(g2.G2Error) as e:
            engine.sample_device([], temperature=T, u=u)
        assert e.value.code == STATE
    engine.prefill([5, 6, 7])
    engine.process_logits(allowed=[g2.EOS])
    assert engine.sample_device([], temperature=T, u=0.5) == g2.EOS
    with pytest.raises(g2.G2Error) as e:
        engine.sample_device([], forbid_eos=True, temperature=T, u=0.5)
    assert e.value.code == STATE
    assert engine.argmax()[0] == g2.EOS
