"""Rules on logits on the GPU (g2k_process_logits, g2_process_logits) against
their definition in 64 bits.

Each of the five operations on a logit (quotient or product, two subtractions,
the frequency product, the bias) rounds once: a result is within 2.5 fp32 steps
(5 * 2^-24) of the largest magnitude on its way.  Untouched logits and masked
ones are exact.
"""
import os

import numpy as np
import pytest

from gpt2b200 import synth

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g2():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import gpt2b200
    return gpt2b200


def want_row(l, ctx=(), n_prompt=0, rep=1.0, pres=0.0, freq=0.0, bias=(), ok=None):
    """The row in 64 bits, and the largest magnitude each value had on its way."""
    l = l.astype(np.float64)
    V = len(l)
    top = np.abs(l)
    rep, pres, freq = (float(np.float32(v)) for v in (rep, pres, freq))
    seen = sorted({int(i) for i in ctx if 0 <= i < V})
    if rep > 0:
        for i in seen:
            l[i] = l[i] / rep if l[i] > 0 else l[i] * rep
    top = np.maximum(top, np.abs(l))
    made = [int(i) for i in ctx[max(n_prompt, 0):] if 0 <= i < V]
    for i in set(made):
        l[i] -= freq * made.count(i)
        top[i] = max(top[i], abs(freq * made.count(i)), abs(l[i]))
        l[i] -= pres
        top[i] = max(top[i], abs(pres), abs(l[i]))
    last = {int(i): float(b) for i, b in bias if 0 <= i < V}
    for i, b in last.items():
        l[i] += b
        top[i] = max(top[i], abs(b), abs(l[i]))
    if ok is not None:
        l[~ok] = np.float32(-1e30)
        top[~ok] = 0
    changed = np.zeros(V, bool)
    changed[seen] = changed[list(last)] = True
    return l, np.where(changed, top, 0)


def close(got, want, top):
    got = got.double().cpu().numpy()
    with np.errstate(over="ignore"):
        want = want.astype(np.float32).astype(np.float64)     # past fp32's range: infinite
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[~fin], want[~fin])
    # half a step more where `want` itself was rounded above
    assert (np.abs(got[fin] - want[fin]) <= 6 * 2.0 ** -24 * top[fin]).all()


def words(ok):
    V = ok.shape[-1]
    pad = np.zeros(ok.shape[:-1] + (-(-V // 32) * 32,), bool)
    pad[..., :V] = ok
    return torch.from_numpy(np.packbits(pad, axis=-1, bitorder="little").view("<i4").copy()).cuda()


def dev(a, dt):
    return torch.from_numpy(np.ascontiguousarray(a, dt)).cuda()


def run(g2, rows, V, seed=0, max_ctx=50, penal=True, n_bias=5, mask=True, in_place=False, ld=None, ld_out=None, offset=0,
        logits=None, stream=0):
    rng = np.random.default_rng(seed)
    ld, ld_out = ld or V, ld_out or V
    buf = rng.standard_normal((rows, ld)).astype(np.float32) * 4
    if logits is not None:
        buf[:, :V] = logits
    ctxs = [rng.integers(0, V, rng.integers(0, max_ctx + 1)) if i % 3 else
            rng.integers(0, max(1, V // 50), max_ctx) for i in range(rows)]
    prompts = [int(rng.integers(0, len(c) + 3)) for c in ctxs]
    rep, pres, freq = (rng.uniform(a, b, rows).astype(np.float32) for a, b in ((0.7, 1.8), (-0.5, 1.5), (-0.2, 0.7)))
    bias = [[(int(rng.integers(0, V)), float(np.float32(rng.standard_normal() * 5))) for _ in range(n_bias if r % 4 != 3 else 0)]
            for r in range(rows)]
    ok = rng.random((rows, V)) < np.array([0.02, 0.9, 0.0, 1.0])[np.arange(rows) % 4][:, None]
    starts = np.cumsum([0] + [len(c) for c in ctxs])
    bstarts = np.cumsum([0] + [len(b) for b in bias])
    flat = [p for b in bias for p in b]
    kw = {}
    if penal:
        kw.update(ctx=dev(np.concatenate(ctxs + [np.zeros(0)]), np.int32), ctx_start=dev(starts, np.int32), n_prompt=dev(prompts, np.int32),
                  rep_penalty=dev(rep, np.float32), presence=dev(pres, np.float32), frequency=dev(freq, np.float32))
    if n_bias:
        kw.update(bias_ids=dev([p[0] for p in flat], np.int32), bias=dev([p[1] for p in flat], np.float32), bias_start=dev(bstarts, np.int32))
    if mask:
        kw.update(mask=words(ok), mask_stride=-(-V // 32))
    store = torch.zeros(offset + rows * ld, device="cuda")
    x = store[offset:]
    x.copy_(dev(buf, np.float32).flatten())
    y = x if in_place else torch.full((offset + rows * ld_out,), 9.25, device="cuda")[offset:]
    g2.process_logits(x, y, rows, V, g2.logit_rules(**kw), ld=ld, ld_out=ld if in_place else ld_out, stream=stream)
    torch.cuda.synchronize()
    got = y.view(rows, ld if in_place else ld_out)
    for r in range(rows):
        want, top = want_row(buf[r, :V], ctxs[r] if penal else (), prompts[r], rep[r] if penal else 1.0, pres[r], freq[r],
                             bias[r] if n_bias else (), ok[r] if mask else None)
        close(got[r, :V], want, top)
    rest = got[:, V:].cpu().numpy()
    np.testing.assert_array_equal(rest, buf[:, V:] if in_place else np.full_like(rest, 9.25))
    if not in_place:
        np.testing.assert_array_equal(x.view(rows, ld).cpu().numpy(), buf)     # NaN equals NaN here


@pytest.mark.parametrize("rows,V", [(1, 1), (1, 31), (2, 33), (4, 1000), (3, 4096), (3, 4097), (1, 50257), (5, 50257), (8, 8191)])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules(g2, rows, V, in_place):
    run(g2, rows, V, in_place=in_place)
    run(g2, rows, V, in_place=in_place, seed=1, ld=V + 3, ld_out=V + 5)


@pytest.mark.parametrize("penal,n_bias,mask", [(False, 0, False), (True, 0, False), (False, 300, False), (False, 0, True), (True, 7, False)])
@pytest.mark.parametrize("in_place", [False, True])
def test_parts(g2, penal, n_bias, mask, in_place):
    run(g2, 4, 5003, penal=penal, n_bias=n_bias, mask=mask, in_place=in_place, seed=2)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_alignment(g2, offset):
    run(g2, 3, 6001, offset=offset, seed=3)
    run(g2, 3, 6000, offset=offset, seed=4, in_place=True, ld=6001)


def test_long_contexts_and_many_biases(g2):
    run(g2, 3, 50257, max_ctx=20000, n_bias=4000, seed=5)


def test_infinities_and_nan(g2):
    rng = np.random.default_rng(6)
    l = rng.standard_normal((4, 900)).astype(np.float32)
    l[rng.random(l.shape) < 0.2] = -np.inf
    l[:, 5], l[:, 6], l[:, 7] = np.inf, np.nan, np.finfo(np.float32).min
    run(g2, 4, 900, logits=l, seed=7, max_ctx=300)
    run(g2, 4, 900, logits=l, seed=7, max_ctx=300, mask=False, in_place=True)


def test_ids_outside_and_repeated(g2):
    V = 100
    l = torch.linspace(-3, 3, V, device="cuda")[None].contiguous()
    ctx = dev([-1, 5, 5, 99, 100, 2 ** 31 - 1, -2 ** 31, 5], np.int32)
    ids, val = dev([7, -1, 7, 100, 99, 7], np.int32), dev([1, 50, 2, 50, 3, -4], np.float32)
    y = torch.empty_like(l)
    one = lambda v: dev([v], np.float32)  # noqa: E731
    g2.process_logits(l, y, 1, V, g2.logit_rules(ctx=ctx, rep_penalty=one(2.0), presence=one(0.5), frequency=one(0.25),
                                                 bias_ids=ids, bias=val))
    want, top = want_row(l[0].cpu().numpy(), ctx.cpu().numpy(), 0, 2.0, 0.5, 0.25, list(zip(ids.tolist(), val.tolist())))
    close(y[0], want, top)
    assert y[0, 7] == l[0, 7] - 4          # the last of three pairs


def test_bad_offsets_are_clamped(g2):
    """Context and pair offsets outside their arrays are ignored, and so are reversed ones."""
    V, l = 64, torch.ones(3, 64, device="cuda")
    ctx, starts = dev([1, 2, 3], np.int32), dev([-5, 2, 1, 900], np.int32)
    y = torch.empty_like(l)
    g2.process_logits(l, y, 3, V, g2.logit_rules(ctx=ctx, ctx_start=starts, rep_penalty=dev([2, 2, 2], np.float32)))
    want = torch.ones(3, 64)
    want[0, [1, 2]] = 0.5
    want[2, [2, 3]] = 0.5
    assert torch.equal(y.cpu(), want)


def test_penalties_of_no_effect(g2):
    l = torch.randn(2, 333, device="cuda")
    y = torch.empty_like(l)
    ctx, st = dev(range(300), np.int32), dev([0, 150, 300], np.int32)
    g2.process_logits(l, y, 2, 333, g2.logit_rules(ctx=ctx, ctx_start=st, rep_penalty=dev([0.0, -1.0], np.float32)))
    assert torch.equal(l, y)
    g2.process_logits(l, y, 2, 333, g2.logit_rules(ctx=ctx, ctx_start=st, presence=dev([0, 0], np.float32)))
    assert torch.equal(l, y)


def test_shared_mask(g2):
    ok = np.random.default_rng(8).random(5000) < 0.5
    l = torch.randn(6, 5000, device="cuda")
    y = torch.empty_like(l)
    g2.process_logits(l, y, 6, 5000, g2.logit_rules(mask=words(ok), mask_stride=0))
    t = torch.from_numpy(ok).cuda()
    assert torch.equal(y, torch.where(t, l, torch.tensor(-1e30, device="cuda")))


def test_capture_and_streams(g2):
    V = 50257
    l = torch.randn(2, V, device="cuda")
    ctx, st, rep = torch.arange(100, device="cuda", dtype=torch.int32), dev([0, 40, 100], np.int32), dev([1.5, 2.0], np.float32)
    rules, y = g2.logit_rules(ctx=ctx, ctx_start=st, rep_penalty=rep), torch.empty_like(l)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g2.process_logits(l, y, 2, V, rules, stream=torch.cuda.current_stream().cuda_stream)
    for shift in (0, 777):
        ctx.copy_(torch.arange(100, device="cuda") + shift)
        graph.replay()
        torch.cuda.synchronize()
        want = l.clone()
        for r, (a, b) in enumerate(((0, 40), (40, 100))):
            part = l[r, a + shift:b + shift]
            want[r, a + shift:b + shift] = torch.where(part > 0, part / rep[r], part * rep[r])
        assert torch.equal(y, want)


def _model():
    from conftest import MODEL_CACHE
    return synth.ensure_model(os.path.join(MODEL_CACHE, "tiny_s2"), synth.TINY, seed=2)


def test_engine_slot(g2):
    """g2_process_logits on an engine's slots, and what the pickers then see."""
    rng = np.random.default_rng(9)
    prompts = [synth.prompt_ids(80 + s, 9 + 3 * s) for s in range(2)]
    with g2.Engine(_model(), max_batch=2) as eng:
        with pytest.raises(g2.G2Error) as ei:
            eng.process_logits(slot=1)
        assert ei.value.code == -7
        V = eng.cfg.vocab_size
        for s, p in enumerate(prompts):
            eng.prefill(p, slot=s)
        before = [eng.logits(s) for s in range(2)]
        best = eng.argmax(1)[0]
        ctx = list(p) + [best, 3, 3]
        ok = rng.random(V) < 0.5
        ok[best] = False
        bias = {11: 2.5, 40000: -1.0}
        eng.process_logits(ctx, n_prompt=len(p), rep_penalty=1.3, presence=0.4, frequency=0.2, bias=bias, allowed=ok, slot=1)
        got = eng.logits(1)
        want, top = want_row(before[1][:V], np.array(ctx), len(p), 1.3, 0.4, 0.2, list(bias.items()), ok)
        close(torch.from_numpy(got[:V]), want, top)
        assert np.array_equal(eng.logits(0), before[0]) and np.array_equal(got[V:], before[1][V:])
        first = int(np.argmax(got[:V]))
        assert eng.argmax(1)[0] == first and eng.topk(3, slot=1)[1][0] == first
        assert eng.sample_device([], temperature=0.0, slot=1) == first
        assert ok[eng.sample_device([], temperature=1.0, u=0.7, slot=1)]
        eng.decode(first, len(p), slot=1)                     # the next step's logits are untouched
        eng.process_logits(allowed=[17], slot=1)
        assert eng.argmax(1)[0] == 17
        for kw in (dict(context=[1] * (eng.cfg.n_ctx + 1)), dict(bias={i: 0.0 for i in range(V + 1)})):
            with pytest.raises(g2.G2Error):
                eng.process_logits(slot=1, **kw)


def test_engine_penalty_is_the_samplers(g2):
    """The repetition penalty equals the one inside g2_sample_device (main.c:1885-1895)."""
    p = synth.prompt_ids(90, 20)
    with g2.Engine(_model()) as eng:
        eng.prefill(p)
        picks = [eng.sample_device(p, temperature=1.0, top_k=50, rep_penalty=1.4, u=u) for u in (0.2, 0.5, 0.9)]
        eng.process_logits(p, rep_penalty=1.4)
        assert picks == [eng.sample_device([], temperature=1.0, top_k=50, u=u) for u in (0.2, 0.5, 0.9)]
