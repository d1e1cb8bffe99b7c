"""Refusals of the 4-bit, 8-bit-cache and logit-rule entry points, on the CPU:
every call here fails a check that comes before any device work, so host
addresses (and addresses that are no memory at all) are never used.
"""
import ctypes as C

import pytest

import gpt2b200 as g2

ARG, CUDA, RANGE, STATE = -1, -4, -6, -7
BUF = C.create_string_buffer(1 << 16)
A = (C.addressof(BUF) + 255) // 256 * 256      # an aligned host address


def code(f, *a):
    with pytest.raises(g2.G2Error) as e:
        f(*a[:-1], **a[-1]) if a and isinstance(a[-1], dict) else f(*a)
    assert str(e.value)
    return e.value.code


def test_q4_sizes():
    for n, k in ((16, 64), (17, 65), (1, 32768), (50257, 1600)):
        pad = -(-n // 32) * 32 * (-(-k // 64) * 64)            # whole blocks of 32 columns and 64 rows
        for g in (32, 64, 128):
            scales = 2 * pad // min(g, 64)                     # a scale for each part of 64 rows at least
            assert g2.q4_bytes(n, k, g) == pad // 2 + scales
    for n, k, g in ((0, 1, 32), (1, 0, 32), (1, 1, 16), (1, 1, 0), (1, 32769, 32), (-4, 64, 64), (2 ** 31 - 1, 64, 64)):
        assert g2.q4_bytes(n, k, g) == 0


@pytest.mark.parametrize("f", [lambda **k: g2.q4_pack(A, k.pop("p", A), **k), lambda **k: g2.q4_unpack(k.pop("p", A), A, **k)])
def test_q4_pack_arguments(f):
    ok = dict(N=16, K=64, group=32)
    assert code(f, {**ok, "p": None}) == ARG
    assert code(f, {**ok, "p": A + 16}) == ARG
    assert code(f, {**ok, "group": 48}) == ARG
    for bad in (dict(N=0), dict(K=0), dict(K=32769), dict(N=-1)):
        assert code(f, {**ok, **bad}) == RANGE


def test_q4_pack_dtype():
    assert code(g2.q4_pack, A, A, 16, 64, 32, dict(dtype=2)) == ARG
    assert code(g2.q4_pack, A + 2, A, 16, 64, 32, {}) == ARG
    assert code(g2.q4_pack, None, A, 16, 64, 32, {}) == ARG


def test_matvec_q4_arguments():
    f = lambda **k: g2.matvec_q4(k.pop("x", A), k.pop("p", A), k.pop("y", A), **k)  # noqa: E731
    ok = dict(M=1, N=16, K=64, group=32)
    for bad in (dict(x=None), dict(p=None), dict(y=None), dict(p=A + 128), dict(x=A + 2), dict(y=A + 1, dtype=1), dict(bias=A + 2),
                dict(residual=A + 2), dict(ln_gamma=A), dict(ln_beta=A), dict(dtype=7), dict(group=0)):
        assert code(f, {**ok, **bad}) == ARG, bad
    for bad in (dict(M=0), dict(M=17), dict(N=0), dict(K=0), dict(K=40000)):
        assert code(f, {**ok, **bad}) == RANGE, bad


def cache(**k):
    f = dict(k=A, v=A, k_scale=A, v_scale=A, n_pages=4, n_kv_head=2, page_size=16, head_dim=64, format=0)
    f.update(k)
    return g2.KV8(**f)


CALLS = {
    "append": lambda c, r: g2.kv8_append(c, r.pop("a", A), r.pop("b", A), r.pop("n_rows", 3), r.pop("n_seq", 3), r.pop("table", A),
                                         r.pop("table_stride", 4), r.pop("per", A), **r),
    "gather": lambda c, r: g2.kv8_gather(c, r.pop("a", A), r.pop("b", A), r.pop("n_rows", 3), r.pop("n_seq", 3), r.pop("table", A),
                                         r.pop("table_stride", 4), r.pop("per", A), **r),
    "attention": lambda c, r: g2.kv8_attention(c, r.pop("a", A), r.pop("b", A), r.pop("heads", 4), r.pop("n_rows", 3),
                                               r.pop("n_seq", 3), r.pop("table", A), r.pop("table_stride", 4), r.pop("per", A),
                                               r.pop("ws", A), r.pop("ws_bytes", 1 << 60), **r),
}


@pytest.mark.parametrize("name", CALLS)
def test_kv8_cache_arguments(name):
    f = CALLS[name]
    for bad in (dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(format=2), dict(page_size=48),
                dict(page_size=0), dict(head_dim=80), dict(k=A + 8), dict(v_scale=A + 2)):
        assert code(lambda: f(cache(**bad), {})) == ARG, bad
    for bad in (dict(n_pages=0), dict(n_kv_head=0), dict(n_kv_head=70000)):
        assert code(lambda: f(cache(**bad), {})) == RANGE, bad


@pytest.mark.parametrize("name", CALLS)
def test_kv8_row_arguments(name):
    f, stride = CALLS[name], "q_stride" if name == "attention" else "row_stride"
    for bad in (dict(a=None), dict(b=None), dict(table=None), dict(per=None), dict(dtype=3), dict(a=A + 8), dict(b=A + 4),
                dict(table=A + 1), dict(per=A + 2), dict(status=A + 2), dict(q_start=A + 3, max_q=2), {stride: 514},
                {stride: 516, "dtype": 1}):
        assert code(lambda: f(cache(), dict(bad))) == ARG, bad
    for bad in (dict(n_rows=-1), dict(n_seq=-1), dict(max_q=0), dict(table_stride=0), dict(n_rows=4), dict(max_q=2), {stride: 64},
                dict(table_stride=2 ** 30), dict(n_seq=2 ** 31 - 1, n_rows=2 ** 31 - 1, max_q=2 ** 31 - 1, q_start=A)):
        assert code(lambda: f(cache(), dict(bad))) == RANGE, bad


def test_kv8_attention_arguments():
    f = CALLS["attention"]
    for bad in (dict(ws=None), dict(ws=A + 64), dict(ws_bytes=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf"))):
        assert code(lambda: f(cache(), dict(bad))) == ARG, bad
    for bad in (dict(heads=0), dict(heads=3), dict(heads=2 * 40000), dict(out_stride=64)):
        assert code(lambda: f(cache(), dict(bad))) == RANGE, bad
    assert g2.kv8_attention_workspace(cache(), 4, 3, 1) > 0
    assert g2.kv8_attention_workspace(cache(), 0, 3, 1) == 0 == g2.kv8_attention_workspace(cache(), 4, 3, 0)


@pytest.mark.parametrize("name", CALLS)
def test_kv8_nothing_to_do(name):
    CALLS[name](cache(), dict(n_rows=0, n_seq=0))
    CALLS[name](cache(), dict(n_rows=0, n_seq=5, q_start=A, max_q=3))


def test_kv8_cache_tensors():
    torch = pytest.importorskip("torch")
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    s = torch.zeros(4, 2)
    for bad in ((k.float(), k, s, s), (k[0], k[0], s, s), (k, k[:3], s, s), (k, k, s[:3], s), (k, k, s.half(), s),
                (k, torch.zeros(4, 2, 64, 16, dtype=torch.int8).transpose(2, 3), s, s)):
        assert code(g2.kv8_cache, *bad) == ARG


def test_logit_rules_arguments():
    def f(**k):
        r = dict(ctx=A, n_ctx=4)
        r.update({n: k.pop(n) for n in list(k) if n in dict(g2.LogitRules._fields_)})
        g2.process_logits(k.pop("a", A), k.pop("b", A), k.pop("rows", 1), k.pop("V", 100), g2.LogitRules(**r), **k)
    for bad in (dict(a=None), dict(b=None), dict(a=A + 2), dict(ctx=None), dict(ctx=A + 1), dict(n_bias=1), dict(n_bias=1, bias_ids=A),
                dict(rows=2), dict(rows=2, ctx_start=A, n_bias=1, bias=A, bias_ids=A), dict(rep_penalty=A + 2), dict(mask=A + 2),
                dict(rows=2, ctx_start=A, ld=100, ld_out=104)):
        assert code(f, bad) == ARG, bad
    for bad in (dict(rows=-1), dict(rows=65536), dict(V=0), dict(n_ctx=-1), dict(n_bias=-1), dict(mask=A, mask_stride=3),
                dict(mask_stride=-1), dict(rows=2, ctx_start=A, ld=99)):
        assert code(f, bad) == RANGE, bad
    assert g2.lib.g2k_process_logits(A, 100, A, 100, 1, 100, None, None) == ARG
    f(rows=0)
    assert g2.lib.g2_process_logits(None, 0, None) == ARG


def test_sizes_past_a_launch():
    """More heads than a grid has rows; a vocabulary whose padded length passes 32 bits."""
    for f in CALLS.values():
        assert code(lambda: f(cache(n_kv_head=32768), dict(heads=32768) if f is CALLS["attention"] else {})) == RANGE
    for V in (2 ** 31 - 1, 2 ** 31 - 4, 2 ** 30 + 1):
        assert code(lambda: g2.process_logits(A, A, 1, V, g2.LogitRules())) == RANGE


def no_device_memory():
    """What host memory gives: it is no memory of the device, or there is no device to ask."""
    try:
        import torch
        return ARG if torch.cuda.is_available() else CUDA
    except ImportError:
        return CUDA


def test_host_tensors_are_refused():
    torch = pytest.importorskip("torch")
    t, want = torch.zeros(1 << 14), no_device_memory()
    t = t[(-t.data_ptr() // 4) % 64:]                      # 256-byte aligned
    assert code(g2.q4_pack, t, t, 1, 64, 32, {}) == want
    assert code(g2.matvec_q4, t, t, t, 1, 16, 64, 32, {}) == want
    assert code(g2.process_logits, t, t, 1, 64, g2.logit_rules(), {}) == want
    assert code(g2.process_logits, t, t, 1, 64, g2.logit_rules(ctx=t, rep_penalty=t), {}) == want


def test_host_addresses_reach_no_kernel():
    """Aligned host memory passes the checks of form; the check of memory refuses it."""
    want = no_device_memory()
    assert code(g2.q4_pack, A, A, 16, 64, 32, {}) == want
    assert code(g2.matvec_q4, A, A, A, 1, 16, 64, 32, {}) == want
    for f in CALLS.values():
        assert code(lambda: f(cache(), {})) == want
    assert code(lambda: g2.process_logits(A, A, 1, 100, g2.LogitRules(ctx=A, n_ctx=3))) == want


def test_tensors_of_another_type():
    """A tensor whose elements are not of the stated size is refused: it would be read past its end."""
    torch = pytest.importorskip("torch")
    f, h, i64 = torch.zeros(4096), torch.zeros(4096, dtype=torch.half), torch.zeros(4096, dtype=torch.int64)
    assert code(g2.q4_pack, h, A, 16, 64, 32, {}) == ARG
    assert code(g2.q4_pack, f, A, 16, 64, 32, dict(dtype=g2.G2_F16)) == ARG
    assert code(g2.q4_unpack, A, h, 16, 64, 32) == ARG
    for bad in (dict(x=h), dict(y=h), dict(residual=h), dict(bias=h), dict(ln_gamma=h, ln_beta=h), dict(x=f, dtype=1)):
        k = dict(bad)
        assert code(g2.matvec_q4, k.pop("x", A), A, k.pop("y", A), 1, 16, 64, 32, k) == ARG, bad
    for name, f8 in CALLS.items():
        for bad in (dict(a=h), dict(b=h), dict(a=f, dtype=1), dict(table=i64), dict(per=i64), dict(status=i64), dict(q_start=i64, max_q=2)):
            assert code(lambda: f8(cache(), dict(bad))) == ARG, (name, bad)
    for bad in (dict(ctx=i64), dict(mask=i64), dict(rep_penalty=h), dict(bias=f, bias_ids=i64), dict(bias=f), dict(bias=f, bias_ids=f[:5])):
        assert code(lambda: g2.logit_rules(**bad)) == ARG, bad
    assert code(g2.process_logits, h, h, 1, 64, g2.logit_rules(), {}) == ARG
