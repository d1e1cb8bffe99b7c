"""The 8-bit cache's calls at the limits of their arguments: bounds on the rows of
a sequence that no sequence reaches (GPU), and refusals (CPU)."""
import math

import pytest

torch = pytest.importorskip("torch")
import gpt2b200 as g2  # noqa: E402
from test_operator_args import A as CALLS_A, CALLS, cache, code, no_device_memory  # noqa: E402


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("most", [5, 64, 2 ** 31 - 1])
@pytest.mark.parametrize("page", [16, 128])
def test_any_bound_on_the_rows(most, page):
    """max_q may be far above every count; counts above it are still refused."""
    H, D, counts, pos = 2, 64, [5, 0, 3], [7, 1, 30]
    k, v = (torch.zeros(9, H, page, D, dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.ones(9, H, device="cuda") for _ in "kv")
    c = g2.kv8_cache(k, v, ks, vs)
    table = ints([[0, 1, 2], [3, 4, 5], [6, 7, 8]])
    x = torch.randn(8, 3, H, D, device="cuda", generator=gen(1))
    starts, st = ints([0, 5, 5, 8]), torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(q_start=starts, max_q=most, status=st)
    g2.kv8_append(c, x[:, 1], x[:, 2], 8, 3, table, 3, ints(pos), row_stride=3 * H * D, **kw)
    back = torch.zeros(8, 2, H, D, device="cuda")
    g2.kv8_gather(c, back[:, 0], back[:, 1], 8, 3, table, 3, ints(pos), row_stride=2 * H * D, **kw)
    # a page with rows that stay keeps its scale of 1: half a step is at most half of that
    assert int(st) == 0 and ((back - x[:, 1:]).abs() <= 0.5 * 1.001).all()
    k5, v5, ks5, vs5, exact = torch.zeros_like(k), torch.zeros_like(v), torch.ones_like(ks), torch.ones_like(vs), dict(kw, max_q=5)
    g2.kv8_append(g2.kv8_cache(k5, v5, ks5, vs5), x[:, 1], x[:, 2], 8, 3, table, 3, ints(pos), row_stride=3 * H * D, **exact)
    assert all(torch.equal(a, b) for a, b in ((k, k5), (v, v5), (ks, ks5), (vs, vs5)))
    lens, out = ints([12, 1, 33]), torch.full((8, H, D), 7.0, device="cuda")
    ws = torch.zeros(g2.kv8_attention_workspace(c, H, 3, most), dtype=torch.uint8, device="cuda")
    g2.kv8_attention(c, x[:, 0], out, H, 8, 3, table, 3, lens, ws, ws.numel(), q_stride=3 * H * D, **kw)
    want = torch.full_like(out, 7.0)
    ws5 = torch.zeros(g2.kv8_attention_workspace(c, H, 3, 5), dtype=torch.uint8, device="cuda")
    g2.kv8_attention(c, x[:, 0], want, H, 8, 3, table, 3, lens, ws5, ws5.numel(), q_stride=3 * H * D, **exact)
    assert int(st) == 0 and (out - want).norm() <= 2 ** -19 * want.norm() and not (out == 7).any()
    if most == 5:
        g2.kv8_append(c, x[:, 1], x[:, 2], 8, 3, table, 3, ints(pos), row_stride=3 * H * D, **dict(kw, max_q=4))
        assert int(st) == -6


@pytest.mark.parametrize("name", CALLS)
def test_longest_table(name):
    """Positions near 2^31, where a tile past the last one no longer fits 32 bits, are refused."""
    f = CALLS[name]
    for page in (16, 128):
        for last in (2 ** 31 - 128, 2 ** 31 - 256 + page):
            assert code(lambda: f(cache(page_size=page), dict(table_stride=last // page))) == -6
        assert code(lambda: f(cache(page_size=page, n_kv_head=1), dict(table_stride=(2 ** 31 - 256) // page, n_rows=1, n_seq=1))) == no_device_memory()


def test_work_goes_by_the_rows_there_are():
    """One long prompt among many sequences with long tables: max_q times n_seq is far above the rows."""
    f = CALLS["attention"]
    call = dict(heads=32, n_seq=256, n_rows=2048 + 255, max_q=2048, q_start=CALLS_A, table_stride=8192)
    assert code(lambda: f(cache(n_kv_head=8), dict(call))) == no_device_memory()
    # as many rows as max_q allows is too much for the kernel's 32-bit counts
    assert code(lambda: f(cache(n_kv_head=8), dict(call, n_rows=2048 * 256, max_q=2048))) == -6
    assert code(lambda: f(cache(n_kv_head=8), dict(call, n_seq=2 ** 22, n_rows=2 ** 22))) == -6


def test_largest_scale():
    """A scale that passes fp32's range in powers of two (times log2 e) would make every score infinite or NaN."""
    f = CALLS["attention"]
    assert code(lambda: f(cache(), dict(scale=3.0e38))) == -1
    assert code(lambda: f(cache(), dict(scale=2.3e38))) == no_device_memory()


@pytest.mark.gpu
def test_2_27_runs():
    """So many (sequence, head) runs that 32 of each pass 32 bits: every output is written."""
    S, H, D = 2 ** 22, 32, 64
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 40 GB of device memory")
    k, v = (torch.randint(-127, 128, (1, H, 16, D), device="cuda", generator=gen(i)).to(torch.int8) for i in range(2))
    ks, vs = (torch.full((1, H), 2.0 ** -6, device="cuda") for _ in "kv")
    c = g2.kv8_cache(k, v, ks, vs)
    q, out = torch.zeros(S, H, D, dtype=torch.half, device="cuda"), torch.full((S, H, D), 9.0, dtype=torch.half, device="cuda")
    table, lens = torch.zeros(S, 1, dtype=torch.int32, device="cuda"), torch.ones(S, dtype=torch.int32, device="cuda")
    ws = torch.zeros(g2.kv8_attention_workspace(c, H, S, 1), dtype=torch.uint8, device="cuda")
    g2.kv8_attention(c, q, out, H, S, S, table, 1, lens, ws, ws.numel(), dtype=g2.G2_F16)
    want = (v[0, :, 0].float() * 2.0 ** -6).half()          # one key: its value, exact in fp16
    assert all(torch.equal(part, want.expand_as(part)) for part in out.split(2 ** 18))


@pytest.mark.gpu
def test_overlapping_rows_past_a_calls_work():
    """q_start that runs back and forth: half of the sequences have all the rows, together too much to count."""
    S, R, H, page, blocks = 4096, 64, 32, 128, 8192
    k = torch.ones(1, H, page, 64, dtype=torch.int8, device="cuda")
    c = g2.kv8_cache(k, k.clone(), torch.ones(1, H, device="cuda"), torch.ones(1, H, device="cuda"))
    q, out = torch.ones(R, H, 64, device="cuda"), torch.full((R, H, 64), 7.0, device="cuda")
    table, st = torch.zeros(S, blocks, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    back_and_forth = ints([0, R] * (S // 2) + [0])
    ws = torch.zeros(g2.kv8_attention_workspace(c, H, S, R), dtype=torch.uint8, device="cuda")
    kw = dict(q_start=back_and_forth, max_q=R, status=st)
    g2.kv8_attention(c, q, out, H, R, S, table, blocks, torch.full((S,), page * blocks, dtype=torch.int32, device="cuda"), ws, ws.numel(), **kw)
    assert int(st) == -6 and (out == 7).all() and not ws[:4096 * 4].any()
    st.zero_()   # few enough: the sequences with rows are computed
    g2.kv8_attention(c, q, out, H, R, S, table, blocks, torch.full((S,), 70, dtype=torch.int32, device="cuda"), ws, ws.numel(), **kw)
    assert int(st) == -6 and (out == 1).all()
