"""g2k_kv8_attention's bits do not depend on what ran before on its SMs."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g2():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import gpt2b200
    return gpt2b200


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def attend(g2, c, q, lens, table):
    S, H, D = q.shape
    out = torch.empty_like(q)
    ws = torch.zeros(g2.kv8_attention_workspace(c, H, S, 1), dtype=torch.uint8, device="cuda")
    g2.kv8_attention(c, q, out, H, S, S, table, table.shape[1], torch.full((S,), lens, dtype=torch.int32, device="cuda"), ws, ws.numel(),
                     scale=1.0)
    return out


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
def test_bits_after_other_kernels(g2, fmt, D):
    """One query a K/V head leaves columns of a tile idle.  What earlier calls left in shared memory there (codes of 448
    are NaN patterns of fp16) must not move the reference of the live column: V scales rise by 2^10 from one page to
    the next while the scores fall by as much."""
    f = g2.G2_KV_E4M3 if fmt == "e4m3" else g2.G2_KV_I8
    H, P, S = 4, 16, 200
    code = (lambda x: x.to(torch.float8_e4m3fn).view(torch.int8)) if fmt == "e4m3" else (lambda x: x.round().to(torch.int8))
    n = 16                                                     # pages: eight of each kind, so that every warp sees both
    k = torch.zeros(n, H, P, D, device="cuda")
    k[8:] = -1.0
    v = torch.randn(n, H, P, D, device="cuda", generator=gen(1)) * 30
    vs = torch.cat([torch.ones(8, H, device="cuda"), torch.full((8, H), 2.0 ** 10, device="cuda")])
    c = g2.kv8_cache(code(k), code(v), torch.ones(n, H, device="cuda"), vs, f)
    table = torch.arange(n, dtype=torch.int32, device="cuda").expand(S, n).contiguous()
    # scores of the later pages: -8 in powers of two, up to 1 / 8 more
    q = 8 * 0.6931 / D * (1 + torch.rand(S, H, 1, device="cuda", generator=gen(2)) / 8).expand(S, H, D).contiguous()
    got = []
    for byte in (0x7e, 0x38, 0x00, 0x55):
        fill = torch.full((32, 16, 64, D), byte, dtype=torch.uint8, device="cuda").view(torch.int8)
        fc = g2.kv8_cache(fill, fill, torch.ones(32, 16, device="cuda"), torch.ones(32, 16, device="cuda"), f)
        many = torch.arange(32, dtype=torch.int32, device="cuda").repeat(64, 2)
        attend(g2, fc, torch.randn(64, 16, D, device="cuda", generator=gen(3)), 64 * 64, many)
        got.append(attend(g2, c, q, n * P, table))
    assert got[0].isfinite().all()
    assert all(torch.equal(got[0], g) for g in got[1:])


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_read_back_right_after_writing(g2, fmt):
    """append, gather and attention one after the other, each started while the one before runs, on the same pages."""
    H, P, D, S, n = 16, 32, 64, 6, 90
    f = g2.G2_KV_E4M3 if fmt == "e4m3" else g2.G2_KV_I8
    k, v = (torch.zeros(S * 3, H, P, D, dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.ones(S * 3, H, device="cuda") for _ in "kv")
    c = g2.kv8_cache(k, v, ks, vs, f)
    table = torch.arange(S * 3, dtype=torch.int32, device="cuda").view(S, 3)
    pos, starts = torch.zeros(S, dtype=torch.int32, device="cuda"), torch.arange(0, S * n + 1, n, dtype=torch.int32, device="cuda")
    x = torch.randn(8, 2, S * n, H, D, device="cuda", generator=gen(4))
    back, outs = torch.zeros_like(x), torch.zeros(8, S, H, D, device="cuda")
    ws = torch.zeros(g2.kv8_attention_workspace(c, H, S, 1), dtype=torch.uint8, device="cuda")
    kw, lens = dict(q_start=starts, max_q=n), torch.full((S,), n, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()

    def step(i, wait):
        for call in (lambda: g2.kv8_append(c, x[i, 0], x[i, 1], S * n, S, table, 3, pos, **kw),
                     lambda: g2.kv8_gather(c, back[i, 0], back[i, 1], S * n, S, table, 3, pos, **kw),
                     lambda: g2.kv8_attention(c, x[i, 0, :S], outs[i], H, S, S, table, 3, lens, ws, ws.numel())):
            call()
            if wait:
                torch.cuda.synchronize()
    for i in range(8):
        step(i, False)
    torch.cuda.synchronize()
    got = back.clone(), outs.clone()
    for i in range(8):
        step(i, True)
    assert torch.equal(got[0], back) and torch.equal(got[1], outs)
    assert ((back - x).abs() <= x.abs().max() / 14).all()       # half a step of e4m3 at its largest is 1 / 28 of it
