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
