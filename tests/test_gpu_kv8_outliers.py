"""g2k_kv8_attention where a row's numbers lie far apart.

Bounds: as in test_gpu_kv8.py an output is within
(2^-17 A + 2^-21 + (n / 16 + 16) 2^-22) sum_j p_j |v_j| of the exact one, with
A the largest sum_d |q_d k_d| * scale over the row's keys (not of |q| by itself),
and half a step of its type; a weight far below the largest ends 2^-42 below it
(n weights times a code of at most 127 or 448).
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TOP = {"i8": 127.0, "e4m3": 448.0}


@pytest.fixture(scope="module")
def g2():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import gpt2b200
    return gpt2b200


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def codes(x, fmt):
    return x.round().clamp(-127, 127).to(torch.int8) if fmt == "i8" else x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.int8)


def values(c, fmt):
    return c.double() if fmt == "i8" else c.view(torch.float8_e4m3fn).double()


def check(g2, fmt, k, v, ks, vs, q, n, scale):
    """One sequence on pages 0, 1, ..., query rows that all see n keys; k, v are codes [pages, heads, P, D]."""
    pages, H, P, D = k.shape
    rows, Hq, _ = q.shape
    c = g2.kv8_cache(k, v, ks, vs, g2.G2_KV_E4M3 if fmt == "e4m3" else g2.G2_KV_I8)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(rows, pages).contiguous()
    lens = torch.full((rows,), n, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    ws = torch.zeros(g2.kv8_attention_workspace(c, Hq, rows, 1), dtype=torch.uint8, device="cuda")
    g2.kv8_attention(c, q, out, Hq, rows, rows, table, pages, lens, ws, ws.numel(), scale=scale,
                     dtype=g2.G2_F16 if q.dtype == torch.half else g2.G2_F32)
    kk, vv = ((values(x, fmt) * s.double()[:, :, None, None]).transpose(0, 1).reshape(H, -1, D)[:, :n] for x, s in ((k, ks), (v, vs)))
    qq = q.double().view(rows, H, -1, D)
    p = (torch.einsum("rhgd,hkd->rhgk", qq, kk) * scale).softmax(-1)
    A = torch.einsum("rhgd,hkd->rhgk", qq.abs(), kk.abs()).amax(-1, keepdim=True) * scale
    want, size = torch.einsum("rhgk,hkd->rhgd", p, vv), torch.einsum("rhgk,hkd->rhgd", p, vv.abs())
    most = (p * vs.double().repeat_interleave(P, 0)[:n].T[:, None]).amax(-1, keepdim=True) * TOP[fmt]
    half = torch.finfo(q.dtype).eps / 2
    tol = (2 ** -17 * A + 2 ** -21 + (n / 16 + 16) * 2 ** -22) * size + n * 2 ** -42 * most + half * want.abs()
    if q.dtype == torch.half:
        tol = tol + 2 ** -25
    assert ((out.double().view_as(want) - want).abs() <= tol).all()


@pytest.mark.parametrize("fmt,ratio", [("i8", 1e4), ("i8", 1e7), ("e4m3", 1e4), ("e4m3", 1e7), ("e4m3", 1e9)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 5, 12])
def test_large_queries_that_meet_code_zero(g2, fmt, ratio, D, group):
    """Two dimensions of each query are `ratio` times the others, and the keys' codes there are 0."""
    H, P, n = 2, 32, 300
    k = codes(torch.randn(10, H, P, D, device="cuda", generator=gen(1)) * (40 if fmt == "i8" else 100), fmt)
    v = codes(torch.randn(10, H, P, D, device="cuda", generator=gen(2)) * (40 if fmt == "i8" else 100), fmt)
    q = torch.randn(3, H * group, D, device="cuda", generator=gen(3))
    k[..., 3] = k[..., D - 9] = 0
    q[..., 3] *= ratio
    q[..., D - 9] = -ratio
    s = torch.full((10, H), 0.02, device="cuda")
    check(g2, fmt, k, v, s, s, q, n, D ** -0.5)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_fp16_queries_of_all_sizes(g2, fmt):
    """fp16's whole range in a query: 60000 beside 1 / 100."""
    H, P, n, D = 3, 16, 100, 64
    k = codes(torch.randn(7, H, P, D, device="cuda", generator=gen(1)) * 40, fmt)
    v = codes(torch.randn(7, H, P, D, device="cuda", generator=gen(2)) * 40, fmt)
    q = torch.randn(2, H, D, device="cuda", generator=gen(3)) * 0.01
    k[..., 5] = 0
    q[..., 5] = 60000.0
    s = torch.full((7, H), 0.5, device="cuda")
    check(g2, fmt, k, v, s, s, q.half(), n, 1.0)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("gap", [15.0, 17.3, 18.3, 19.7, 20.1])
@pytest.mark.parametrize("D", [64, 128])
def test_small_weights_beside_a_large_one(g2, fmt, gap, D):
    """The first key takes nearly all of the weight and has a value of 0: what is left are weights e^-gap of it."""
    H, P, n = 2, 64, 16
    k = torch.zeros(4, H, P, D, dtype=torch.int8, device="cuda")
    one = codes(torch.ones(1, device="cuda"), fmt)
    k[0, :, 0, 0] = one
    v = codes(70 + 20 * torch.rand(4, H, P, D, device="cuda", generator=gen(4)), fmt)
    v[0, :, 0] = 0
    q = torch.zeros(1, H, D, device="cuda")
    q[..., 0] = gap
    s = torch.ones(4, H, device="cuda")
    check(g2, fmt, k, v, s, s, q, n, 1.0)
