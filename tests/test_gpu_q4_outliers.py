"""g2k_matvec_q4 where the values of a row of x lie far apart.

A column whose codes are 0 at a row's large values must not inherit their step:
every output is held to the fp32 bound over its own products,
(K / 16 + 16) 2^-22 sum_k |x'_k w_kn| (as in test_gpu_q4.py: one 2^-22 of the
partial sum for each 16 terms and 16 more for splits and reductions), plus half a
step of its type; fp16's least step is 2^-24.
"""
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


def values(g2, p, N, K, group):
    out = torch.empty(K, N, device="cuda")
    g2.q4_unpack(p, out, N, K, group)
    return out.double()


def check(g2, x, W, group, dtype=0, ga=None, be=None):
    M, (K, N) = len(x), W.shape
    p = torch.empty(g2.q4_bytes(N, K, group), dtype=torch.uint8, device="cuda")
    g2.q4_pack(W, p, N, K, group)
    w, xd = values(g2, p, N, K, group), x.double()
    size = xd.abs()
    if ga is not None:
        mu = xd.mean(1, keepdim=True)
        rstd = (xd.var(1, correction=0, keepdim=True) + 1e-5).rsqrt()
        size = (size + mu.abs()) * rstd * ga.double().abs() + be.double().abs()
        xd = (xd - mu) * rstd * ga.double() + be.double()
    y = torch.empty(M, N, device="cuda", dtype=x.dtype)
    g2.matvec_q4(x, p, y, M, N, K, group, ln_gamma=ga, ln_beta=be, dtype=dtype)
    want, S = xd @ w, size @ w.abs()
    half = torch.finfo(x.dtype).eps / 2
    tol = (K / 16 + 16) * 2 ** -22 * S + half * want.abs() + (2 ** -25 if dtype else 0)
    good = (y.double() - want).abs() <= tol
    # half a step past the type's largest value (65520 for fp16) and above, rounding gives an infinity
    top = torch.finfo(x.dtype).max * (1 + half / 2)
    good |= y.isinf() & (y.sign() == want.sign()) & (want.abs() + tol >= top)
    assert good.all()


SHAPES = [(1600, 400, 64), (640, 5000, 32), (2100, 96, 128), (9000, 64, 128), (333, 130, 32)]


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("ratio", [3e2, 1e6, 1e10])
@pytest.mark.parametrize("K,N,group", SHAPES)
def test_large_values_that_meet_code_zero(g2, M, ratio, K, N, group):
    """A few values of each row are `ratio` times the others and meet codes of 0 in most columns."""
    x = torch.randn(M, K, device="cuda", generator=gen(K + M))
    W = torch.randn(K, N, device="cuda", generator=gen(N)) * 0.05
    for m in range(M):
        at = torch.randperm(K, device="cuda", generator=gen(m))[:3]
        x[m, at] *= ratio
        W[at, : N - N // 8] = 0
    check(g2, x, W, group)


@pytest.mark.parametrize("M", [1, 2, 4, 8, 16])
def test_columns_of_one_row(g2, M):
    """W picks single values of x, each held to its own size; rows from 2^-30 to 2^30."""
    K = 700
    x = torch.randn(M, K, device="cuda", generator=gen(3)) * torch.exp2(torch.linspace(-15, 15, K, device="cuda"))
    check(g2, x, torch.eye(K, device="cuda"), 32)


@pytest.mark.parametrize("M", [1, 2, 3, 8, 16])
@pytest.mark.parametrize("K,N", [(1600, 400), (1000, 83), (999, 40)])
def test_fp16_rows(g2, M, K, N):
    """fp16's whole range in a row: 60000 beside values near 1 / 1000."""
    x = torch.randn(M, K, device="cuda", generator=gen(M)) * 1e-3
    W = torch.randn(K, N, device="cuda", generator=gen(N))
    x[:, 5], x[:, K // 2] = 60000.0, -50000.0
    W[5, :N // 2], W[K // 2, :N // 2] = 0, 0
    check(g2, x.half(), W, 64, g2.G2_F16)


@pytest.mark.parametrize("M", [1, 2, 3, 8, 16])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_layer_norm_weights_far_apart(g2, M, dtype):
    """LayerNorm whose gamma and beta lie 10^8 apart."""
    K, N = 1600, 300
    x = torch.randn(M, K, device="cuda", generator=gen(M))
    ga, be = torch.ones(K, device="cuda"), torch.randn(K, device="cuda", generator=gen(1)) * 0.1
    W = torch.randn(K, N, device="cuda", generator=gen(2)) * 0.05
    ga[7], ga[900], be[901] = 1e8, -1e8, 3e8
    W[[7, 900, 901], :200] = 0
    half = dtype == "f16"
    check(g2, x.half() if half else x, W, 64, g2.G2_F16 if half else g2.G2_F32, ga=ga, be=be)
