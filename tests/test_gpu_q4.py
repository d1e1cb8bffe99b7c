"""Weights in 4 bits on the GPU: g2k_q4_pack / g2k_q4_unpack and g2k_matvec_q4
against the definitions in 64 bits.

Packing is exact: the values read back must equal, bit for bit, code * scale
with scale = bf16(fp32(max|w| / 7)) and code the nearest integer of the exact
quotient.  The product is held to two bounds, both over S = sum_k |x'| |w| of
each output:
  * every output: each of the K / 16 accumulation steps may be off by 2^-22 of
    the largest partial sum (<= S), 16 more for the operands' split and the
    reductions, plus half a step of the output type;
  * the 2-norm over the outputs: 2^-20 of the result's (the roundings of 2^-23
    per term are independent, so they grow as the sum itself does).
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


def quantise(W, group):
    """Values in 64 bits of the 4-bit form of W [K, N] (fp32)."""
    K, N = W.shape
    out = torch.empty(K, N, dtype=torch.double, device=W.device)
    for k in range(0, K, group):
        w = W[k:k + group].double()
        peak = w.abs().amax(0)
        s = (peak / 7).float().bfloat16().double()
        c = torch.where(s > 0, (w / torch.where(s > 0, s, 1.0)).round().clamp(-7, 7), 0.0)
        out[k:k + group] = torch.where(peak.isfinite(), c * s, torch.nan)
    return out


def pack(g2, W, group, transposed=False, dtype=0):
    N, K = W.shape if transposed else W.shape[::-1]
    p = torch.full((g2.q4_bytes(N, K, group),), 0x5a, dtype=torch.uint8, device="cuda")
    g2.q4_pack(W, p, N, K, group, transposed=transposed, dtype=dtype)
    return p


def unpack(g2, p, N, K, group):
    out = torch.full((K, N), 7.0, device="cuda")
    g2.q4_unpack(p, out, N, K, group)
    return out


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K,N", [(1, 1), (31, 15), (64, 16), (65, 17), (200, 33), (768, 100), (1600, 7)])
def test_pack_is_exact(g2, K, N, group):
    W = torch.randn(K, N, device="cuda", generator=gen(K + N))
    W[:, 0] = 0                                                     # a zero scale
    W[::3, N // 2] = W[0, N // 2] * 0.5                             # many quotients on a border
    W = W * torch.exp2(torch.randint(-60, 60, (1, N), device="cuda", generator=gen(1)).float())
    assert torch.equal(unpack(g2, pack(g2, W, group), N, K, group).double(), quantise(W, group))


def test_pack_borders(g2):
    """Quotients on and next to every border k + 1/2 of a scale that is not a power of two."""
    s = 0.2109375   # a bf16 value; 7 s is the group's largest
    at = (torch.arange(-7, 7, dtype=torch.double) + 0.5) * s
    f = at.float()
    w = torch.cat([f, torch.nextafter(f, f + 1), torch.nextafter(f, f - 1), torch.tensor([7 * s])]).cuda()[:, None]
    assert torch.equal(unpack(g2, pack(g2, w, 64), 1, len(w), 64).double(), quantise(w, 64))


def test_pack_non_finite(g2):
    W = torch.randn(96, 20, device="cuda", generator=gen(3))
    W[40, 3], W[5, 4], W[70, 19] = float("inf"), float("nan"), float("-inf")
    got = unpack(g2, pack(g2, W, 32), 20, 96, 32)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[32:64, 3] = bad[0:32, 4] = bad[64:96, 19] = True
    assert torch.equal(got.isnan(), bad)


@pytest.mark.parametrize("transposed", [False, True])
def test_pack_types_and_layouts(g2, transposed):
    W = torch.randn(130, 37, device="cuda", generator=gen(4)).half()
    src = W.t().contiguous() if transposed else W
    got = unpack(g2, pack(g2, src, 32, transposed, g2.G2_F16), 37, 130, 32)
    assert torch.equal(got.double(), quantise(W.float(), 32))


def gelu(y):
    return 0.5 * y * (1 + torch.tanh(0.7978845608 * (y + 0.044715 * y ** 3)))


def check_matvec(g2, M, K, N, group, dtype="f32", ln=False, bias=False, act=False, residual=False, seed=0, stream=None,
                 in_place=False, x=None):
    g = gen(seed + K * 31 + N)
    dt, code = (torch.float32, g2.G2_F32) if dtype == "f32" else (torch.float16, g2.G2_F16)
    W = torch.randn(K, N, device="cuda", generator=g) * 0.05
    x = (torch.randn(M, K, device="cuda", generator=g) + 0.3 if x is None else x).to(dt)
    ga, be = 1 + 0.3 * torch.randn(K, device="cuda", generator=g), torch.randn(K, device="cuda", generator=g) * 0.2
    b = torch.randn(N, device="cuda", generator=g)
    y = torch.randn(M, N, device="cuda", generator=g).to(dt)
    r = y.clone() if in_place else torch.randn(M, N, device="cuda", generator=g).to(dt)
    p = pack(g2, W, group)
    w = quantise(W, group)
    xd = x.double()
    size = xd.abs()
    if ln:
        mu = xd.mean(1, keepdim=True)
        rstd = (xd.var(1, correction=0, keepdim=True) + 1e-5).rsqrt()
        size = (size + mu.abs()) * rstd * ga.double().abs() + be.double().abs()
        xd = (xd - mu) * rstd * ga.double() + be.double()
    want, S = xd @ w, size @ w.abs()
    if bias:
        want, S = want + b.double(), S + b.double().abs()
    if act:
        want, S = gelu(want), S * 1.2      # |gelu'| < 1.13, and its own rounding
    if residual:
        want, S = want + r.double(), S + r.double().abs()
    if stream is not None:
        torch.cuda.synchronize()
    g2.matvec_q4(x, p, y, M, N, K, group, bias=b if bias else None, residual=(y if in_place else r) if residual else None,
                 gelu=act, ln_gamma=ga if ln else None, ln_beta=be if ln else None, dtype=code,
                 stream=0 if stream is None else stream.cuda_stream)
    torch.cuda.synchronize()
    half = torch.finfo(dt).eps / 2
    assert ((y.double() - want).abs() <= (K / 16 + 16) * 2 ** -22 * S + half * want.abs() + 2 ** -25).all()
    assert (y.double() - want).norm() <= (2 ** -20 + (half if dtype == "f16" else 0)) * S.norm().clamp(min=0) / S.norm() * want.norm() + 1e-30 \
        or M * N < 8
    return y


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 13, 16])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows(g2, M, dtype):
    check_matvec(g2, M, 768, 1000, 64, dtype, bias=True)


@pytest.mark.parametrize("K,N", [(1, 1), (5, 3), (64, 16), (63, 50), (65, 17), (129, 768), (768, 2304), (1000, 31), (1600, 1601),
                                 (6400, 1600), (4096, 50257), (20000, 48), (32768, 20)])
@pytest.mark.parametrize("M", [1, 7])
def test_shapes(g2, K, N, M):
    for group in (32, 64, 128):
        check_matvec(g2, M, K, N, group, residual=True)


@pytest.mark.parametrize("M", [1, 4, 16])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("K,N", [(1600, 6400), (333, 65), (8192, 512), (32768, 32)])
def test_fused_parts(g2, M, K, N, dtype):
    check_matvec(g2, M, K, N, 128, dtype, ln=True, bias=True, act=True, residual=True)
    check_matvec(g2, M, K, N, 32, dtype, ln=True)


def test_residual_in_place(g2):
    check_matvec(g2, 3, 768, 768, 64, residual=True, in_place=True)


@pytest.mark.parametrize("size", [1e-12, 1e-5, 1e5, 1e20])
def test_scale_of_x(g2, size):
    """x far outside fp16's range keeps fp32 accuracy: every row is scaled by itself."""
    K, N = 640, 96
    x = torch.randn(4, K, device="cuda", generator=gen(9)) * torch.tensor([[size], [1.0], [1 / size], [0.0]], device="cuda")
    W = torch.randn(K, N, device="cuda", generator=gen(10))
    y = torch.empty(4, N, device="cuda")
    g2.matvec_q4(x, pack(g2, W, 64), y, 4, N, K, 64)
    want = x.double() @ quantise(W, 64)
    S = x.double().abs() @ quantise(W, 64).abs()
    assert ((y.double() - want).abs() <= (K / 16 + 16) * 2 ** -22 * S).all()
    assert (y[3] == 0).all()


@pytest.mark.parametrize("M", [1, 3, 5])
def test_largest_x(g2, M):
    """Values in fp32's last power of two, 2^127 and above."""
    K, N = 200, 96
    x = torch.randn(M, K, device="cuda", generator=gen(18)) * 1e38
    x[:, 3], x[:, 100], x[:, 150] = 3.4e38, -3.2e38, 2.0 ** 127
    x = x.clamp(-3.4e38, 3.4e38)
    W = torch.randn(K, N, device="cuda", generator=gen(19)) * 1e-4
    y = torch.empty(M, N, device="cuda")
    g2.matvec_q4(x, pack(g2, W, 64), y, M, N, K, 64)
    want = x.double() @ quantise(W, 64)
    S = x.double().abs() @ quantise(W, 64).abs()
    assert ((y.double() - want).abs() <= (K / 16 + 16) * 2 ** -22 * S).all()


def test_non_finite_rows_stay_apart(g2):
    """A NaN or infinity in one row reaches that row's outputs and no other's."""
    x = torch.randn(3, 256, device="cuda", generator=gen(11))
    x[1, 7], x[2, 9] = float("nan"), float("inf")
    W = torch.randn(256, 64, device="cuda", generator=gen(12))
    y = torch.empty(3, 64, device="cuda")
    g2.matvec_q4(x, pack(g2, W, 32), y, 3, 64, 256, 32)
    assert y[0].isfinite().all() and y[1].isnan().all() and not y[2].isfinite().any()


def test_same_bits_each_time(g2):
    a = check_matvec(g2, 5, 1600, 4801, 32, ln=True, bias=True)
    for _ in range(3):
        assert torch.equal(a, check_matvec(g2, 5, 1600, 4801, 32, ln=True, bias=True))


def test_row_alone_has_the_same_bits(g2):
    """A row's result does not depend on the other rows of the call (no row: another kernel)."""
    x = torch.randn(8, 768, device="cuda", generator=gen(13))
    W = torch.randn(768, 320, device="cuda", generator=gen(14))
    p, y, one = pack(g2, W, 64), torch.empty(8, 320, device="cuda"), torch.empty(1, 320, device="cuda")
    g2.matvec_q4(x, p, y, 8, 320, 768, 64)
    for m in range(8):
        g2.matvec_q4(x[m], p, one, 1, 320, 768, 64)
        torch.testing.assert_close(one[0], y[m], rtol=0, atol=float(y.abs().max()) * 2 ** -20)


def test_streams_and_capture(g2):
    """Two streams at once, and a captured call replayed on new contents."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    W = torch.randn(1600, 1600, device="cuda", generator=gen(15))
    p = pack(g2, W, 64)
    xs = torch.randn(2, 40, 2, 1600, device="cuda", generator=gen(16))
    ys = torch.empty(2, 40, 2, 1600, device="cuda")
    torch.cuda.synchronize()
    for i in range(40):
        for k, st in enumerate((a, b)):
            g2.matvec_q4(xs[k, i], p, ys[k, i], 2, 1600, 1600, 64, stream=st.cuda_stream)
    torch.cuda.synchronize()
    want = xs.double() @ quantise(W, 64)
    assert (ys - want).norm() <= 2 ** -20 * want.norm()
    x, y = xs[0, 0].clone(), torch.empty(2, 1600, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g2.matvec_q4(x, p, y, 2, 1600, 1600, 64, stream=torch.cuda.current_stream().cuda_stream)
    for i in (3, 5):
        x.copy_(xs[1, i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ys[1, i])


def test_writes_nothing_else(g2):
    for M, N, K in ((1, 37, 100), (16, 50, 129)):
        y = torch.full((M * N + 64,), 3.5, device="cuda")
        W = torch.randn(K, N, device="cuda", generator=gen(17))
        x = torch.randn(M, K, device="cuda", generator=gen(18))
        g2.matvec_q4(x, pack(g2, W, 32), y, M, N, K, 32)
        assert (y[M * N:] == 3.5).all() and not (y[:M * N] == 3.5).any()
        n = g2.q4_bytes(N, K, 32)
        p = torch.full((n + 512,), 0x5a, dtype=torch.uint8, device="cuda")
        g2.q4_pack(W, p, N, K, 32)
        assert (p[n:] == 0x5a).all()
