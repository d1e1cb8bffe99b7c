"""Every form that g2k_matvec_q4 takes x in, at the shapes where its staging or its
sharing of work changes: K that ends inside a chunk or is cut into slices, rows
that are copied as they are or one by one, more tiles than are summed at a time.
Bounds: those of test_gpu_q4.py.
"""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_q4 import check_matvec  # noqa: E402


@pytest.fixture(scope="module")
def g2():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import gpt2b200
    return gpt2b200


@pytest.mark.parametrize("K,N", [(5, 48), (100, 1601), (129, 6400), (1004, 6400), (1003, 1601), (3400, 6400), (8192, 1601), (20000, 48)])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16])
def test_fp16_rows(g2, M, K, N):
    for group in (32, 64, 128):
        check_matvec(g2, M, K, N, group, "f16", residual=group == 64)


@pytest.mark.parametrize("K,N", [(100, 6400), (3000, 6400), (2999, 1601), (8192, 4800), (32768, 48)])
@pytest.mark.parametrize("M", [2, 4, 6, 8, 12])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_layer_norm_in_slices(g2, M, K, N, dtype):
    for group in (32, 128):
        check_matvec(g2, M, K, N, group, dtype, ln=True, bias=True)


@pytest.mark.parametrize("M", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_more_tiles_than_are_summed_at_a_time(g2, M, dtype):
    check_matvec(g2, M, 100, 170000, 32, dtype, bias=True)
    check_matvec(g2, M, 1028, 90001, 128, dtype, ln=M != 4)


@pytest.mark.parametrize("M,K,N,dtype", [(16, 4224, 85000, "f16"), (8, 2816, 80000, "f32"), (4, 4800, 80000, "f32")])
def test_slices_and_many_tiles(g2, M, K, N, dtype):
    check_matvec(g2, M, K, N, 64, dtype)


@pytest.mark.parametrize("M", [3, 5, 16])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows_that_begin_anywhere(g2, M, dtype):
    """x, residual and y aligned to their elements only."""
    dt, code = (torch.float32, g2.G2_F32) if dtype == "f32" else (torch.float16, g2.G2_F16)
    g = torch.Generator(device="cuda").manual_seed(M)
    K, N = 640, 320
    W = torch.randn(K, N, device="cuda", generator=g) * 0.05
    p = torch.empty(g2.q4_bytes(N, K, 64), dtype=torch.uint8, device="cuda")
    g2.q4_pack(W, p, N, K, 64)
    x, r = torch.randn(M, K, device="cuda", generator=g).to(dt), torch.randn(M, N, device="cuda", generator=g).to(dt)
    want, far = torch.empty(M, N, device="cuda", dtype=dt), torch.full((M * N + 9,), 3.0, device="cuda", dtype=dt)
    g2.matvec_q4(x, p, want, M, N, K, 64, residual=r, dtype=code)
    x1, r1 = torch.cat([x.new_zeros(1), x.flatten()])[1:], torch.cat([r.new_zeros(3), r.flatten()])[3:]
    g2.matvec_q4(x1, p, far[5:], M, N, K, 64, residual=r1, dtype=code)
    assert torch.equal(far[5:5 + M * N].view(M, N), want)
    assert (far[:5] == 3).all() and (far[5 + M * N:] == 3).all()
