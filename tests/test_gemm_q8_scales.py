"""Scales of the 8-bit GEMM whose product, or product with alpha, leaves the fp32 range although the result does not; and the
library's choice of a kernel over many heights, with sums that fp32 holds exactly."""
import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
THIN, PAIR = 1, 2


@pytest.fixture(scope="module")
def G():
    from decx_b200 import gemm
    return gemm


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _operand(dev, g, rows, cols, size):
    buf = torch.full((rows, -(-cols // 16) * 16), 0x7F, dtype=torch.uint8, device=dev)
    v = buf.view(E4M3)[:, :cols]
    v.copy_((torch.randn(rows, cols, generator=g, device=dev) * size).clamp(-448, 448).to(E4M3))
    return v


# magnitude of the operands' values, of their scales, and alpha
RANGES = [(100, 1e-22, 1e-20, 1.0),          # the scales' product is subnormal
          (100, 1e-30, 1e-28, 1e22),         # ... zero; alpha brings it back
          (0.002, 1e24, 1e15, 1.0),          # ... infinite, of small sums
          (100, 1e30, 1e-32, 1.0),           # one large, one small
          (100, 1e-32, 1e30, -3.0),
          (100, 1e-14, 1e26, 1e-28),         # alpha times the first scale is subnormal
          (100, 1e20, 1e-30, 1e20),          # ... infinite
          (100, 1e-30, 1e20, 1e20)]


@gpu
@pytest.mark.parametrize("tile", [THIN, PAIR])
@pytest.mark.parametrize("shape", [(3, 200, 300), (20, 130, 2048), (100, 300, 4096), (300, 520, 512), (130, 260, 4096)])
def test_scales_far_from_one(G, dev, shape, tile):
    M, N, K = shape
    g = torch.Generator(device=dev).manual_seed(M + N + K)
    for size, ma, mb, alpha in RANGES:
        A, B = _operand(dev, g, M, K, size), _operand(dev, g, N, K, size)
        sa = (torch.rand(M, generator=g, device=dev) + 0.5) * ma
        sb = (torch.rand(N, generator=g, device=dev) + 0.5) * mb
        sa[M // 2] = 0.0
        a, b = A.float().double(), B.float().double()
        factor = alpha * sa.double()[:, None] * sb.double()[None, :]
        ref, mag = (a @ b.t()) * factor, (a.abs() @ b.abs().t()) * factor.abs()
        assert 1e-37 < float(mag[0].max()) < 1e38
        # as for ordinary scales: truncating fp32 sums, and a few half steps for the factors; results down to 2^-126
        tol = (K / 32 + 16) * 2.0 ** -23 * mag + 2.0 ** -149
        for C, beta in ((None, None), (torch.randn(M, N, generator=g, device=dev) * float(mag[0].max()), 0.5)):
            D = G.gemm_q8(A, sa, B, sb, C=C, alpha=alpha, beta=beta, out_dtype=torch.float32, tile=tile)
            torch.cuda.synchronize()
            want, most = (ref, tol) if C is None else (ref + beta * C.double(), tol + 2.0 ** -23 * beta * C.double().abs())
            err = (D.double() - want).abs()
            assert torch.all(err <= most), ((size, ma, mb, alpha), float((err / most).max()))
            assert torch.all(D[M // 2] == (0.0 if C is None else D[M // 2]))


@gpu
@pytest.mark.parametrize("tile", [THIN, PAIR])
def test_one_such_row_does_not_change_the_others(G, dev, tile):
    g = torch.Generator(device=dev).manual_seed(3)
    A, B = _operand(dev, g, 150, 700, 100), _operand(dev, g, 300, 700, 100)
    sa, sb = torch.rand(150, generator=g, device=dev) + 0.5, torch.rand(300, generator=g, device=dev) + 0.5
    D0 = G.gemm_q8(A, sa, B, sb, out_dtype=torch.float32, tile=tile).clone()
    sa[77] = 1e-35
    D1 = G.gemm_q8(A, sa, B, sb, out_dtype=torch.float32, tile=tile)
    torch.cuda.synchronize()
    rows = torch.arange(150, device=dev) != 77
    # the factors' product may be rounded another way: three roundings each
    assert torch.all((D0[rows] - D1[rows]).abs() <= 6 * 2.0 ** -24 * D0[rows].abs())


@gpu
@pytest.mark.parametrize("N,K", [(384, 640), (4096, 2048), (1000, 4100)])
def test_library_choice_at_every_height(G, dev, N, K):
    """Small whole numbers and powers of two as scales: all sums are exact, so every kernel that the library may choose gives
    the same bits."""
    g = torch.Generator(device=dev).manual_seed(N)
    A = _operand(dev, g, 1100, K, 0)
    A.copy_(torch.randint(-4, 5, A.shape, generator=g, device=dev).float().to(E4M3))
    B = _operand(dev, g, N, K, 0)
    B.copy_(torch.randint(-4, 5, B.shape, generator=g, device=dev).float().to(E4M3))
    sa = 2.0 ** torch.randint(-3, 4, (1100,), generator=g, device=dev).float()
    sb = 2.0 ** torch.randint(-3, 4, (N,), generator=g, device=dev).float()
    want = ((A.float().double() @ B.float().double().t()) * sa.double()[:, None] * sb.double()[None, :]).float()
    status = G.new_status(dev)
    for M in (1, 2, 15, 16, 17, 31, 33, 48, 64, 65, 96, 127, 128, 129, 160, 200, 255, 256, 257, 300, 384, 511, 513, 640, 768, 1000, 1100):
        D = G.gemm_q8(A[:M], sa[:M], B, sb, out_dtype=torch.float32, status=status)
        torch.cuda.synchronize()
        assert int(status.item()) == 0 and torch.equal(D, want[:M]), M
