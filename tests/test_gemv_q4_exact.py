"""4-bit products whose sums fp32 holds exactly, so that a lost column, group or piece of a long row shows; and weights that
are their own zero point."""
import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def Bl():
    from decx_b200 import blas
    return blas


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _case(dev, rows, cols, group, n, zeros, x8, seed):
    """Whole numbers: |x| <= 2, z <= 31, scales 1 or 2.  A sum of 65536 terms q x or z x is below 2^23."""
    g = torch.Generator(device=dev).manual_seed(seed)
    groups = -(-cols // group)
    q = torch.randint(0, 16, (rows, cols), generator=g, device=dev, dtype=torch.uint8)
    s = 2.0 ** torch.randint(0, 2, (rows, groups), generator=g, device=dev).half()
    z = torch.randint(0, 32, (rows, groups), generator=g, device=dev, dtype=torch.uint8) if zeros else None
    x = torch.randint(-2, 3, (n, cols), generator=g, device=dev).float()
    xs = 2.0 ** torch.randint(-2, 3, (n,), generator=g, device=dev).float() if x8 else None
    return q, s, z, x, x.to(E4M3 if x8 else torch.float16), xs


def _exact(q, s, z, x, xs, group):
    at = torch.arange(q.shape[1], device=q.device) // group
    w = (q.double() - (z.double()[:, at] if z is not None else 8.0)) * s.double()[:, at]
    return (x.double() @ w.t()) * (xs.double()[:, None] if xs is not None else 1.0)


SHAPES = [(33, 4096), (65, 4099), (40, 8191), (70, 16384), (9, 16385), (40, 20001), (33, 40000), (50, 50001), (17, 65535), (17, 65536)]


@gpu
@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_long_rows_exactly(Bl, dev, shape, group, zeros, x8):
    rows, cols = shape
    for n in (1, 8, 9, 16):
        q, s, z, x, v, xs = _case(dev, rows, cols, group, n, zeros, x8, cols + n)
        y = Bl.gemv_q4(Bl.pack_q4(q), s, v, group, zeros=z, x_scales=xs)
        torch.cuda.synchronize()
        assert torch.equal(y.double(), _exact(q, s, z, x, xs, group)), n


@gpu
@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("cols", [257, 4099, 20001, 65536])
def test_every_piece_of_a_row_counts(Bl, dev, cols, group, x8):
    """Sixteen vectors (and the first eight of them) that have one entry each: at the ends of the row, of its groups, of the
    pieces of 128 and 256 columns, and somewhere."""
    q, s, z, x, v, xs = _case(dev, 50, cols, group, 16, True, x8, 11)
    places = [0, 1, 31, 32, 127, 128, 255, 256, cols // 2, cols // 3, cols - 2, cols - 1, cols - cols % 128 - 1, cols - cols % 256 - 1,
              max(0, cols - 33), max(0, cols - 129)]
    x.zero_()
    for k, at in enumerate(places):
        x[k, at] = 1.0
    v = x.to(v.dtype)
    W = Bl.pack_q4(q)
    for n in (8, 16):
        y = Bl.gemv_q4(W, s, v[:n], group, zeros=z, x_scales=xs[:n] if x8 else None)
        torch.cuda.synchronize()
        assert torch.equal(y.double(), _exact(q, s, z, x[:n], xs[:n] if x8 else None, group))


@gpu
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("cols", [300, 4096, 20001])
def test_weights_that_are_their_zero_point(Bl, dev, cols, group):
    """q = z throughout stands for zeros.  Sums of q x and of x are made apart, so what is left is their rounding: (cols / 16 +
    32) steps of 2^-23 at the very most, each of the sum of q |x|; exactly zero where all sums are exact."""
    g = torch.Generator(device=dev).manual_seed(cols)
    groups = -(-cols // group)
    z = torch.randint(0, 16, (40, groups), generator=g, device=dev, dtype=torch.uint8)
    q = z.repeat_interleave(group, 1)[:, :cols].contiguous()
    s = (torch.rand(40, groups, generator=g, device=dev) + 0.5).half()
    W = Bl.pack_q4(q)
    for n in (1, 16):
        x = torch.randn(n, cols, generator=g, device=dev).half()
        y = Bl.gemv_q4(W, s, x, group, zeros=z)
        whole = torch.randint(-8, 9, (n, cols), generator=g, device=dev).half()
        y0 = Bl.gemv_q4(W, s, whole, group, zeros=z)
        torch.cuda.synchronize()
        mag = x.double().abs() @ (2 * q.double() * s.double().repeat_interleave(group, 1)[:, :cols]).t()
        assert torch.all(y.double().abs() <= (cols / 16 + 32) * 2.0 ** -23 * mag)
        assert torch.all(y0 == 0)
