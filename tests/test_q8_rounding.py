"""e4m3 rounding of the 8-bit cast at the borders between neighbours: the quotient x * 448 / max|x| is exact enough that ties
go to the even neighbour, whatever the row's maximum is."""
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


def _nearest(y):
    """Rows of y (64 bits) as e4m3 values, nearest even.  y * 448 and the quotient's ties are exact in 64 bits."""
    v = y * 448 / y.abs().amax(1, keepdim=True)
    step = torch.exp2(torch.clamp(torch.frexp(v.abs())[1].double() - 1, min=-6.0) - 3)
    return torch.round(v / step) * step


def _ties(dev, cols, dtype):
    """Rows with every maximum n / 64, n = 448 .. 895, that hold the midpoints between e4m3 neighbours of their scale where the
    type has them: 448 x / max = m, x = m n / (64 * 448); every row also has random values.  At most 11 bits each."""
    codes = torch.arange(0, 0x7F, dtype=torch.uint8, device=dev).view(E4M3).double()
    mid = (codes[1:] + codes[:-1]) / 2
    top = torch.arange(448, 896, device=dev).double() / 64
    x = mid[None, :] * top[:, None] / 448
    g = torch.Generator(device=dev).manual_seed(cols)
    rows = (torch.randn(len(top), cols, generator=g, device=dev).clamp(-7, 7)).to(torch.float16).double()
    rows[:, :x.shape[1]] = x.to(torch.float16).double()
    rows[:, x.shape[1]:2 * x.shape[1]] = -rows[:, :x.shape[1]]
    rows[:, -1] = top
    return rows.to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [256, 1000, 1001, 4096, 17000, 33000])
def test_cast_is_nearest_even_for_every_maximum(Bl, dev, cols, dtype):
    """Numbers of 11 bits: the quotient of two of them (times 448) is a midpoint or at least 2^-17 away from it, relatively,
    so one fp32 rounding of the quotient cannot make or hide a tie: equality, no tolerance."""
    x = _ties(dev, cols, dtype)
    want = _nearest(x.double())
    hit = (x.double() * 448 / x.double().abs().amax(1, keepdim=True)) / torch.exp2(
        torch.clamp(torch.frexp(want.abs())[1].double() - 1, min=-6.0) - 3)
    assert int((hit.abs() % 1 == 0.5).sum()) > 1000, "the rows hold ties"
    out = torch.empty(x.shape[0], cols + 5, dtype=torch.uint8, device=dev).view(E4M3)[:, :cols]      # single elements
    for q in (Bl.cast_q8(x)[0], Bl.cast_q8(x, out=out)[0]):
        torch.cuda.synchronize()
        assert torch.equal(q.float().double(), want), int((q.float().double() != want).sum())


@gpu
def test_rows_of_every_magnitude(Bl, dev):
    """The same row times powers of two that fp32 holds exactly: the same q."""
    x = _ties(dev, 1000, torch.float32)[::7]
    want = _nearest(x.double())
    for e in (-100, -97, -60, 0, 60, 99, 101, 120):
        q, s = Bl.cast_q8(x * 2.0 ** e)
        torch.cuda.synchronize()
        assert torch.equal(q.float().double(), want), e
        assert torch.equal(s, Bl.cast_q8(x)[1] * 2.0 ** e)
