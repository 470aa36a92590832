"""Matrix-vector products with 4-bit weights, against the definition in 64 bits."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn

# one row, one column, part of a row block, several; part of a group, of a slice, several slices, more than a cluster holds
SHAPES = [(1, 1), (1, 32), (5, 31), (64, 33), (65, 64), (63, 513), (130, 1000), (200, 2049), (64, 4099), (300, 8192),
          (70, 16384), (9, 20001), (33, 40000), (17, 65536), (4800, 544),
          (20000, 1056)]


@pytest.fixture(scope="module")
def Bl():
    from decx_b200 import blas
    return blas


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _case(dev, rows, cols, group, n, zeros, x8, seed, pad=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    groups = -(-cols // group)
    q = torch.randint(0, 16, (rows, cols), generator=g, device=dev, dtype=torch.uint8)
    s = torch.full((rows, groups + pad), float("nan"), dtype=torch.float16, device=dev)[:, :groups]
    s.copy_((torch.rand(rows, groups, generator=g, device=dev) + 0.5) * 0.1)
    z = None
    if zeros:
        z = torch.full((rows, groups + pad), 255, dtype=torch.uint8, device=dev)[:, :groups]
        z.copy_(torch.randint(0, 16, (rows, groups), generator=g, device=dev, dtype=torch.uint8))
    x = torch.randn(n, cols, generator=g, device=dev)
    v = torch.full((n, cols + pad), 0xFF, dtype=torch.uint8, device=dev).view(E4M3)[:, :cols] if x8 else \
        torch.full((n, cols + pad), float("nan"), dtype=torch.float16, device=dev)[:, :cols]
    v.copy_((x * 20).to(E4M3) if x8 else x.half())
    xs = torch.rand(n, generator=g, device=dev) + 0.5 if x8 else None
    return q, s, z, v, xs


def _exact(q, s, z, v, xs, group):
    """The result, and the sum of the magnitudes of its terms: q x and z x are summed apart."""
    cols = q.shape[1]
    at = torch.arange(cols, device=q.device) // group
    zero = z.double()[:, at] if z is not None else 8.0
    w = (q.double() - zero) * s.double()[:, at]
    x = v.float().double() * (xs.double()[:, None] if xs is not None else 1.0)
    return x @ w.t(), x.abs() @ ((q.double() + zero) * s.double()[:, at]).t()


def _check(y, ref, mag, cols):
    # fp32 sums: no chain is longer than the row has terms; in practice each term passes through the instruction's own
    # tree, at most 2048 / 128 group sums, the row's slices and four quarters.  The instruction may truncate instead of
    # rounding (one whole step, 2^-23).  An fp16 result is rounded once: half a step, or half the smallest subnormal.
    tol = (cols / 16 + 32) * 2.0 ** -23 * mag
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * ref.abs() + 2.0 ** -25
    assert torch.all((y.double() - ref).abs() <= tol), float(((y.double() - ref).abs() / tol).max())


@gpu
@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_gemv_q4(Bl, dev, shape, group, zeros, x8):
    rows, cols = shape
    for n, out_dtype, pad in ((1, torch.float32, 0), (3, torch.float16, 3), (8, torch.float32, 1), (9, torch.float16, 0), (16, torch.float32, 5)):
        q, s, z, v, xs = _case(dev, rows, cols, group, n, zeros, x8, rows + cols + n, pad)
        W = Bl.pack_q4(q)
        raw = torch.full((n + 2, rows + 7), 77.0, dtype=out_dtype, device=dev)
        y = Bl.gemv_q4(W, s, v, group, zeros=z, x_scales=xs, out=raw[1:n + 1, :rows])
        torch.cuda.synchronize()
        _check(y, *_exact(q, s, z, v, xs, group), cols)
        assert torch.all(raw[0] == 77) and torch.all(raw[n + 1] == 77) and torch.all(raw[1:n + 1, rows:] == 77)


@gpu
def test_one_vector_by_itself(Bl, dev):
    q, s, z, v, xs = _case(dev, 100, 300, 64, 1, True, False, 5)
    W = Bl.pack_q4(q)
    y = Bl.gemv_q4(W, s, v[0], 64, zeros=z)
    torch.cuda.synchronize()
    assert y.shape == (100,) and y.dtype == torch.float32
    assert torch.equal(y, Bl.gemv_q4(W, s, v, 64, zeros=z)[0])


@gpu
def test_nibbles_behind_an_odd_row_and_bytes_behind_a_row_do_not_count(Bl, dev):
    q, s, z, v, xs = _case(dev, 70, 333, 32, 2, False, False, 6)
    W = Bl.pack_q4(q)
    y = Bl.gemv_q4(W, s, v, 32).clone()
    full = torch.as_strided(W, (70, W.stride(0)), (W.stride(0), 1))
    full[:, 167:] = 0xFF
    full[:, 166] |= 0xF0
    assert torch.equal(y, Bl.gemv_q4(W, s, v, 32))


@gpu
def test_extreme_zero_points_and_scales(Bl, dev):
    """Zero points use all of uint8; a subnormal, a huge, an infinite and a NaN scale stay in their own row."""
    q, s, z, v, xs = _case(dev, 40, 256, 128, 4, True, False, 7)
    z[3] = 255
    z[4] = 0
    s[5] = 6e-8
    s[6] = 65504
    s[7, 1] = float("inf")
    s[8, 0] = float("nan")
    y = Bl.gemv_q4(Bl.pack_q4(q), s, v, 128, zeros=z)
    torch.cuda.synchronize()
    good = torch.tensor([r for r in range(40) if r not in (7, 8)], device=dev)
    ref, mag = _exact(q, s, z, v, xs, 128)
    _check(y[:, good], ref[:, good], mag[:, good], 256)
    assert torch.isinf(y[:, 7]).all() and torch.isnan(y[:, 8]).all()


@gpu
def test_nan_in_one_vector_stays_there(Bl, dev):
    q, s, z, v, xs = _case(dev, 64, 700, 64, 5, False, False, 8)
    W = Bl.pack_q4(q)
    y0 = Bl.gemv_q4(W, s, v, 64).clone()
    v[2, 650] = float("nan")
    y1 = Bl.gemv_q4(W, s, v, 64)
    torch.cuda.synchronize()
    assert torch.isnan(y1[2]).all()
    for k in (0, 1, 3, 4):
        assert torch.equal(y0[k], y1[k])


@gpu
@pytest.mark.parametrize("n", [1, 7, 16])
def test_same_result_every_time_and_for_every_company(Bl, dev, n):
    """No atomics: repeated calls agree bit for bit, and so does a captured one on another stream."""
    q, s, z, v, xs = _case(dev, 1000, 5000, 32, n, True, True, 9)
    W = Bl.pack_q4(q)
    y0 = Bl.gemv_q4(W, s, v, 32, zeros=z, x_scales=xs).clone()
    for _ in range(3):
        assert torch.equal(y0, Bl.gemv_q4(W, s, v, 32, zeros=z, x_scales=xs))
    y = torch.zeros_like(y0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        Bl.gemv_q4(W, s, v, 32, zeros=z, x_scales=xs, out=y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y0, y)


def test_pack_q4_on_the_host():
    from decx_b200 import blas
    q = torch.arange(3 * 5).reshape(3, 5) % 16
    W = blas.pack_q4(q)
    assert W.shape == (3, 3) and W.stride(0) % 16 == 0
    assert torch.equal(W[:, 0], (q[:, 0] | q[:, 1] << 4).to(torch.uint8)) and torch.equal(W[:, 2], q[:, 4].to(torch.uint8))


def test_refusals_of_the_c_abi():
    from decx_b200 import capi
    buf = (ctypes.c_float * 1024)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def call(xt=capi.FP16, yt=capi.FP32, rows=4, cols=64, n=2, group=32, W=p, ldw=32, s=p, lds=2, z=None, ldz=0, x=p, ldx=64,
             xs=None, y=p, ldy=4):
        return capi.lib.decxb200_gemv_q4(xt, yt, None, rows, cols, n, group, W, ldw, s, lds, z, ldz, x, ldx, xs, y, ldy)

    assert call(xt=capi.FP32) == -1 and call(yt=capi.E4M3) == -1 and call(xt=0) == -1
    assert call(rows=0) == -1 and call(cols=0) == -1 and call(n=0) == -1
    assert call(W=None) == -1 and call(s=None) == -1 and call(x=None) == -1 and call(y=None) == -1
    assert call(group=16) == -1 and call(group=0) == -1 and call(group=256) == -1
    assert call(ldw=16) == -1 and call(lds=1) == -1 and call(z=p, ldz=1) == -1 and call(ldx=63) == -1 and call(ldy=3) == -1
    assert call(n=17) == -5 and call(cols=65537, ldw=32784, lds=2049, ldx=65537) == -5 and call(ldw=1 << 27) == -5
    assert call(W=p + 8) == -2 and call(ldw=40) == -2 and call(s=p + 1) == -2 and call(x=p + 1) == -2
    assert call(y=p + 2) == -2 and call(xs=p + 2) == -2


def test_refusals_of_the_front_end():
    from decx_b200 import blas
    with pytest.raises(RuntimeError):
        blas.gemv_q4(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1).half(), torch.zeros(32).half(), 32)


@gpu
def test_refusals_of_the_front_end_on_the_gpu(Bl, dev):
    from decx_b200 import capi
    W = torch.zeros(4, 16, dtype=torch.uint8, device=dev)
    s, x = torch.zeros(4, 1, device=dev).half(), torch.zeros(32, device=dev).half()
    assert Bl.gemv_q4(W, s, x, 32).shape == (4,)
    with pytest.raises(TypeError):
        Bl.gemv_q4(W, s.float(), x, 32)
    with pytest.raises(TypeError):
        Bl.gemv_q4(W, s, x.float(), 32)
    with pytest.raises(ValueError):
        Bl.gemv_q4(W, s, x[:20], 32)
    with pytest.raises(ValueError):
        Bl.gemv_q4(W, s, x, 32, zeros=torch.zeros(4, 2, dtype=torch.uint8, device=dev))
    with pytest.raises(ValueError):
        Bl.gemv_q4(W, s, x, 32, x_scales=torch.ones(2, device=dev))
    with pytest.raises(ValueError):
        Bl.gemv_q4(W, s, x, 32, out=torch.zeros(5, device=dev))
    with pytest.raises(ValueError):
        Bl.gemv_q4(W, s.cpu(), x, 32)
    with pytest.raises(capi.DecxB200Error):
        Bl.gemv_q4(W, s, x, 16 * 3)
    with pytest.raises(capi.DecxB200Error):
        Bl.gemv_q4(W, s, torch.zeros(17, 32, device=dev).half(), 32)
    with pytest.raises(ValueError):
        Bl.gemv_q4(W, s, x, 2 ** 32 + 32)                    # would be 32 in 32 bits
    with pytest.raises(ValueError):
        Bl.gemv_q4(W, s, x, -32)
