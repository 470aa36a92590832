"""The 8-bit cast and the RMS norm that writes an 8-bit operand, against the definition in 64 bits."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
# warp-per-row, CTA-per-row and re-reading kernels; 16-byte multiples and odd lengths; one element
SHAPES = [(1, 1), (3, 7), (1, 64), (9, 255), (17, 256), (5, 257), (8, 512), (33, 1000), (2, 1024), (7, 1025), (300, 1536),
          (1, 4096), (4, 4099), (299, 3001), (2, 8192), (1, 16384), (310, 9000), (2, 16385), (3, 32768), (2, 32769), (1, 70001)]


@pytest.fixture(scope="module")
def Bl():
    from decx_b200 import blas
    return blas


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _view(t, extra, shift=0):
    """A copy whose rows are `extra` elements further apart than they are long, `shift` elements into its buffer."""
    rows, cols = t.shape
    raw = torch.full((rows * (cols + extra) + shift + 64,), float("nan"), dtype=t.dtype, device=t.device)
    v = raw[shift:shift + rows * (cols + extra)].view(rows, cols + extra)[:, :cols]
    v.copy_(t)
    return v


def _half_step(v):
    """Half the distance between e4m3 neighbours at |v| <= 448 (exponents from -6 on)."""
    e = torch.frexp(v.abs().clamp(min=2.0 ** -6, max=448.0))[1].double() - 1
    return torch.exp2(e - 4)


def _check(q, scales, y, scale_rel):
    """q, scales against the exact rows y.  A q may be half a step off, and fp32 arithmetic in front of the rounding
    (product, factor, scaling: each 2^-24) may move a value across a border."""
    top = y.abs().amax(1)
    assert torch.all((scales.double() - top / 448).abs() <= scale_rel * top / 448)
    v = torch.where(top[:, None] > 0, y / torch.where(top > 0, top, 1.0)[:, None] * 448, 0.0)
    err = (q.float().double() - v).abs()
    assert torch.all(err <= _half_step(v) + 8 * 2.0 ** -24 * v.abs())


def _norm64(x, r, w, eps):
    h = x.double() + (r.double() if r is not None else 0.0)
    return h, h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w.double()


def _raw_q(rows, cols, pitch, dev):
    raw = torch.full((rows, pitch), 0xA5, dtype=torch.uint8, device=dev)
    return raw, raw.view(E4M3)[:, :cols]


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_cast_q8(Bl, dev, shape, dtype):
    rows, cols = shape
    g = torch.Generator(device=dev).manual_seed(rows + 13 * cols)
    x = (torch.randn(rows, cols, generator=g, device=dev) * torch.exp(2 * torch.randn(rows, 1, generator=g, device=dev))).to(dtype)
    for src, pitch in ((x, -(-cols // 16) * 16), (_view(x, 3, 1), cols + 5)):
        raw, out = _raw_q(rows, cols, pitch, dev)
        q, s = Bl.cast_q8(src, out=out)
        torch.cuda.synchronize()
        _check(q, s, x.double(), 2 * 2.0 ** -24)
        assert torch.all(raw[:, cols:] == 0xA5), "pitch padding was written"


@gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_rmsnorm_q8(Bl, dev, shape, dtype, residual):
    rows, cols = shape
    g = torch.Generator(device=dev).manual_seed(7 * rows + cols)
    x = (torch.randn(rows, cols, generator=g, device=dev) * torch.exp(2 * torch.randn(rows, 1, generator=g, device=dev))).to(dtype)
    r = torch.randn(rows, cols, generator=g, device=dev).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(cols, generator=g, device=dev)).to(dtype)
    h, y = _norm64(x, r, w, 1e-5)
    half_ulp = torch.finfo(dtype).eps / 2
    # a chain of up to cols / 1024 + 32 squares per thread and a tree of ten sums; the root halves what they lose
    rel = (cols / 1024 + 48) * 2.0 ** -24
    for extra, shift, pitch in ((0, 0, -(-cols // 16) * 16), (3, 1, cols + 5)):
        vx = _view(x, extra, shift) if extra else x
        vr = (_view(r, extra, shift) if extra else r) if residual else None
        raw, out = _raw_q(rows, cols, pitch, dev)
        total = _view(torch.zeros_like(x), extra, shift) if residual else None
        q, s, total = Bl.rmsnorm_q8(vx, w, residual=vr, eps=1e-5, out=out, sum_out=total)
        torch.cuda.synchronize()
        _check(q, s, y, rel)
        assert torch.all(raw[:, cols:] == 0xA5), "pitch padding was written"
        if residual:
            assert torch.all((total.double() - h).abs() <= (half_ulp + 2.0 ** -23) * h.abs() + 2.0 ** -25)
        else:
            assert total is None


@gpu
@pytest.mark.parametrize("cols", [200, 4096, 4099, 40000])
@pytest.mark.parametrize("into", ["x", "residual"])
def test_sum_may_replace_an_input(Bl, dev, cols, into):
    g = torch.Generator(device=dev).manual_seed(cols)
    x, r = (torch.randn(6, cols, generator=g, device=dev).half() for _ in range(2))
    w = torch.ones(cols, dtype=torch.float16, device=dev)
    q0, s0, t0 = Bl.rmsnorm_q8(x, w, residual=r)
    a, b = x.clone(), r.clone()
    q1, s1, t1 = Bl.rmsnorm_q8(a, w, residual=b, sum_out=a if into == "x" else b)
    torch.cuda.synchronize()
    assert torch.equal(t0, t1) and torch.equal(s0, s1) and torch.equal(q0.view(torch.uint8), q1.view(torch.uint8))
    assert torch.equal(b if into == "x" else a, r if into == "x" else x)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [100, 1024, 5000, 8192, 40000])
def test_rows_without_a_form(Bl, dev, cols, dtype):
    """Zero rows, tiny rows, rows with NaN or infinity; the rows beside them are as without them."""
    g = torch.Generator(device=dev).manual_seed(cols)
    x = torch.randn(8, cols, generator=g, device=dev).to(dtype)
    clean = x.clone()
    x[1] = 0
    x[3, cols // 2] = float("nan")
    x[5, cols - 1] = float("-inf")
    x[6] = 0
    x[6, 0] = torch.finfo(dtype).smallest_normal if dtype == torch.float16 else 1e-37
    w = torch.ones(cols, dtype=dtype, device=dev)
    for q, s, want in ((*Bl.cast_q8(x), Bl.cast_q8(clean)), (*Bl.rmsnorm_q8(x, w)[:2], Bl.rmsnorm_q8(clean, w))):
        torch.cuda.synchronize()
        assert s[1] == 0 and torch.all(q[1].float() == 0)
        for bad in (3, 5):
            assert torch.isnan(s[bad]) and torch.isnan(q[bad].float()).all()
        assert q[6, 0].float() == 448 and torch.all(q[6, 1:].float() == 0) and 0 < s[6] < 1e-3
        for same in (0, 2, 4, 7):
            assert s[same] == want[1][same] and torch.equal(q[same].view(torch.uint8), want[0][same].view(torch.uint8))


@gpu
def test_sum_of_squares_beyond_fp32_is_not_a_zero_row(Bl, dev):
    x = torch.full((2, 2048), 1e19, device=dev)
    x[0] = 1.0
    q, s, _ = Bl.rmsnorm_q8(x, torch.ones(2048, device=dev))
    torch.cuda.synchronize()
    assert torch.isfinite(s[0]) and torch.isnan(s[1]) and torch.isnan(q[1].float()).all()


@gpu
def test_every_e4m3_border_rounds_to_even(Bl, dev):
    """All midpoints between neighbouring e4m3 values, and the floats next to them, in a row whose scale is 1."""
    codes = torch.arange(0, 0x7F, dtype=torch.uint8, device=dev).view(E4M3).float()
    mid = (codes[1:] + codes[:-1]) / 2
    row = torch.cat([mid, torch.nextafter(mid, torch.zeros_like(mid)), torch.nextafter(mid, mid + 1), codes])
    row = torch.cat([row, -row])[None]
    q, s = Bl.cast_q8(row.contiguous())
    torch.cuda.synchronize()
    assert s[0] == 1
    assert torch.equal(q[0].float(), row[0].to(E4M3).float())


@gpu
def test_on_another_stream_and_in_a_graph(Bl, dev):
    g = torch.Generator(device=dev).manual_seed(1)
    x, r = (torch.randn(50, 2048, generator=g, device=dev).half() for _ in range(2))
    w = torch.ones(2048, dtype=torch.float16, device=dev)
    q0, s0, t0 = Bl.rmsnorm_q8(x, w, residual=r)
    out, scales = Bl.new_q8(50, 2048, dev)
    total = torch.empty_like(x)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        Bl.rmsnorm_q8(x, w, residual=r, out=out, scales=scales, sum_out=total)
    for k in range(2):
        x.mul_(-1), r.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        sign = -1 if k == 0 else 1
        assert torch.equal(s0, scales) and torch.equal(t0 * sign, total) and torch.equal(q0.float() * sign, out.float())


def test_refusals_of_the_c_abi():
    """Checked before anything is launched, so no GPU is needed."""
    from decx_b200 import capi
    buf = (ctypes.c_float * 256)()
    p = ctypes.addressof(buf)

    def cast(dt=capi.FP16, rows=2, cols=16, src=p, lds=16, q=p, ldq=16, scales=p):
        return capi.lib.decxb200_cast_q8(dt, None, rows, cols, src, lds, q, ldq, scales)

    assert cast(dt=capi.FP64) == -1 and cast(dt=9) == -1
    assert cast(rows=0) == -1 and cast(cols=0) == -1
    assert cast(src=None) == -1 and cast(q=None) == -1 and cast(scales=None) == -1
    assert cast(lds=15) == -1 and cast(ldq=15) == -1
    assert cast(src=p + 1) == -2 and cast(scales=p + 2) == -2 and cast(dt=capi.FP32, src=p + 2) == -2

    def norm(dt=capi.FP16, x=p, ldx=16, r=p, ldr=16, total=p, ldt=16, w=p, eps=1e-5, q=p, ldq=16, scales=p, rows=2, cols=16):
        return capi.lib.decxb200_rmsnorm_q8(dt, None, rows, cols, x, ldx, r, ldr, total, ldt, w, eps, q, ldq, scales)

    assert norm(dt=capi.CPLXF) == -1 and norm(rows=0) == -1 and norm(cols=0) == -1
    assert norm(x=None) == -1 and norm(w=None) == -1 and norm(q=None) == -1 and norm(scales=None) == -1
    assert norm(ldx=15) == -1 and norm(ldr=15) == -1 and norm(ldt=15) == -1 and norm(ldq=15) == -1
    assert norm(r=None) == -1                                     # a sum of nothing
    assert norm(total=p, ldt=32) == -1                            # in place with another pitch
    for eps in (0.0, -1e-5, float("nan"), float("inf"), 1e-42):
        assert norm(eps=eps) == -1
    assert norm(w=p + 1) == -2


def test_refusals_of_the_front_end():
    from decx_b200 import blas
    with pytest.raises(RuntimeError):
        blas.cast_q8(torch.zeros(4, 16))
    with pytest.raises(RuntimeError):
        blas.rmsnorm_q8(torch.zeros(4, 16), torch.zeros(16))


@gpu
def test_refusals_of_the_front_end_on_the_gpu(Bl, dev):
    x, w = torch.zeros(4, 16, device=dev), torch.zeros(16, device=dev)
    with pytest.raises(TypeError):
        Bl.cast_q8(x.double())
    with pytest.raises(TypeError):
        Bl.rmsnorm_q8(x, w.half())
    with pytest.raises(ValueError):
        Bl.rmsnorm_q8(x, w[:8])
    with pytest.raises(ValueError):
        Bl.rmsnorm_q8(x, w, residual=x[:3])
    with pytest.raises(ValueError):
        Bl.rmsnorm_q8(x, w, sum_out=x)
    with pytest.raises(ValueError):
        Bl.cast_q8(x.t())
    with pytest.raises(ValueError):
        Bl.cast_q8(x, out=torch.empty(4, 16, dtype=torch.uint8, device=dev))
    with pytest.raises(ValueError):
        Bl.cast_q8(x, scales=torch.empty(3, device=dev))
    from decx_b200 import capi
    with pytest.raises(capi.DecxB200Error):
        Bl.rmsnorm_q8(x, w, eps=0.0)
