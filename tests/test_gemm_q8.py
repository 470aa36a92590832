"""The 8-bit GEMM against the definition in 64 bits, both of its kernels, and the operators of a quantised layer in a row."""
import contextlib
import ctypes

import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
THIN, PAIR = 1, 2

# M, N, K: single elements, edges of the 16/32/64/128-row tiles and of the 256 x 256 ones, K of one stage, of fewer
# stages than the ring has, of a short last stage, long enough to be cut eight ways; several rounds of tiles
SHAPES = [(1, 1, 1), (1, 128, 128), (7, 40, 16), (16, 256, 300), (17, 129, 1000), (32, 1000, 4096), (33, 64, 130), (64, 513, 2047),
          (65, 300, 513), (128, 128, 8192), (129, 257, 1025), (256, 256, 256), (300, 700, 777), (513, 1030, 384), (1, 5000, 520),
          (2600, 2100, 160), (40, 20000, 300),
          (400, 600, 1100), (1000, 900, 4000), (500, 2100, 2050), (255, 257, 16384)]


@pytest.fixture(scope="module")
def G():
    from decx_b200 import gemm
    return gemm


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _operand(dev, g, rows, cols, pad=0):
    """A pitched 8-bit operand; the bytes between its rows are NaN."""
    pitch = -(-cols // 16) * 16 + 16 * pad
    buf = torch.full((rows, pitch), 0x7F, dtype=torch.uint8, device=dev)
    v = buf.view(E4M3)[:, :cols]
    v.copy_((torch.randn(rows, cols, generator=g, device=dev) * 100).clamp(-448, 448).to(E4M3))
    return v, (torch.rand(rows, generator=g, device=dev) + 0.5) / 100


def _exact(A, sa, B, sb, C, alpha, beta):
    a, b = A.float().double() * sa.double()[:, None], B.float().double() * sb.double()[:, None]
    d, mag = alpha * (a @ b.t()), abs(alpha) * (a.abs() @ b.abs().t())
    if C is not None:
        d, mag = d + beta * C.double(), mag + abs(beta) * C.double().abs()
    return d, mag


def _check(D, ref, mag, K):
    # fp32 sums whose adder may truncate (2^-23 of the running sum per 32 products, of which there are at most K / 32 + 1,
    # plus eight slices), scales and the addition of C: a few half steps.  fp16: one rounding, half a step or half the
    # smallest subnormal.
    tol = (K / 32 + 16) * 2.0 ** -23 * mag
    if D.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * ref.abs() + 2.0 ** -25
    err = (D.double() - ref).abs()
    assert torch.all(err <= tol), f"largest error over tolerance: {float((err / tol).max()):.3f}"


@gpu
@pytest.mark.parametrize("tile", [THIN, PAIR])
@pytest.mark.parametrize("shape", SHAPES)
def test_gemm_q8(G, dev, shape, tile):
    M, N, K = shape
    g = torch.Generator(device=dev).manual_seed(M + 3 * N + 5 * K)
    status = G.new_status(dev)
    for dtype, with_c, pad in ((torch.float16, False, 0), (torch.float32, True, 1), (torch.float16, True, 3), (torch.float32, False, 2)):
        A, sa = _operand(dev, g, M, K, pad)
        B, sb = _operand(dev, g, N, K, pad + 1)
        alpha, beta = (0.5, -1.25) if with_c else (None, None)
        # pitches with and without 16-byte aligned rows
        extra = 8 - N % 8 if pad != 3 else 3
        C = torch.randn(M, N + extra, generator=g, device=dev).to(dtype)[:, :N] if with_c else None
        raw = torch.full((M + 2, N + extra), 77.0, dtype=dtype, device=dev)
        D = G.gemm_q8(A, sa, B, sb, C=C, alpha=alpha, beta=beta, out=raw[1:M + 1, :N], status=status, tile=tile)
        torch.cuda.synchronize()
        assert int(status.item()) == 0
        _check(D, *_exact(A, sa, B, sb, C, alpha or 1.0, beta or 0.0), K)
        assert torch.all(raw[0] == 77) and torch.all(raw[M + 1] == 77) and torch.all(raw[1:M + 1, N:] == 77)


@gpu
@pytest.mark.parametrize("shape", [(1, 4096, 4096), (20, 8192, 1024), (100, 1000, 16384), (700, 2048, 2048), (2048, 4096, 1024)])
def test_library_choice(G, dev, shape):
    M, N, K = shape
    g = torch.Generator(device=dev).manual_seed(1)
    A, sa = _operand(dev, g, M, K)
    B, sb = _operand(dev, g, N, K)
    D = G.gemm_q8(A, sa, B, sb, out_dtype=torch.float32)
    torch.cuda.synchronize()
    _check(D, *_exact(A, sa, B, sb, None, 1.0, 0.0), K)


@gpu
@pytest.mark.parametrize("tile", [THIN, PAIR])
def test_long_sums_of_one_sign(G, dev, tile):
    """All products positive: what a truncating or short accumulator loses adds up instead of cancelling."""
    M, N, K = 64, 256, 16384
    A = torch.full((M, K), 1.0, device=dev).to(E4M3)
    g = torch.Generator(device=dev).manual_seed(2)
    B = (torch.rand(N, K, generator=g, device=dev) + 0.5).to(E4M3)
    sa, sb = torch.ones(M, device=dev), torch.ones(N, device=dev)
    D = G.gemm_q8(A, sa, B, sb, out_dtype=torch.float32, tile=tile)
    torch.cuda.synchronize()
    _check(D, *_exact(A, sa, B, sb, None, 1.0, 0.0), K)


@gpu
@pytest.mark.parametrize("tile", [THIN, PAIR])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_c_may_be_the_result(G, dev, tile, dtype):
    g = torch.Generator(device=dev).manual_seed(3)
    A, sa = _operand(dev, g, 200, 600)
    B, sb = _operand(dev, g, 328, 600)
    C = torch.randn(200, 328, generator=g, device=dev).to(dtype)
    D = G.gemm_q8(A, sa, B, sb, C=C, alpha=1.0, beta=1.0, tile=tile)
    E = C.clone()
    G.gemm_q8(A, sa, B, sb, C=E, alpha=1.0, beta=1.0, out=E, tile=tile)
    torch.cuda.synchronize()
    assert torch.equal(D, E)


@gpu
@pytest.mark.parametrize("tile", [THIN, PAIR])
def test_nan_and_beta_zero(G, dev, tile):
    """A NaN row stays in its row; C is not read when beta is 0."""
    g = torch.Generator(device=dev).manual_seed(4)
    A, sa = _operand(dev, g, 70, 512)
    B, sb = _operand(dev, g, 300, 512)
    D0 = G.gemm_q8(A, sa, B, sb, tile=tile).clone()
    sa[5] = float("nan")
    sb[17] = float("nan")
    C = torch.full((70, 300), float("nan"), dtype=torch.float16, device=dev)
    D1 = G.gemm_q8(A, sa, B, sb, C=C, alpha=1.0, beta=0.0, tile=tile)
    torch.cuda.synchronize()
    bad = torch.zeros(70, 300, dtype=torch.bool, device=dev)
    bad[5], bad[:, 17] = True, True
    assert torch.isnan(D1[bad]).all() and torch.equal(D0[~bad], D1[~bad])


@gpu
@pytest.mark.parametrize("shape", [(8, 2048, 8192), (600, 3000, 1024)])
def test_same_result_every_time_in_a_graph_and_on_another_stream(G, dev, shape):
    M, N, K = shape
    g = torch.Generator(device=dev).manual_seed(5)
    A, sa = _operand(dev, g, M, K)
    B, sb = _operand(dev, g, N, K)
    D0 = G.gemm_q8(A, sa, B, sb).clone()
    assert torch.equal(D0, G.gemm_q8(A, sa, B, sb))
    D = torch.zeros_like(D0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        G.gemm_q8(A, sa, B, sb, out=D)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(D0, D)


@gpu
@pytest.mark.parametrize("tokens", [1, 6, 200])
def test_quantised_layer(G, dev, tokens):
    """The operators in a row: norm with residual into an 8-bit operand; a projection with 8-bit weights and (few tokens)
    one with 4-bit weights read it; the first result becomes an 8-bit operand again and comes back to the residual
    stream through the second projection's C."""
    from decx_b200 import blas
    H, F, group = 768, 2056, 64
    g = torch.Generator(device=dev).manual_seed(6)
    x, r = (torch.randn(tokens, H, generator=g, device=dev).half() for _ in range(2))
    w = (1 + 0.1 * torch.randn(H, generator=g, device=dev)).half()
    up, s_up = blas.cast_q8(torch.randn(F, H, generator=g, device=dev) / H ** 0.5)
    down, s_down = blas.cast_q8(torch.randn(H, F, generator=g, device=dev) / F ** 0.5)

    q, s, total = blas.rmsnorm_q8(x, w, residual=r)
    mid = G.gemm_q8(q, s, up, s_up)
    act = torch.relu(mid)
    qa, sa = blas.cast_q8(act)
    out = G.gemm_q8(qa, sa, down, s_down, C=total, alpha=1.0, beta=1.0)
    torch.cuda.synchronize()
    _check(mid, *_exact(q, s, up, s_up, None, 1.0, 0.0), H)
    _check(out, *_exact(qa, sa, down, s_down, total, 1.0, 1.0), F)
    # against the layer in 64 bits on the unquantised input: two e4m3 roundings of at most 2^-4 each; products with
    # random matrices keep a relative error, and the residual stream that is added has none
    h = x.double() + r.double()
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * w.double()
    a = torch.relu(y @ (up.float().double() * s_up.double()[:, None]).t())
    ref = h + a @ (down.float().double() * s_down.double()[:, None]).t()
    assert float((out.double() - ref).norm() / ref.norm()) < 2 * 2.0 ** -4 + 2.0 ** -10

    if tokens <= 16:
        q4 = torch.randint(0, 16, (F, H), generator=g, device=dev, dtype=torch.uint8)
        s4 = (torch.rand(F, H // group, generator=g, device=dev) / 16 / H ** 0.5).half()
        y4 = blas.gemv_q4(blas.pack_q4(q4), s4, q, group, x_scales=s)
        torch.cuda.synchronize()
        w4 = (q4.double() - 8) * s4.double().repeat_interleave(group, 1)
        xq = q.float().double() * s.double()[:, None]
        tol = (H / 16 + 32) * 2.0 ** -23 * (xq.abs() @ ((q4.double() + 8) * s4.double().repeat_interleave(group, 1)).t())
        assert torch.all((y4.double() - xq @ w4.t()).abs() <= tol)


@gpu
def test_first_calls_inside_a_capture():
    """Nothing has to be called beforehand: in a fresh process, each operator's first call is a captured one."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = r"""
import sys, torch
sys.path.insert(0, %r)
from decx_b200 import blas, gemm as G
dev = torch.device("cuda:0")
x, r = (torch.randn(24, 4096, device=dev).half() for _ in range(2))
big = torch.randn(700, 2048, device=dev)
w = torch.ones(4096, device=dev).half()
W4 = blas.pack_q4(torch.randint(0, 16, (512, 4096), device=dev, dtype=torch.uint8))
s4 = torch.rand(512, 64, device=dev).half()
stream = torch.cuda.Stream()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    q, s, t = blas.rmsnorm_q8(x, w, residual=r)
    y = blas.gemv_q4(W4, s4, q[:9], 64, x_scales=s[:9])
    d = G.gemm_q8(q, s, q, s, out_dtype=torch.float32)
    qb, sb = blas.cast_q8(big)
    e = G.gemm_q8(qb, sb, qb, sb)
graph.replay()
torch.cuda.synchronize()
q2, s2, t2 = blas.rmsnorm_q8(x, w, residual=r)
y2 = blas.gemv_q4(W4, s4, q2[:9], 64, x_scales=s2[:9])
d2 = G.gemm_q8(q2, s2, q2, s2, out_dtype=torch.float32)
qb2, sb2 = blas.cast_q8(big)
e2 = G.gemm_q8(qb2, sb2, qb2, sb2)
torch.cuda.synchronize()
print("SAME", torch.equal(t, t2), torch.equal(y, y2), torch.equal(d, d2), torch.equal(e, e2))
""" % root
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert "SAME True True True True" in run.stdout, run.stdout + run.stderr


@gpu
def test_calls_on_two_streams_at_once(G, dev):
    """No workspace and no state between calls: two streams that overlap give what one after the other gives."""
    from decx_b200 import blas
    g = torch.Generator(device=dev).manual_seed(8)
    x = [torch.randn(300, 2048, generator=g, device=dev).half() for _ in range(2)]
    w = torch.ones(2048, dtype=torch.float16, device=dev)
    B, sb = _operand(dev, g, 1536, 2048)
    W4 = blas.pack_q4(torch.randint(0, 16, (2000, 2048), generator=g, device=dev, dtype=torch.uint8))
    s4 = torch.rand(2000, 16, generator=g, device=dev).half()

    def chain(v):
        q, s, _ = blas.rmsnorm_q8(v, w)
        return G.gemm_q8(q, s, B, sb), G.gemm_q8(q[:5], s[:5], B, sb), blas.gemv_q4(W4, s4, q[:3], 128, x_scales=s[:3])

    want = [chain(v) for v in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(chain(x[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


@gpu
def test_a_captured_fork_and_join_replays(G, dev):
    """One graph in which the norm's output goes two ways, to a GEMM and, on another stream, to a 4-bit product that a cast
    and a GEMM then join: replayed on new inputs it gives what the calls give one after the other."""
    from decx_b200 import blas
    g = torch.Generator(device=dev).manual_seed(18)
    x = torch.randn(12, 2048, generator=g, device=dev).half()
    w = torch.rand(2048, generator=g, device=dev).half()
    B, sb = _operand(dev, g, 640, 2048)
    E, se = _operand(dev, g, 320, 2640)
    W4 = blas.pack_q4(torch.randint(0, 16, (2000, 2048), generator=g, device=dev, dtype=torch.uint8))
    s4 = torch.rand(2000, 16, generator=g, device=dev).half()
    q, s = blas.new_q8(12, 2048, dev)
    joined = torch.empty(12, 2640, dtype=torch.float16, device=dev)
    q2, s2 = blas.new_q8(12, 2640, dev)
    out = torch.empty(12, 320, dtype=torch.float16, device=dev)

    def calls(fork, join):
        blas.rmsnorm_q8(x, w, out=q, scales=s)
        with fork():
            blas.gemv_q4(W4, s4, q, 128, x_scales=s, out=joined[:, 640:])
        G.gemm_q8(q, s, B, sb, out=joined[:, :640])
        join()
        blas.cast_q8(joined, out=q2, scales=s2)
        G.gemm_q8(q2, s2, E, se, out=out)

    side = torch.cuda.Stream()

    def forked():
        side.wait_stream(torch.cuda.current_stream())
        return torch.cuda.stream(side)

    calls(contextlib.nullcontext, lambda: None)              # the plain order
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(forked, lambda: torch.cuda.current_stream().wait_stream(side))
    for k in range(8):
        x.normal_(generator=g)
        calls(contextlib.nullcontext, lambda: None)
        want = [t.clone() for t in (q, s, joined, q2, s2, out)]
        for t in (q, s, joined, q2, s2, out):
            t.zero_()
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((q, s, joined, q2, s2, out), want):
            assert torch.equal(a.float(), b.float()), k


def test_refusals_of_the_c_abi():
    from decx_b200 import capi
    buf = (ctypes.c_float * 4096)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def call(dt=capi.FP16, M=4, N=8, K=32, A=p, lda=32, sa=p, B=p, ldb=32, sb=p, C=None, ldc=0, D=p, ldd=8, tile=0):
        return capi.lib.decxb200_gemm_q8(dt, None, M, N, K, A, lda, sa, B, ldb, sb, C, ldc, D, ldd, None, None, None, tile)

    assert call(dt=capi.FP64) == -1 and call(dt=capi.E4M3) == -1
    assert call(M=0) == -1 and call(N=0) == -1 and call(K=0) == -1
    assert call(A=None) == -1 and call(B=None) == -1 and call(D=None) == -1 and call(sa=None) == -1 and call(sb=None) == -1
    assert call(lda=16) == -1 and call(ldb=16) == -1 and call(ldd=7) == -1 and call(C=p, ldc=7) == -1
    assert call(tile=3) == -1 and call(tile=-1) == -1
    assert call(C=p, ldc=16) == -1                           # C is D, with another pitch
    assert call(M=0x7fffffff) == -5
    assert call(A=p + 8) == -2 and call(B=p + 4) == -2 and call(lda=40) == -2 and call(ldb=33) == -2
    assert call(sa=p + 2) == -2 and call(sb=p + 1) == -2 and call(D=p + 1) == -2 and call(dt=capi.FP32, C=p + 2, ldc=8) == -2


def test_refusals_of_the_front_end():
    from decx_b200 import gemm
    with pytest.raises(RuntimeError):
        gemm.gemm_q8(torch.zeros(4, 32).to(E4M3), torch.ones(4), torch.zeros(8, 32).to(E4M3), torch.ones(8))


@gpu
def test_refusals_of_the_front_end_on_the_gpu(G, dev):
    from decx_b200 import capi
    A, B = torch.zeros(4, 32, device=dev).to(E4M3), torch.zeros(8, 32, device=dev).to(E4M3)
    sa, sb = torch.ones(4, device=dev), torch.ones(8, device=dev)
    assert G.gemm_q8(A, sa, B, sb).shape == (4, 8)
    with pytest.raises(TypeError):
        G.gemm_q8(A.half(), sa, B, sb)
    with pytest.raises(ValueError):
        G.gemm_q8(A, sa, B[:, :16], sb)
    with pytest.raises(ValueError):
        G.gemm_q8(A, sb, B, sb)
    with pytest.raises(ValueError):
        G.gemm_q8(A, sa, B, sb.double())
    with pytest.raises(TypeError):
        G.gemm_q8(A, sa, B, sb, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        G.gemm_q8(A, sa, B, sb, C=torch.zeros(4, 8, device=dev), out=torch.zeros(4, 8, device=dev).half())
    with pytest.raises(ValueError):
        G.gemm_q8(A, sa, B, sb, out=torch.zeros(4, 9, device=dev))
    with pytest.raises(ValueError):
        G.gemm_q8(A, sa, B, sb.cpu())
    with pytest.raises(capi.DecxB200Error):
        G.gemm_q8(A, sa, B, sb, tile=2 ** 32)
    with pytest.raises(capi.DecxB200Error):
        G.gemm_q8(A[:, :24].contiguous(), sa, B[:, :24].contiguous(), sb)
