"""Kernels that start while the one in front of them still runs: what that one may be writing is read by ordinary loads only,
and chains on the same buffers with changing data give what the calls give one by one."""
import os
import re

import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "decx_b200", "csrc")


def _code(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def test_no_read_only_loads_in_kernels_that_start_early():
    """The read-only path (ld.global.nc, __ldg, const __restrict__) is for memory that nobody writes while the kernel lives; a
    kernel that lets itself be started early lives while its inputs are being written."""
    early = [f for f in sorted(os.listdir(CSRC)) if f.endswith((".cuh", ".cu")) and f != "sm100_ptx.cuh" and "griddep_launch()" in _code(f)]
    assert {"gemm_q8.cuh", "gemv_q4.cuh", "rownorm_q8.cuh"} <= set(early)
    for name in early:
        found = re.findall(r"ld\.global(?:\.\w+)*\.nc\b|__ldg\b|__restrict__", _code(name))
        assert not found, (name, found)


@gpu
@pytest.mark.parametrize("tokens", [3, 16, 200])
def test_chains_on_the_same_buffers(tokens):
    from decx_b200 import blas, gemm
    dev = torch.device("cuda:0")
    H, N = 2048, 1000
    g = torch.Generator(device=dev).manual_seed(tokens)
    xs = [torch.randn(tokens, H, generator=g, device=dev).half() * (k + 1) for k in range(8)]
    ws = [(1 + 0.3 * torch.randn(H, generator=g, device=dev)).half() for _ in range(8)]
    Bs = [torch.randn(N, H, generator=g, device=dev) * (8 - k) for k in range(8)]
    W4 = blas.pack_q4(torch.randint(0, 16, (N, H), generator=g, device=dev, dtype=torch.uint8))
    s4 = torch.rand(N, H // 64, generator=g, device=dev).half()
    x, w, B = xs[0].clone(), ws[0].clone(), Bs[0].clone()
    q, s = blas.new_q8(tokens, H, dev)
    qb, sb = blas.new_q8(N, H, dev)
    few = min(tokens, 16)

    def chain(k, wait):
        x.copy_(xs[k])
        w.copy_(ws[k])
        B.copy_(Bs[k])
        wait()
        blas.cast_q8(B, out=qb, scales=sb)
        wait()
        blas.rmsnorm_q8(x, w, out=q, scales=s)                # x, its scales, and the GEMM's B and its scales change just before
        wait()
        y = blas.gemv_q4(W4, s4, q[:few], 64, x_scales=s[:few])
        wait()
        d = gemm.gemm_q8(q, s, qb, sb)
        wait()
        blas.cast_q8(B, out=qb, scales=sb)
        e = gemm.gemm_q8(q, s, qb, sb, out_dtype=torch.float32)
        return y, d, e

    want = [chain(k, torch.cuda.synchronize) for k in range(8)]
    torch.cuda.synchronize()
    got = [chain(i % 8, lambda: None) for i in range(160)]
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 8])), i
