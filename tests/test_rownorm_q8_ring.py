"""The ring form of the 8-bit row kernels: the shared memory it asks for, and rows, residuals and sums that start anywhere."""
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E4M3 = torch.float8_e4m3fn


def test_every_ring_fits_the_memory_that_its_kernel_may_use(tmp_path):
    """All launch shapes (types, residual, unaligned rows, threads) with every register count that a kernel of that many
    threads can have: at least two slots, no more shared memory than is asked for once per kernel, and with the static
    arrays no more than a CTA can have."""
    src = tmp_path / "plan.cpp"
    src.write_text(r"""
#include <cstdio>
#include "rownorm_q8_plan.h"
using namespace dxb;
int main() {
    long n = 0;
    if (Q8_RING_SMEM + 1024 > 227 * 1024) return std::printf("more than a CTA can have\n"), 1;
    for (unsigned esz = 2; esz <= 4; esz += 2)
        for (unsigned mats = 1; mats <= 2; ++mats)
            for (unsigned shift = 0; shift < 2; ++shift)
                for (unsigned threads = 96; threads <= 1024; threads += 32)
                    for (unsigned nch = 1; nch <= 4; nch *= 2) {
                        const bool warp = threads == 256;                // one row per warp; else a row per CTA, nch = 2
                        if (!warp && nch != 2) continue;
                        const unsigned slot = q8_ring_slot(threads, shift != 0, nch * 8 * esz / 16 * mats);
                        if (2ull * slot > Q8_RING_SLOTS) continue;       // such rows go another way
                        for (unsigned regs = 24; regs * threads <= 65536 && regs <= 255; ++regs) {
                            const Q8RingPlan r = q8_ring_plan(slot, threads, regs);
                            ++n;
                            if (r.depth < 2 || r.depth > 4 || r.per_sm < 1 || r.depth * slot > Q8_RING_SMEM ||
                                r.per_sm * (r.depth * slot + 1024 + 1024) > 228 * 1024)
                                return std::printf("esz %u mats %u shift %u threads %u nch %u regs %u: depth %u, %u bytes, %u per SM\n", esz,
                                                   mats, shift, threads, nch, regs, r.depth, r.depth * slot, r.per_sm), 1;
                        }
                    }
    std::printf("OK %ld\n", n);
}
""")
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "decx_b200", "csrc"), str(src), "-o", exe], check=True)
    run = subprocess.run([exe], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.startswith("OK "), run.stdout


@pytest.fixture(scope="module")
def Bl():
    from decx_b200 import blas
    return blas


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _at(t, extra, shift):
    """A copy whose rows are `extra` elements further apart than they are long, `shift` elements into a buffer of NaN."""
    rows, cols = t.shape
    raw = torch.full((rows * (cols + extra) + shift + 64,), float("nan"), dtype=t.dtype, device=t.device)
    v = raw[shift:shift + rows * (cols + extra)].view(rows, cols + extra)[:, :cols]
    v.copy_(t)
    return raw, v


def _half_step(v):
    """Half the distance between e4m3 neighbours at |v| <= 448 (exponents from -6 on)."""
    e = torch.frexp(v.abs().clamp(min=2.0 ** -6, max=448.0))[1].double() - 1
    return torch.exp2(e - 4)


def _check(q, scales, y, scale_rel):
    # a q may be half a step off, and fp32 arithmetic in front of the rounding (product, factor, scaling: each 2^-24) may
    # move a value across a border
    top = y.abs().amax(1)
    assert torch.all((scales.double() - top / 448).abs() <= scale_rel * top / 448)
    v = y / top[:, None] * 448
    assert torch.all((q.float().double() - v).abs() <= _half_step(v) + 8 * 2.0 ** -24 * v.abs())


def _norm_rel(cols):
    # a chain of up to cols / 1024 + 32 squares per thread and a tree of ten sums; the root halves what they lose
    return (cols / 1024 + 48) * 2.0 ** -24


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [8705, 8999, 9215, 12799, 13313, 13501, 13823, 16383])
def test_long_rows_of_odd_length(Bl, dev, cols, dtype):
    """Contiguous rows of an odd length into an aligned operand: the largest rings."""
    rows = 5
    g = torch.Generator(device=dev).manual_seed(cols)
    x, r = (torch.randn(rows, cols, generator=g, device=dev).to(dtype) for _ in range(2))
    w = (1 + 0.3 * torch.randn(cols, generator=g, device=dev)).to(dtype)
    q, s = Bl.cast_q8(x)
    torch.cuda.synchronize()
    _check(q, s, x.double(), 2 * 2.0 ** -24)
    for res in (None, r):
        q, s, total = Bl.rmsnorm_q8(x, w, residual=res, eps=1e-5)
        torch.cuda.synchronize()
        h = x.double() + (r.double() if res is not None else 0.0)
        _check(q, s, h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5) * w.double(), _norm_rel(cols))
        if res is not None:
            assert torch.equal(total, (x.float() + r.float()).to(dtype))


# shifts of x, residual and sum in elements, and what their rows have between them: an aligned matrix beside unaligned ones,
# all of them inside their first unit, each at another place
PLACES = [((1, 0), (0, 0), (0, 0)), ((0, 0), (3, 5), (0, 0)), ((0, 0), (0, 0), (1, 1)), ((7, 1), (7, 1), (7, 1)), ((3, 2), (5, 7), (2, 3)),
          ((1, 7), (1, 7), (4, 4))]


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [16, 20, 255, 500, 513, 1000, 1025, 3001, 5003, 8704])
def test_inputs_that_start_anywhere_into_an_aligned_operand(Bl, dev, cols, dtype):
    rows = 37
    g = torch.Generator(device=dev).manual_seed(cols + 1)
    x, r = (torch.randn(rows, cols, generator=g, device=dev).to(dtype) for _ in range(2))
    w = (1 + 0.3 * torch.randn(cols, generator=g, device=dev)).to(dtype)
    h32 = x.float() + r.float()
    for (sx, ex), (sr, er), (st, et) in PLACES:
        raw_x, vx = _at(x, ex, sx)
        raw_r, vr = _at(r, er, sr)
        raw_t, vt = _at(torch.zeros_like(x), et, st)
        q, s = Bl.cast_q8(vx)
        q1, s1, _ = Bl.rmsnorm_q8(vx, w, eps=1e-5)
        q2, s2, total = Bl.rmsnorm_q8(vx, w, residual=vr, eps=1e-5, sum_out=vt)
        torch.cuda.synchronize()
        _check(q, s, x.double(), 2 * 2.0 ** -24)
        _check(q1, s1, x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-5) * w.double(), _norm_rel(cols))
        h = x.double() + r.double()
        _check(q2, s2, h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5) * w.double(), _norm_rel(cols))
        assert torch.equal(total, h32.to(dtype))
        assert int(torch.isnan(raw_t).sum()) == raw_t.numel() - rows * cols, "the sum's padding was written"
        # in place, from the same places: another sum may mean another form (aligned or not), which adds the squares in another order
        q3, s3, _ = Bl.rmsnorm_q8(vx, w, residual=vr, eps=1e-5, sum_out=vx)
        torch.cuda.synchronize()
        _check(q3, s3, h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5) * w.double(), _norm_rel(cols))
        assert torch.equal(vx, h32.to(dtype))
        assert int(torch.isnan(raw_x).sum()) == raw_x.numel() - rows * cols
