"""decx_b200/_front.so is loaded by the low-precision calls alone, and not for another torch than the one it was built for."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code):
    r = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {ROOT!r})\n" + code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


LOW_PRECISION = """
x = torch.zeros(4, 32)
q = x.to(torch.float8_e4m3fn)
calls = [lambda: blas.cast_q8(x), lambda: blas.rmsnorm_q8(x, x[0]), lambda: gemm.gemm_q8(q, x[:, 0], q, x[:, 0]),
         lambda: blas.gemv_q4(torch.zeros(4, 16, dtype=torch.uint8), x[:, :1].half(), x[0].half(), 32)]
for call in calls:
    try:
        call()
    except ImportError as e:
        assert "decx_b200.build" in str(e), e
    else:
        raise SystemExit("no ImportError")
print("REFUSED")
"""


def test_the_other_front_ends_do_not_need_it():
    out = _run("""
import torch
sys.modules["decx_b200._front"] = None           # as if it were missing, or did not fit this torch
from decx_b200 import blas, capi, gemm
for call in (lambda: gemm.gemm(torch.zeros(4, 4), torch.zeros(4, 4)), lambda: blas.gemv(torch.zeros(4, 4), torch.zeros(4)),
             lambda: blas.cast(torch.zeros(4, 4), torch.float16), lambda: blas.transpose(torch.zeros(4, 4))):
    try:
        call()
    except RuntimeError as e:
        assert "CUDA tensors only" in str(e), e
print("IMPORTED", capi.workspace_bytes(capi.FP32, 64, 64, 64) > 0)
""" + LOW_PRECISION)
    assert "IMPORTED True" in out and "REFUSED" in out


def test_not_for_another_torch():
    assert "REFUSED" in _run("""
import torch
torch.__version__ = "1.0.0"
from decx_b200 import blas, gemm
""" + LOW_PRECISION)


def test_it_is_loaded_once_and_checks_as_before():
    assert "OK" in _run("""
import torch
from decx_b200 import blas, capi, gemm
assert "decx_b200._front" not in sys.modules
for _ in range(2):
    try:
        blas.cast_q8(torch.zeros(4, 16))
    except RuntimeError as e:
        assert "CUDA tensors only" in str(e), e
assert "cast_q8" in vars(capi.front) and sys.modules["decx_b200._front"].built_for == torch.__version__
print("OK")
""")


def test_another_torch_makes_it_stale(monkeypatch):
    from decx_b200 import build
    assert not build.front_stale()
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    assert build.front_stale()
