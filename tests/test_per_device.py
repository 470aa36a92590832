"""What the low-precision launches ask the driver once: kept per device, and not when the query failed."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "decx_b200", "csrc")


def test_kept_per_device_and_a_failure_is_not_kept(tmp_path):
    src = tmp_path / "t.cpp"
    src.write_text(r"""
#include <cstdio>
#include "per_device.h"
static dxb_host::PerDevice known;
int main() {
    int asked = 0, answer = -1;
    auto get = [&](int device) { return known.get(device, [&] { ++asked; return answer; }); };
    bool ok = get(0) == -1 && get(0) == -1 && asked == 2;          // failed: asked again
    answer = 0;
    ok = ok && get(0) == 0 && asked == 3;
    answer = 7;
    ok = ok && get(0) == 7 && get(0) == 7 && asked == 4;
    answer = 9;
    ok = ok && get(0) == 7 && get(1) == 9 && get(1) == 9 && asked == 5;
    ok = ok && get(63) == 9 && get(64) == 9 && get(64) == 9 && get(-1) == 9 && asked == 9;     // beyond the table: asked every time
    std::puts(ok ? "OK" : "WRONG");
}
""")
    exe = str(tmp_path / "t")
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, str(src), "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True).stdout == "OK\n"


def test_launches_keep_no_occupancy_by_themselves():
    text = open(os.path.join(CSRC, "capi_lowbit.cu")).read()
    text = re.sub(r"//[^\n]*", "", text)
    assert text.count("cudaOccupancyMax") == text.count(".get(device, [&]") + 1      # one lambda asks in one of two ways
    assert "known.store" not in text and "held[p.ranks - 1][warps - 1].store" not in text
    assert not re.search(r"\b(74|73|147)\b", text), "SMs are asked for"
