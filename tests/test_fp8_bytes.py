"""The ends of rows in 8-bit floating point: no byte behind a row's last value is read (CPU: the kernel's own load, with a page that may not be touched right
behind the row)."""
import shutil
import subprocess

import pytest

from jllm_serve_b200.csrc.build import CSRC

PROGRAM = r"""
#include "fp8_view.h"
#include <cstdio>
#include <sys/mman.h>
#include <unistd.h>
int main() {
    const long page = sysconf(_SC_PAGESIZE);
    uint8_t* two = static_cast<uint8_t*>(mmap(nullptr, 2 * page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
    for (long i = 0; i < page; ++i) two[i] = (uint8_t)(i * 7 + 3);
    if (two == MAP_FAILED || mprotect(two + page, page, PROT_NONE)) return 1;
    for (int left = 1; left <= 8; ++left) {
        const uint8_t* p = two + page - left;
        const Bytes8 b = bytes_of(p, left);
        const uint64_t both = (uint64_t)b.hi << 32 | b.lo;
        for (int j = 0; j < 8; ++j)
            if ((uint8_t)(both >> 8 * j) != (j < left ? p[j] : 0)) return 2;
    }
    const Bytes8 more = bytes_of(two, 100);
    if (more.lo != *reinterpret_cast<uint32_t*>(two) || more.hi != *reinterpret_cast<uint32_t*>(two + 4)) return 3;
    puts("within");
    return 0;
}
"""


def test_a_row_that_ends_its_memory(tmp_path):
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "ends.cpp").write_text(PROGRAM)
    made = subprocess.run([compiler, "-std=c++17", "-O1", "-I", str(CSRC), str(tmp_path / "ends.cpp"), "-o", str(tmp_path / "ends")], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    run = subprocess.run([str(tmp_path / "ends")], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout.strip() == "within", (run.returncode, run.stderr)
    # (and the kernel has no other load of a row's bytes)
    kernel = (CSRC / "fp8_rows.cu").read_text().split("fp8_values_kernel(", 1)[1].split("\n}\n", 1)[0]
    assert "bytes_of(src" in kernel and "reinterpret_cast<const uint2*>(src" not in kernel
