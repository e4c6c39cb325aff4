"""What the 8-bit cache's libraries remember between calls belongs to a device: several may be current in turn."""
import os
import re
import subprocess

import pytest

from go_tinygrad_b200.kernels import build

E4M3 = ["kv_e4m3.cu", "attention_e4m3.cu", "attention_e4m3_few.cuh", "attention_e4m3_tcgen05.cu", "e4m3.cuh"]


@pytest.mark.parametrize("name", E4M3)
def test_nothing_is_remembered_for_all_devices(name):
    """Shared memory above 48 KB is allowed per device and kernel: no plain flag or size says that it has been, and only
    allow_shared and the count of workers, which keep a place a device, ask for it."""
    with open(os.path.join(build.CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    kept = re.findall(r"static (?:bool|int|size_t) (\w+(?:\[\w+\])?) = ", text)
    assert all(k.endswith("[kMaxDevices]") for k in kept), kept
    asked = len(re.findall(r"cudaFuncSetAttribute\(", text))
    assert asked == {"e4m3.cuh": 1, "attention_e4m3_few.cuh": 1}.get(name, 0)


PROGRAM = r"""
#include <cstdio>
#include <cstddef>
// stands in for the runtime: a current device and, per device, what a kernel may take
typedef int cudaError_t;
enum { cudaSuccess = 0, cudaFuncAttributeMaxDynamicSharedMemorySize = 8 };
static int current = 0, calls = 0;
static size_t may[200];
static cudaError_t cudaGetDevice(int* d) { *d = current; return cudaSuccess; }
static cudaError_t cudaFuncSetAttribute(const void*, int, int bytes) { ++calls; if (bytes < 0) return 1; may[current] = bytes; return cudaSuccess; }
%s
int main() {
    static bool done[kMaxDevices] = {};
    const int devices[] = {0, 1, 0, 63, 1, 150, 150, 0};
    for (int d : devices) {
        current = d;
        if (allow_shared((const void*)&calls, 1000, done) != 0 || may[d] != 1000) return 1;
    }
    if (calls != 5) return 2;                          // once for 0, 1 and 63; each time where there is no place
    static bool other[kMaxDevices] = {};
    current = 2;
    if (allow_shared((const void*)&calls, (size_t)-1, other) == 0 || other[2]) return 3;      // a failure is not remembered
    return allow_shared((const void*)&calls, 7, other) != 0 || may[2] != 7;
}
"""


def test_shared_memory_is_allowed_once_a_device(tmp_path):
    with open(os.path.join(build.CSRC, "e4m3.cuh")) as f:
        text = f.read()
    at = text.index("constexpr int kMaxDevices")
    function = text[at: text.index("\n}\n", at) + 3]
    (tmp_path / "p.cpp").write_text(PROGRAM % function)
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "p"), str(tmp_path / "p.cpp")], check=True)
    assert subprocess.run([str(tmp_path / "p")]).returncode == 0
