"""Numbers that are asked for once per device (csrc/per_device.h): one GPU's answer is not another's, nor one kernel's another's."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include "per_device.h"
#include <type_traits>
using aristos::PerDevice;
int asked = 0;
int main() {
    // as a launch keeps it: a table per kernel, which is a template of the values that name it
    auto pairs = [](auto kernel, int device) {
        static PerDevice known;
        int n = known.get(device);
        if (n == 0) {
            ++asked;
            n = 100 * decltype(kernel)::value + 10 + device;
            known.set(device, n);
        }
        return n;
    };
    std::integral_constant<int, 1> a;
    std::integral_constant<int, 2> b;
    for (int round = 0; round < 2; ++round) {
        if (pairs(a, 0) != 110 || pairs(a, 1) != 111 || pairs(b, 0) != 210 || pairs(b, 63) != 273) return 1;
        if (asked != 4) return 2;
    }
    if (pairs(a, 64) != 174 || pairs(a, -1) != 109 || pairs(a, 64) != 174 || asked != 7) return 3;   // outside: asked every time
    return 0;
}
'''


def test_a_number_per_device_and_kernel(tmp_path):
    src, exe = tmp_path / "use.cpp", tmp_path / "use"
    src.write_text(PROGRAM)
    subprocess.check_call(["/usr/bin/g++", "-std=c++17", "-Wall", "-Werror", "-I",
                           os.path.join(ROOT, "cuplayground_b200", "csrc"), str(src), "-o", str(exe)])
    assert subprocess.run([str(exe)], timeout=60).returncode == 0

