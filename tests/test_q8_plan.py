"""Which kernel takes an 8-bit product (csrc/q8plan.h), compiled for the host: no
GPU needed."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STAGING = 96 * 1024

MAIN = r"""
#include <cstdio>
#include "q8plan.h"
int main() {
    long m, k, n, sms;
    while (scanf("%ld %ld %ld %ld", &m, &k, &n, &sms) == 4) {
        const dz::Q8Plan p = dz::q8_plan(m, k, n, sms, 96 * 1024);
        printf("%d %d %.3f\n", p.rows, p.parts, p.time);
    }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    src, exe = d / "plan.cpp", d / "plan"
    src.write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "dranzer_b200", "csrc"),
                    str(src), "-o", str(exe)], check=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout
        return [(int(r), int(p), float(t)) for r, p, t in (line.split() for line in out.splitlines())]
    return run


CASES = [(m, k, n, sms) for m in (1, 2, 8, 9, 16, 17, 33, 128, 257, 4096, 1 << 24) for k in (1, 128, 515, 4096, 12032, 131072)
         for n in (1, 130, 5003, 32000, 1 << 20) for sms in (148, 132, 20)]


def test_every_product_has_a_kernel_that_takes_it(plan):
    for (m, k, n, sms), (rows, parts, time) in zip(CASES, plan(CASES)):
        assert rows in (8, 16, 32, 64, 128, 256) and 0 < time < 1e12
        steps = -(-k // 128)
        assert parts in (1, 2, 4, 8) and (parts == 1 or 2 * parts <= steps) and (parts == 1 or 32 <= rows <= 128)
        if rows <= 16:
            assert m <= 16
        if rows == 16:
            assert m > 8 and m * (steps * 128 + 64) <= STAGING
        if 32 <= rows <= 128:      # blocks of a launch
            assert -(-n // 128) * -(-m // rows) * parts < 2 ** 31


def test_more_of_a_product_is_never_estimated_to_take_less(plan):
    """More columns or more k: the next size up, in whole tiles and steps."""
    for m in (1, 8, 16, 40, 130, 700, 4096):
        for k in (256, 4096):
            times = [t for _, _, t in plan([(m, k, n, 148) for n in range(256, 256 * 400, 256 * 8)])]
            assert all(b >= a - 1e-9 for a, b in zip(times, times[1:])), (m, k)


def test_measured_sides(plan):
    """The cases of the comment: the faster side is chosen."""
    got = plan([(8, 2048, 2048, 148), (1, 4096, 32000, 148), (32, 4096, 5120, 148), (131, 4096, 5120, 148),
                (256, 4096, 16384, 148), (256, 4096, 5120, 148), (4096, 4096, 16384, 148)])
    assert [g[:2] for g in got] == [(8, 1), (32, 1), (32, 4), (64, 2), (256, 1), (64, 1), (256, 1)]
