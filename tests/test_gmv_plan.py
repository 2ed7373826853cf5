"""How a group-scaled product is cut (csrc/gmvplan.h), compiled for the host: no
GPU needed. A device partition that cannot hold a cluster size is a room of 0."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MAIN = r"""
#include <cstdio>
#include "gmvplan.h"
using namespace dz;
// lines of: rows K N group scale_bytes parts, then the room's ten counts
int main() {
    long rows, k, n;
    int group, sb, parts;
    while (scanf("%ld %ld %ld %d %d %d", &rows, &k, &n, &group, &sb, &parts) == 6) {
        GmvRoom room;
        for (int two = 0; two < 2; two++)
            for (int c = 0; c < 5; c++) {
                int v;
                if (scanf("%d", &v) != 1) return 1;
                room.clusters[two][c] = v;
            }
        GmvShape s{(int)((n + 31) / 32), (int)((k + 127) / 128), group, GMV_CODES + 128 / group * 32 * sb, parts};
        GmvPlan p{};
        int ok = gmv_plan(s, (int)rows, room, &p);
        if (!ok) {
            const int tiles = gmv_plan_tiles(s, s.ntiles, (int)rows, room, &p);
            ok = -tiles;   // the first launch of several takes so many
        }
        printf("%d %d %d %d %d %d %d %d\n", ok, p.rows, p.digits, p.cluster, p.clusters, p.slice, p.tiles,
               ok ? gmv_smem(s, p) : 0);
    }
}
"""
FULL = [148, 74, 36, 17, 8, 296, 148, 72, 34, 16]


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    src, exe = d / "plan.cpp", d / "plan"
    src.write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "dranzer_b200", "csrc"),
                    str(src), "-o", str(exe)], check=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, [*c, *room])) for c, room in cases)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout
        names = ("ok", "rows", "digits", "cluster", "clusters", "slice", "tiles", "smem")
        return [dict(zip(names, map(int, line.split()))) for line in out.splitlines()]
    return run


CASES = [(rows, k, n, group, sb, parts) for rows in (1, 2, 3, 8, 16, 40) for k in (1, 128, 515, 4096, 12032, 100000)
         for n in (1, 32, 5003, 32000) for group, sb in ((128, 2), (32, 4)) for parts in (1, 3)]


def _check(c, room, p):
    rows, k, n, *_ = c
    blocks, tiles = -(-k // 128), -(-n // 32)
    i = p["cluster"].bit_length() - 1
    assert 1 << i == p["cluster"] <= blocks and 1 <= p["rows"] <= min(rows, 16)
    assert p["digits"] == 0 or p["rows"] == 1
    assert p["slice"] * p["cluster"] >= blocks and p["tiles"] * p["clusters"] >= tiles >= p["clusters"]
    held = [two for two in range(2) if room[5 * two + i] >= p["clusters"] and p["smem"] <= (227, 113)[two] * 1024 - 128]
    assert held, (c, room, p)


def test_plans_fit_and_cover(plan):
    for c, p in zip(CASES, plan([(c, FULL) for c in CASES])):
        assert p["ok"], c
        _check(c, FULL, p)


@pytest.mark.parametrize("most", [1, 2, 4, 8])
def test_clusters_that_the_device_cannot_hold_are_not_chosen(plan, most):
    """Rooms without clusters of more than `most` blocks; what still fits is planned within them."""
    keep = [1 << i <= most for i in range(5)] * 2
    room = [v if k else 0 for v, k in zip([20, 10, 5, 2, 1, 40, 20, 10, 4, 2], keep)]
    for c, p in zip(CASES, plan([(c, room) for c in CASES])):
        if p["ok"] > 0:
            assert p["cluster"] <= most
            _check(c, room, p)
        else:
            assert c[1] == 100000      # only rows too long for `most` blocks are refused
    assert all(p["ok"] for c, p in zip(CASES, plan([(c, room) for c in CASES])) if c[1] <= 12032)


def test_a_device_that_holds_no_block_has_no_plan(plan):
    assert not plan([((1, 4096, 4096, 128, 4, 3), [0] * 10)])[0]["ok"]


def test_wide_matrices_go_in_several_launches(plan):
    """Tiles whose sums do not fit shared memory beside long rows; the first launch's plan holds its share."""
    cases = [(rows, k, n, group, 4, parts) for rows in (1, 16) for k, n in ((100000, 300000), (200000, 200000), (64, 1 << 24),
             (4096, 1 << 24)) for group in (32, 128) for parts in (1, 3)]
    for c, p in zip(cases, plan([(c, FULL) for c in cases])):
        assert p["ok"] != 0, c
        if p["ok"] < 0:
            assert -p["ok"] < -(-c[2] // 32)
            _check((c[0], c[1], -p["ok"] * 32), FULL, p)
        else:
            _check(c, FULL, p)


def test_the_longest_rows(plan):
    """Rows of 348000 (what three digits of fp32 fitted) and more still have a plan, of any type and group."""
    cases = [(rows, 350000, 64, group, sb, parts) for rows in (1, 2, 16) for group in (32, 64, 128) for sb in (2, 4)
             for parts in (1, 3)]
    for c, p in zip(cases, plan([(c, FULL) for c in cases])):
        assert p["ok"] > 0, c
        _check(c, FULL, p)
