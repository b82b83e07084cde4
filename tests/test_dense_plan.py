"""The plans of products with 16-bit weights (rwkv-infer-next_amd/csrc/dense_plan.h, the very header that the library includes) carried through
what the kernel assumes of them, over sizes up to the largest; and the sizes of the GPU tests against the tiles that they name."""
import os
import shutil
import subprocess

import pytest

from test_gpu_dense_tiles import SHAPES

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC, INCLUDE = os.path.join(REPO, "rwkv-infer-next_amd", "csrc"), os.path.join(REPO, "include")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "dense.h"
#include "dense_plan.h"
using namespace dense;

static void check(int32_t M, int32_t N, int32_t K, int cus) {
    const Plan p = plan(M, N, K, cus);
    auto fail = [&](const char* what) {
        printf("M %d, N %d, K %d on %d CUs: %s\n", M, N, K, cus, what);
        exit(1);
    };
    const Tile t = kTiles[p.shape];
    // every tile begins at a row and a column of the result, and they hold all of them
    if (p.row_groups * t.rows < M || (p.row_groups - 1) * t.rows >= M) fail("rows");
    if (p.strip_groups * t.columns < N || (p.strip_groups - 1) * t.columns >= N) fail("columns");
    const int64_t panels = (steps(K) + kPanelSteps - 1) / kPanelSteps;
    if (p.parts < 1 || p.parts > 16 || (p.parts > 1 && p.parts * t.k_groups * kPartPanels > panels)) fail("parts");
    if (p.parts > 1 ? p.workspace < (size_t)p.parts * M * N * 4 : p.workspace != 0) fail("the workspace");
    if (M <= DENSE_UNSPLIT_ROWS && K < DENSE_UNSPLIT_K && p.workspace) fail("a workspace that nobody asks for");
    // offsets of 32 bits: the rows of A among which a wavefront group's lanes choose
    if ((uint64_t)(t.threads / t.k_groups / 8 - 1) * DENSE_MAX_ROW_STRIDE * 2 + (uint64_t)DENSE_MAX_ROW_STRIDE * 2 > 0xFFFFFFFFu) fail("an offset in A");
    if (p.grid % 8 || p.grid < p.row_groups * p.strip_groups * p.parts) fail("the grid");
    // K's panels: each in one group of one part
    const int64_t groups = p.parts * t.k_groups, each = (panels + groups - 1) / groups;
    int64_t next = 0;
    for (int64_t g = 0; g < groups; ++g) {
        const int64_t first = std::min(g * each, panels), end = std::min(first + each, panels);
        if (first != next) fail("a panel twice or not at all");
        next = end;
    }
    if (next != panels) fail("panels");
    if (p.grid > 300000) return;
    std::vector<char> seen((size_t)(p.row_groups * p.strip_groups * p.parts));
    for (uint32_t b = 0; b < (uint32_t)p.grid; ++b) {  // as the kernel does
        const uint32_t rows = (uint32_t)p.row_groups, tiles = rows * (uint32_t)p.strip_groups, units = tiles * (uint32_t)p.parts;
        const uint32_t share = (units + 7) / 8, unit = (b & 7) * share + (b >> 3);
        if ((b >> 3) >= share || unit >= units) continue;
        const uint32_t tile = unit % tiles, band = tile / (4 * rows), in = tile % (4 * rows);
        const uint32_t width = std::min(4u, (uint32_t)p.strip_groups - 4 * band), row = in / width, column = 4 * band + in % width;
        if (row >= rows || column >= (uint32_t)p.strip_groups) fail("a tile outside");
        char& s = seen[((size_t)(unit / tiles) * rows + row) * p.strip_groups + column];
        if (s) fail("a tile twice");
        s = 1;
    }
    for (char s : seen)
        if (!s) fail("a tile without a workgroup");
}

int main(int argc, char** argv) {
    if (argc > 1) {
        for (int i = 1; i + 2 < argc; i += 3) {
            const Plan p = plan(atoi(argv[i]), atoi(argv[i + 2]), atoi(argv[i + 1]), 256);
            printf("%d/%d%s\n", (int)p.shape, p.parts, p.stream ? "s" : "");
        }
        return 0;
    }
    const int32_t rows[] = {1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 129, 255, 257, 500, 1000, 2049, 4096, 10000, 65536};
    const int32_t cols[] = {1, 15, 16, 17, 63, 64, 65, 96, 255, 256, 257, 768, 1000, 2560, 4096, 4099, 8192, 8193, 16384, 65536, 151936};
    const int32_t ks[] = {32, 64, 96, 768, 2560, 2592, 4096, 6080, 6112, 6144, 10240, 16384, 65536};
    for (int cus : {1, 64, 256, 304})
        for (int32_t M : rows)
            for (int32_t N : cols)
                for (int32_t K : ks) check(M, N, K, cus);
    check(0x7FFFFFFF, 1, 32, 256);
    check(1, 0x7FFFFFFF, 32, 256);
    check(0x7FFFFFFF, 0x7FFFFFFF, 0x7FFFFFE0, 256);
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    compiler = shutil.which("g++")
    if not compiler:
        pytest.skip("no g++")
    where = tmp_path_factory.mktemp("dense_plan")
    (where / "plan.cpp").write_text(PROGRAM)
    subprocess.run([compiler, "-std=c++17", "-O2", "-Wall", f"-I{CSRC}", f"-I{INCLUDE}", str(where / "plan.cpp"), "-o", str(where / "plan")],
                   check=True)
    return str(where / "plan")


def test_plans_are_what_the_kernel_assumes(program):
    res = subprocess.run([program], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout


def test_the_gpu_tests_reach_every_tile(program):
    args = [str(x) for shape in SHAPES for x in shape]
    got = subprocess.run([program, *args], capture_output=True, text=True, check=True).stdout.split()
    assert len(got) == len(SHAPES)
    assert {int(x.split("/")[0]) for x in got} == set(range(6))
    # in parts too, but for 16 x 64: more than two tiles of 16 x 16 a CU are more than half a one of 16 x 64
    assert {int(x.split("/")[0]) for x in got if x.rstrip("s").split("/")[1] != "1"} == {0, 2, 3, 4, 5}, got
    streams = {int(x.split("/")[0]) for x in got if x.endswith("s")}
    assert streams == {1, 2, 3}, got
