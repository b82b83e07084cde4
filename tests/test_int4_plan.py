"""The plans of 4-bit products (rwkv-infer-next_amd/csrc/w4a16_plan.h, the very header that the library includes) carried through what the
kernels assume of them, over sizes up to the largest; and the sizes of the GPU tests against the variants that they name."""
import os
import shutil
import subprocess

import pytest

from test_gpu_int4_variants import DEPTHS, SIZES

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC, INCLUDE = os.path.join(REPO, "rwkv-infer-next_amd", "csrc"), os.path.join(REPO, "include")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "w4a16.h"
#include "w4a16_plan.h"
using namespace w4;

static void check(int32_t M, int32_t N, int32_t K, int cus) {
    const Plan p = plan(M, N, K, cus);
    auto fail = [&](const char* what) {
        printf("M %d, N %d, K %d on %d CUs: %s\n", M, N, K, cus, what);
        exit(1);
    };
    const bool blocks = p.shape != kStrips;
    const int rows = 16 * p.mt, columns = p.shape == kBlock256 ? 256 : p.shape == kBlock128 ? 128 : p.shape == kBlock64 ? 64 : 16 * p.nt;
    if (blocks ? p.mt != 2 && p.mt != 4 : p.mt != 1 || (p.nt != 1 && p.nt != 2 && p.nt != 4)) fail("no such variant");
    if (blocks && M <= 16) fail("blocks for the rows of one strip");
    if (blocks && p.strip_groups * p.row_groups < cus) fail("blocks that leave a CU without one");
    if (p.waves < 1 || p.waves > 8 || (!blocks && p.waves > chunks(K))) fail("wavefronts");
    if (!blocks && p.waves * p.nt * 1024 > 65536) fail("LDS");
    // every row group begins at a row of A, and they hold all rows; so for columns
    if (p.row_groups * rows < M || (p.row_groups - 1) * rows >= M) fail("rows");
    if (p.strip_groups * columns < N || (p.strip_groups - 1) * columns >= N) fail("columns");
    // offsets of 32 bits: a block's rows of A
    if ((uint64_t)(rows - 1) * W4A16_MAX_ROW_STRIDE * 2 > 0xFFFFFFFFu) fail("an offset in A");
    if (p.grid % 8 || p.grid < p.strip_groups * p.row_groups) fail("the grid");
    if (p.strip_groups * (columns / 16) > 0x7FFFFFFF) fail("a strip's number");
    if (p.grid > 2000000) return;
    std::vector<bool> seen(p.strip_groups * p.row_groups);
    for (uint32_t b = 0; b < (uint32_t)p.grid; ++b) {  // as the kernels do
        const uint32_t on_xcd = b >> 3, group = on_xcd / (uint32_t)p.row_groups * 8 + (b & 7), row = on_xcd % (uint32_t)p.row_groups;
        if (group >= (uint32_t)p.strip_groups) continue;
        if (seen[(size_t)group * p.row_groups + row]) fail("a tile twice");
        seen[(size_t)group * p.row_groups + row] = true;
    }
    for (bool s : seen)
        if (!s) fail("a tile by nobody");
}

int main(int argc, char** argv) {
    if (argc == 4) {  // M N K: the plan on 256 CUs
        const Plan p = plan(atoi(argv[1]), atoi(argv[2]), atoi(argv[3]), 256);
        const char* names[] = {"strips", "block 256", "block 128", "block 64"};
        printf("%s %d %d\n", names[p.shape], p.mt, p.shape == kStrips ? p.nt : p.shape == kBlock64 ? 1 : 2);
        return 0;
    }
    const int32_t ms[] = {1, 2, 15, 16, 17, 31, 32, 33, 48, 64, 65, 128, 129, 203, 256, 1000, 4096, 65537, 2147483647};
    const int32_t ns[] = {1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 768, 2560, 4096, 4897, 8191, 9857, 10240, 16384, 33000, 65281, 65536,
                          1000003, 2147483632, 2147483647};
    const int32_t ks[] = {32, 128, 160, 1024, 1056, 4096, 2147483616};
    for (int32_t M : ms)
        for (int32_t N : ns)
            for (int32_t K : ks)
                for (int cus : {1, 104, 228, 256, 304}) check(M, N, K, cus);
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("amdclang++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("int4_plan")
    (d / "p.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{CSRC}", f"-I{INCLUDE}", "-o", str(d / "p"), str(d / "p.cpp")],
                   check=True, capture_output=True, text=True)
    return str(d / "p")


def test_every_plan_is_one_that_its_kernel_takes(program):
    r = subprocess.run([program], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("shape,M,N", SIZES)
def test_the_tests_sizes_reach_their_variants(program, shape, M, N):
    for K, _ in DEPTHS:
        r = subprocess.run([program, str(M), str(N), str(K)], capture_output=True, text=True, timeout=60, check=True)
        assert r.stdout.strip() == "%s %d %d" % shape
