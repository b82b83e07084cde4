"""Where the chunks of ragged rows lie in the gated delta rule's workspace (rwkv-infer-next_amd/csrc/delta_plan.h, the very header that the
library includes): every chunk of every row that runs by chunks has a slot of its own within it, the search that the kernels make finds
its row, and the workspace is in proportion to the chunks that there can be."""
import ctypes
import os
import shutil
import subprocess

import pytest

pytest.importorskip("torch")

from rwkv_next_amd import _lib  # noqa: E402

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "rwkv-infer-next_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "delta_plan.h"
using namespace delta;

static void check(const std::vector<int64_t>& cu, int64_t total, int32_t token_len, bool proper) {
    const int n = (int)cu.size() - 1;
    const Slots s = ragged_slots(n, total, token_len);
    auto fail = [&](const char* what) {
        printf("%d rows, %lld tokens, token_len %d: %s\n", n, (long long)total, token_len, what);
        exit(1);
    };
    if (s.count < 0 || s.count > total / kChunk + n || (s.rows == 0 && (s.shift > 5 || (1 << s.shift) > token_len + 1))) fail("the slots");
    std::vector<int> owner(s.count, -1);
    int64_t many = 0;
    for (int i = 0; i < n; ++i) {
        const int64_t len = cu[i + 1] - cu[i];
        if (len <= token_len) continue;
        ++many;
        for (int64_t c = 0; c < (len + kChunk - 1) / kChunk; ++c) {
            const int64_t at = ragged_slot(s.shift, s.rows, i, cu[i]) + c;
            if (at < 0 || at >= s.count) fail("a chunk outside");
            if (!proper) continue;
            if (owner[at] >= 0) fail("a slot twice");
            owner[at] = i;
            int lo = 0, hi = n;  // as the kernels do
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (ragged_slot(s.shift, s.rows, mid, cu[mid]) <= at) lo = mid; else hi = mid;
            }
            if (lo != i) fail("another row found");
        }
    }
    if (proper && many > long_rows(n, total, token_len)) fail("more rows than can be long");
}

int main() {
    std::mt19937 rng(7);
    const auto pick = [&](int64_t below) { return (int64_t)(rng() % (uint64_t)below); };
    const int32_t lens[] = {0, 1, 2, 3, 7, 14, 15, 16, 17, 30, 31, 32, 33, 62, 63, 64, 65, 200};
    for (int pass = 0; pass < 60000; ++pass) {
        const int32_t token_len = lens[pick(18)];
        const int kind = (int)pick(4), n = 1 + (int)pick(kind == 3 ? 300 : 20);
        std::vector<int64_t> cu{pick(3) ? 0 : pick(100)};
        for (int i = 0; i < n; ++i) {
            const int64_t len = kind == 0 ? pick(400) : kind == 1 ? (pick(4) ? 1 : pick(3000))
                              : kind == 2 ? token_len + pick(3) : (pick(9) ? pick(3) : token_len + 1 + pick(130));
            cu.push_back(cu.back() + len);
        }
        check(cu, cu.back() + (pick(3) ? 0 : pick(200)), token_len, true);
        const int64_t total = cu.back();  // and offsets in disorder, as the kernels clamp them: inside the workspace
        for (auto& x : cu) x = pick(total + 1);
        check(cu, total, token_len, false);
    }
    for (int32_t t : lens)  // every length at every place
        for (int64_t len = t + 1; len < t + 200; ++len)
            for (int64_t at = 0; at < 70; ++at) check({0, at, at + len, at + 2 * len, at + 2 * len + 1}, at + 2 * len + 1, t, true);
    return 0;
}
"""


def test_every_chunk_has_a_slot_of_its_own(tmp_path):
    compiler = shutil.which("g++")
    if not compiler:
        pytest.skip("no g++")
    (tmp_path / "plan.cpp").write_text(PROGRAM)
    subprocess.run([compiler, "-std=c++17", "-O2", "-Wall", f"-I{CSRC}", str(tmp_path / "plan.cpp"), "-o", str(tmp_path / "plan")], check=True)
    res = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout


def _workspace(rows, tokens, token_len=-1, Hk=16, Hv=32, K=128):
    a = _lib.DeltaArgs(cu_seqlens=0x100000, total_tokens=tokens, num_seqs=rows, T=0, Hk=Hk, Hv=Hv, K=K, V=128, scale=1.0, token_len=token_len)
    n = ctypes.c_size_t(0)
    _lib.check(_lib.load().delta_workspace_size(ctypes.byref(a), ctypes.byref(n)))
    return n.value


@pytest.mark.parametrize("rows,tokens", [(64, 64), (1024, 1024), (65536, 65536), (1024, 3071), (64, 2111), (1, 4096), (64, 10000), (300, 300)])
def test_the_workspace_is_in_proportion_to_the_tokens(rows, tokens):
    """Of rows of more than 16 tokens a chunk's slot holds 17 tokens at least: never more than one slot for each 16 tokens and one, nor than
    one for each 64 tokens and each row."""
    slot = 16 * 3 * 128 * 64 * 2 + 32 * (30 * 1024 + 1280)
    assert _workspace(rows, tokens) <= min(tokens // 16 + 1, tokens // 64 + rows) * slot + 4 * (rows + 1)


def test_no_workspace_where_no_row_can_be_long():
    assert _workspace(16, 16) == 0 and _workspace(1024, 1024, token_len=1024) == 0 and _workspace(8, 0) == 0
