"""The 4-bit paged cache's launches on the CPU, and its formulas where they are
easiest to get wrong."""

from __future__ import annotations

import math
import os
import shutil
import subprocess

import pytest
import torch

import fp4_ref as ref
from quantumdlblocks_amd import _native, flash_born_attention_paged_fp4
from quantumdlblocks_amd.kernels import born_fp4

HEADER = os.path.abspath(os.path.join(os.path.dirname(born_fp4.__file__), "..", "csrc", "fp4_plan.h"))


def _run(tmp_path, body):
    """A program over the launches' rules; its output's last line where it fails."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "plan.cpp").write_text('#include <cstdio>\n#include <random>\n#include "%s"\nusing namespace qdl;\n'
                                       'const int64_t kMost = (1 << 24) - 1;\nint main() {\n%s\nreturn 0;\n}\n' % (HEADER, body))
    subprocess.run([gxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", str(tmp_path / "plan.cpp"), "-o",
                    str(tmp_path / "plan")], check=True)
    got = subprocess.run([str(tmp_path / "plan")], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout + got.stderr


def test_sequences_without_tokens_do_not_choose_the_kernel(tmp_path):
    """Which sequences are narrow goes by the tokens, heads and keys: a prompt does
    not fall to the narrow kernel for the empty sequences beside it."""
    _run(tmp_path, r"""
    std::mt19937_64 g(2);
    auto upto = [&](int64_t most) { return (int64_t)(g() % (uint64_t)(most + 1)); };
    for (int i = 0; i < 100000; ++i) {
        const int64_t h_kv = 1 + upto(8), H = h_kv * (1 + upto(8)), n = 1 + upto(700), page = 16, pages = 1 + upto((int64_t)1 << upto(12));
        const int64_t window = upto(1) ? 0 : 1 + upto(5000);
        int limit = 0;
        for (int64_t B : {1, 2, 8, 63, 500}) {
            const Fp4Plan r = fp4_plan(n, B, H, h_kv, 64, pages, page, window, true, false, kMost);
            if (limit && r.limit != limit) return printf("%ld rows of %ld sequences: %d and %d\n", (long)(n * H / h_kv), (long)B, limit, r.limit), 1;
            limit = r.limit;
        }
    }
    // 128 tokens behind a long conversation, beside seven empty sequences; drafts.
    if (fp4_plan(128, 8, 32, 8, 128, 1900, 16, 0, true, false, kMost).slots == 0) return printf("a prompt\n"), 1;
    if (fp4_plan(80, 16, 16, 4, 128, 512, 16, 0, true, false, kMost).slots != 0) return printf("drafts\n"), 1;
    """)


def test_sequences_of_several_column_blocks_fit_a_launch(tmp_path):
    """As many sequences as a call takes, whatever the heads of a group."""
    _run(tmp_path, r"""
    for (int64_t G : {1, 16, 17, 20, 33, 40, 64, 100})
        for (int weighed : {0, 1})
            for (int64_t B : {1000, 1025, 22000, 33000, 65535, 65536})
                for (int64_t pages : {1, 8, 1000})
                    if (!fp4_plan(B, B, G, 1, 128, pages, 16, 0, false, weighed, kMost).fits)
                        return printf("%ld sequences of %ld heads, %ld pages, %d\n", (long)B, (long)G, (long)pages, weighed), 1;
    """)


def test_weights_of_few_keys_take_little_room(tmp_path):
    """What is kept of the keys sizes the workspace, not the table; wide tables do
    not make a launch too large."""
    _run(tmp_path, r"""
    for (int64_t B : {1, 64, 300, 4000})
        for (int64_t pages : {1, 100, 65536}) {
            const int64_t room = pages * 16;
            for (int64_t keys : {1, 31, 100, 5000, 1 << 20}) {
                const Fp4Plan r = fp4_plan(B, B, 32, 8, 128, pages, 16, 0, false, true, kMost, keys);
                const int64_t kept = keys < room ? keys : room;
                if (!r.fits || r.raw_bytes > B * 32 * 4 * (kept + 93) || r.raw_ld < kept) return printf("%ld %ld %ld\n", (long)B, (long)pages, (long)keys), 1;
                if (r.join.weigh * B * 8 > kFp4Weigh && r.join.weigh > 1) return printf("launch\n"), 1;
            }
        }
    """)
    lib = _native.load()
    size = lambda *a: lib.qdl_flash_born_fp4_paged_workspace_size(64, 64, 32, 8, 128, 8192, 16, 0, 0, *a)  # noqa: E731
    assert size(0) < size(4096) < 64 << 20 < 1 << 30 < size(1) == size(1 << 20) and size(-1) == 0


def test_workspaces_of_calls_that_are_refused_are_empty():
    """More workgroups than a launch counts, or more bytes than 64 bits do."""
    size = _native.load().qdl_flash_born_fp4_paged_workspace_size
    for a in ((1 << 16, 1 << 16, 256, 256, 8, 1, 16, 0, 0, 1), (1 << 28, 5, 64, 64, 64, 4, 16, 0, 1, 0),
              (1 << 16, 1 << 16, 1 << 16, 1, 64, 1 << 14, 1 << 16, 0, 0, 1)):
        assert size(*a) == 0
    assert size(1 << 16, 1 << 16, 128, 128, 8, 1, 16, 0, 0, 1) > 0


@pytest.mark.parametrize("window", [0, 30])
def test_keys_that_are_not_seen_keep_their_weights(window):
    """A row that is not a number makes NaN of the weights that it sees, of no other."""
    cache, table, n, _ = ref.make_cache([90, 60], 5, 2, 64, seed=51)
    table[0, 8] = -1
    t, r = int(table[0, 17]), 0
    cache[2][t, r, 1, 0] = 255  # key 85
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(52))
    q[1, 0, 7] = math.nan
    weight = torch.full((2, 2, 120), 0.5)
    flash_born_attention_paged_fp4(q, cache, table, n, 1.0, window_size=window, key_weight=weight)
    j = torch.arange(120)
    for b, h, m in ((0, 1, 90), (1, 0, 60)):
        seen = (j < m) & (j >= (m - window if window else 0)) & ~((b == 0) & (j // 5 == 8))
        assert torch.equal(weight[b, h].isnan(), seen) and (weight[b, h][~seen] == 0.5).all()
    assert weight[0, 0].isfinite().all() and weight[1, 1].isfinite().all()
