"""How the attention over shared pages cuts keys (csrc/shared_plan.h), compiled for the host: every begin that a task may form lies
within 32 bits, and where it lies is what the definition says, for all that the entry accepts (no GPU)."""

import ctypes as C
import os
import shutil
import subprocess

import pytest

from draftkv import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "draft-kv_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "pages.h"
#include "shared_plan.h"
int main(int n, char**) {
    if (n > 1) return printf("%lld %d\n", (long long)dkv::COPY_BLOCKS, dkv::COPY_THREADS), 0;
    long long keys, max_len, groups, least, most, prefix, unit, B, held;
    while (scanf("%lld %lld %lld %lld %lld %lld %lld %lld %lld", &keys, &max_len, &groups, &least, &most, &prefix, &unit, &B, &held) == 9) {
        int p = 0, s = 0;
        dkv::sa_units(keys, (int)max_len, groups != 0, (int)least, (int)most, (int)prefix, (int)unit, p, s);
        printf("%d %d", p, s);
        for (int u : {0, 1, s / 2, s - 2, s - 1}) printf(" %d %d", u, u < 0 ? 0 : dkv::sa_unit_begin((int)B, u, (int)unit, (int)held));
        printf("\n");
    }
}
"""

MOST_POSITIONS = (1 << 31) - (1 << 16) - 1      # what the entry accepts


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("needs g++")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-fwrapv", "-I", CSRC, str(d / "plan.cpp"), "-o", str(d / "plan")], check=True)

    def run(rows):
        if rows is None:
            return [int(x) for x in subprocess.run([str(d / "plan"), "copies"], check=True, capture_output=True, text=True).stdout.split()]
        text = "\n".join(" ".join(str(int(x)) for x in r) for r in rows)
        out = subprocess.run([str(d / "plan")], input=text, check=True, capture_output=True, text=True).stdout
        return [[int(x) for x in line.split()] for line in out.splitlines()]

    return run


def test_begins_stay_within_32_bits(plan):
    """Units are counted from the least that any sequence shares, and begin behind what their own shares: a unit past the
    sequence's keys has no begin (-1), and no other passes 2^31."""
    rows = []
    for keys in (MOST_POSITIONS, 16 * 134213631, 1 << 30, (1 << 30) + 4096, 5000, 1):
        for unit in (32, 128, 65536):
            for B in (0, 32, 4096, 131072, 1 << 29, 1 << 30, keys // 2 // 32 * 32, keys // 32 * 32):
                for held in (keys, keys - 1, keys // 2, B + 1, B, 1, 0):
                    if B <= keys and 0 <= held <= keys:
                        for least in {0, min(B, 64), B}:
                            rows.append((keys, keys, 1, least, B, 65536, unit, B, held))
    assert len(rows) > 1000
    past = 0
    for r, got in zip(rows, plan(rows)):
        keys, _, _, least, most, prefix, unit, B, held = r
        units_p, units_s = got[:2]
        assert units_p == -(-(most // 32 * 32) // prefix)
        assert units_s == (-(-(keys - least // 32 * 32) // unit) if least // 32 * 32 < keys else 0)
        assert units_p * prefix < 1 << 31 and max(units_s - 1, 0) * unit < 1 << 31
        for u, begin in zip(got[2::2], got[3::2]):
            if u < 0 or u >= max(units_s, 1):
                continue
            true = B + u * unit
            if u > 0 and true >= held:
                assert begin == -1, (r, u)
                past += true >= 1 << 31
            else:
                assert begin == true and begin + unit < 1 << 31, (r, u)
    assert past > 0


def test_launches_of_page_copies_stay_below_2_to_the_32_work_items(plan):
    """The runtime refuses a launch of 2^32 work-items and more, which pages of any power of two would come to."""
    blocks, threads = plan(None)
    assert blocks * threads < 1 << 32
    for pieces in (1, 2, 3, 512, 4096, 1 << 23, blocks):
        assert 1 <= blocks // pieces * pieces <= blocks


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_padding_rows_stay_within_32_bits():
    """start + t of a padding row, t up to T past the table's last position: calls in which it passes 2^31 are refused."""
    L = _lib.lib()
    fake = 4096      # an address that is never read
    groups = _lib.Groups()
    for blocks, T, fine in (((1 << 31) - (1 << 16) - 1, 70000, False), ((1 << 31) - 100000, 100000, False), ((1 << 31) - 100000, 99999, True),
                            (1 << 20, 1 << 20, True)):
        cache = _lib.Paged(pool=fake, block_table=fake, batch=1, n_layers=1, n_kv_heads=1, head_dim=64, block_size=1, max_blocks=blocks,
                           dtype=1)
        need = L.dkv_shared_attention_workspace(C.byref(cache), C.byref(groups), T, 1, 100, 32, 32)
        assert (need > 0) == fine, (blocks, T)
        if not fine:
            rc = L.dkv_shared_attention(C.byref(cache), C.byref(groups), 0, fake, 0, T, 1, fake, fake, 100, 32, 32, fake, None, 0, None)
            assert rc == -1 and b"2^31" in L.dkv_last_error()


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_attention_of_more_workgroups_than_a_launch_takes():
    """Work-items of a launch stay below 2^32: rows are cut into launches, and where one row per sequence is too much the call is
    refused before anything is launched."""
    L = _lib.lib()
    fake = 4096      # an address that is never read
    groups = _lib.Groups()

    def cache(**kw):
        return _lib.Paged(**dict(dict(pool=fake, block_table=fake, batch=1, n_layers=1, n_kv_heads=1, head_dim=1, block_size=1, max_blocks=64,
                                      dtype=1), **kw))

    c = cache(batch=2, max_blocks=MOST_POSITIONS)      # 2^27 units, a wave each
    need = L.dkv_shared_attention_workspace(C.byref(c), C.byref(groups), 1, 1, MOST_POSITIONS, 32, 32)
    assert need >= 2 * 12 * 67106816
    rc = L.dkv_shared_attention(C.byref(c), C.byref(groups), 0, fake, 0, 1, 1, fake, None, MOST_POSITIONS, 32, 32, fake, fake, need, None)
    assert rc == -1 and b"grid too large" in L.dkv_last_error(), (rc, L.dkv_last_error())
    # the merge takes a workgroup per row: 64 keys in two units, rows of a call by the workspace and by the launch
    c = cache(batch=8)
    for Hq, T in ((1, 1 << 22), (1 << 10, 1 << 12)):
        need = L.dkv_shared_attention_workspace(C.byref(c), C.byref(groups), T, Hq, 64, 32, 32)
        rows = (need - 8) // (4 * 2 * 3)
        assert 0 < rows < 1 << 24 and rows % (8 * Hq) == 0, rows
