"""The shares of the attention over a paged cache, followed block by block on the
host: the schedule's own headers, compiled for a wave of 64 host lanes.  Every key
of every item is taken once, and where the table is too narrow for a workspace no
item is divided, whatever the lengths."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "bluewolf-plus-plus_amd", "csrc")

# Tiles' rows, blocks on 256 CUs, keys up to which items stay whole, an item's own cost in keys.
KINDS = {"f32": (16, 512, 256, 96), "f32_rows": (128, 512, 256, 96), "f32_rows_wide": (128, 256, 256, 96),
         "few": (32, 512, 512, 192), "r128": (128, 512, 1024, 384), "r128_wide": (128, 256, 1024, 384),
         "r256": (256, 256, 1024, 384)}
EVERY = 2 ** 31 - 1


@pytest.fixture(scope="module")
def schedule(tmp_path_factory):
    top = tmp_path_factory.mktemp("schedule")
    inner = top / "kernels"
    inner.mkdir()
    for name in ("kv_cache.h", "kv_schedule.h", "kv_items.h"):
        shutil.copy(os.path.join(CSRC, "kernels", name), inner)
    shutil.copy(os.path.join(CSRC, "kargs.h"), top)
    shutil.copy(os.path.join(ROOT, "tests", "c", "host_wave.h"), inner / "common.h")
    shutil.copy(os.path.join(ROOT, "tests", "c", "cache_schedule.cpp"), inner)
    exe = str(top / "cache_schedule")
    subprocess.run(["g++", "-std=c++17", "-O1", "-U_FORTIFY_SOURCE", "-Wall", "-Wno-unknown-pragmas", "-Werror", "-o", exe,
                    str(inner / "cache_schedule.cpp")], check=True)

    def run(kind, seqs, group=4, heads=8, page_shift=6, pages=None, mask=0):
        rows, blocks, whole, item = KINDS[kind]
        if pages is None:  # a table that holds every sequence
            pages = max(((max(h, 0) + n) >> page_shift) + 1 for h, n in seqs)
        args = [rows, blocks, whole, item, group, heads, page_shift, pages, mask]
        r = subprocess.run([exe] + [str(x) for x in args] + [f"{h}:{n}" for h, n in seqs], capture_output=True, text=True,
                           timeout=100)
        assert r.returncode == 0, (kind, args, seqs[:8], r.stdout, r.stderr)
        return int(r.stdout.split()[-1])

    return run


@pytest.mark.parametrize("kind", KINDS)
def test_every_key_is_taken_once(schedule, kind):
    schedule(kind, [(0, 1)])
    schedule(kind, [(0, 0), (5, 0), (63, 1), (0, 0)])
    schedule(kind, [(1000, 1), (0, 3), (64, 1), (7000, 1)], group=1, heads=3, page_shift=4)
    schedule(kind, [(h * 37 % 5000, 1 + h % 2) for h in range(100)])
    schedule(kind, [(4096, 48), (100, 48), (0, 48), (12000, 13)], mask=1)
    schedule(kind, [(0, 700), (3000, 1), (17, 333)], group=8, heads=2)
    assert schedule(kind, [(30000, 1)]) > 0  # long sequences are shared out


@pytest.mark.parametrize("mask", [0, 1])
@pytest.mark.parametrize("kind", KINDS)
def test_narrow_tables_divide_nothing(schedule, kind, mask):
    """Tables of at most the keys whose items stay whole have no workspace: sequences that
    fill them, end past them or name any length leave every item whole."""
    whole = KINDS[kind][2]
    for slots in (whole // 2, whole):
        for held in (0, slots, EVERY):
            for n in (1, 2000):
                assert schedule(kind, [(held, n)], pages=slots // 64, mask=mask) == 0
        assert schedule(kind, [(slots, 1), (slots, 1), (3, 2), (EVERY, 3)], pages=slots // 64, mask=mask) == 0
        assert schedule(kind, [(slots - 24, 48)] * 8, pages=slots // 64, mask=mask) == 0


@pytest.mark.parametrize("kind", KINDS)
def test_sequences_past_a_wider_table(schedule, kind):
    """With a workspace: sequences that end past the table, and a table that is cut at 2^31 slots."""
    whole = KINDS[kind][2]
    for held, n in ((whole + 64, 1), (whole + 10, 300), (EVERY, 5)):
        schedule(kind, [(held, n), (70, 2)], pages=whole // 64 + 1)
    schedule(kind, [(2 ** 20, 3)], pages=2 ** 26)
