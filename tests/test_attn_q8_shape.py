"""Sizes of pages of 8 bits, and which kernel attends over them (attn_shape.h)."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("attn") / "attn_q8_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "moe4all_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "attn_q8_check.cpp"), "-o", exe], check=True)
    return lambda *a: subprocess.run([exe, *map(str, a)], capture_output=True, text=True, check=True).stdout.split()


def test_bytes(ask):
    assert ask("bytes", 7, 48, 3, 80, 1) == [str(7 * 48 * 3 * 80)]
    assert ask("bytes", 7, 48, 3, 80, 2) == [str(2 * 7 * 48 * 3 * 80)]
    # past 64 bits: more than any buffer has
    big = (1 << 32) - 1
    assert ask("bytes", big, big, 4096, 256, 1) == [str((1 << 64) - 1)]


@pytest.mark.parametrize("seed", range(30))
def test_room_for_f16_pages(ask, seed):
    """Every page that some sequence names has a place: its own, or one of the sequence's."""
    r = random.Random(seed)
    n_seq, max_pages, n_pages = r.choice([1, 3, 64, 4096]), r.choice([1, 5, 200, 1 << 20]), r.choice([1, 16, 1000, 1 << 30])
    page, n_kv, hd = 16 * r.choice([1, 3, 64]), r.choice([1, 8, 128]), 16 * r.choice([1, 5, 16])
    got = ask("unpack", n_seq, max_pages, n_pages, page, n_kv, hd)
    fewer, bytes_ = min(n_seq * max_pages, n_pages), 2 * page * n_kv * hd
    if fewer * bytes_ > 1 << 47:
        assert got == ["no"]
        return
    by_sequence, pages, table, side = map(int, got)
    assert by_sequence == (n_seq * max_pages < n_pages) and pages == fewer and side == fewer * bytes_
    # the table has a number to each place, and the pages behind it begin on a 256-byte border
    assert table % 256 == 0 and (table >= 4 * n_seq * max_pages if by_sequence else table == 0)
    assert side % 16 == 0


def test_which_kernel(ask):
    for hd, limit in ((16, 16), (128, 16), (144, 8), (256, 8)):
        for g in (1, limit, limit + 1):
            got = ask("few", 1, g, hd, 64)
            assert got == [str(limit), str(int(g <= limit))]
    for pairs, most in ((1, 64), (8, 64), (9, 48), (16, 48), (17, 32), (10 ** 6, 32)):
        assert [ask("few", n, 1, 128, pairs)[1] for n in (0, most, most + 1)] == ["1", "1", "0"]
