"""The far ends of what an attention call may be given: sizes, windows and row numbers whose arithmetic needs more bits than the values have."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("attn") / "attn_ranges_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fwrapv", "-I", os.path.join(ROOT, "moe4all_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "attn_ranges_check.cpp"), "-o", exe], check=True)
    return lambda *args: subprocess.run([exe, *map(str, args)], capture_output=True, text=True, check=True).stdout.split()


@pytest.mark.parametrize("pages,page,heads,hd", [(10, 16, 4, 128), (1 << 30, 1 << 16, 1024, 256), (1 << 30, 1 << 30, 1, 16), (1 << 30, 1 << 30, 16, 16), (1 << 30, 16, 1024, 256),
                                                 ((1 << 30) - 1, 0x7FFF0000, 1000, 240), (1, 0x7FFF0000, 1, 16)])
def test_bytes_of_a_cache(ask, pages, page, heads, hd):
    # accepted sizes go past 64 bits: no buffer holds those, and none may pass for holding them
    assert ask("bytes", 1, 1, heads, heads, hd, pages, page, 1, 1) == ["ok", str(min(pages * page * heads * hd * 2, 2 ** 64 - 1))]


def test_bytes_of_packed_rows(ask):
    assert ask("bytes", 1 << 22, 1, 1024, 1024, 256, 0, 0, 0, 0) == ["ok", str((1 << 22) * 1024 * 256 * 2)]


@pytest.mark.parametrize("tb,rows,n_seq", [(1, 1 << 22, 4096), (1, 1 << 22, 1025), (2, 1 << 22, 4096), (16, 64, 600), (128, 64, 600), (1, 1, 4096), (1, 5, 2), (4, 9, 1)])
def test_blocks_of_sequences_out_of_order(ask, tb, rows, n_seq):
    # every second sequence has all of the rows: 2^33 of them at most
    blocks = (n_seq + 1) // 2 * -(-rows // tb)
    assert ask("blocks", tb, rows, n_seq) == [str(min(blocks, rows + 1)), str(int(n_seq > 1))]


@pytest.mark.parametrize("past,q_len,most", [(-4, 10, 64), (-5, 16, 64), (-150, 200, 640), (-(1 << 22), (1 << 22) + 0, 16), (0, 300, 300), (1000, 5, 4096), (0x7FFF0000 - 200, 200, 0x7FFF0000)])
@pytest.mark.parametrize("window", [0, 1, 3, 200, 0x7FFEFFFF, 0x7FFF0000, 2 ** 31 - 5, 2 ** 31 - 1])
def test_windows_and_negative_positions(ask, past, q_len, most, window):
    for tb, log2_tile in ((16, 7), (128, 6)) if q_len < 1000 else ((128, 7),):
        assert ask("window", past, q_len, tb, log2_tile, window, most) == ["ok"]
