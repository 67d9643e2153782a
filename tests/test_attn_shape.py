"""How an attention call is cut into work, and the sizes it refuses (attn_shape.h): every (row, key) pair of every sequence belongs to
exactly one CTA, every partial result has a place and a counter of its own, whatever the batch - also one whose arrays are wrong."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("attn") / "attn_shape_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "moe4all_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "attn_shape_check.cpp"), "-o", exe], check=True)
    return exe


def line(exe, tb, log2_tile, window, n_kv, ctas, cap, packed, rows, cu, kv, extra=1, join=0):
    args = [exe, "line", tb, log2_tile, window, n_kv, ctas, cap, int(packed), rows, extra, join, len(kv), *cu, *kv]
    r = subprocess.run([str(a) for a in args], capture_output=True, text=True)
    assert r.returncode == 0, (r.stdout, args)
    return [int(x) for x in r.stdout.split()]


def test_one_token(exe):
    # 513 keys: five tiles of 128 for each of four heads, a CTA each
    assert line(exe, 2, 7, 0, 4, 148, 1024, False, 1, [0, 1], [513]) == [20, 4, 4, 0]


def test_no_rows_no_keys(exe):
    assert line(exe, 2, 7, 0, 4, 148, 1024, False, 0, [0, 0, 0], [5, 0])[:2] == [0, 0]
    # rows without keys still have an item: their zeros are written
    assert line(exe, 2, 7, 0, 1, 148, 1024, False, 3, [0, 3], [0])[:2] == [2, 2]


def test_window_leaves_tiles_out(exe):
    # position 1000 with a window of 100: keys 901 .. 1000, tiles 7 (896 ..) and nothing before
    assert line(exe, 1, 7, 100, 1, 148, 2048, False, 1, [0, 1], [1001])[0] == 1
    assert line(exe, 1, 7, 106, 1, 148, 2048, False, 1, [0, 1], [1001])[0] == 2


@pytest.mark.parametrize("seed", range(40))
def test_batches(exe, seed):
    r = random.Random(seed)
    n = r.choice([1, 2, 5, 17])
    packed = r.random() < 0.3
    q = [r.choice([0, 1, 1, 3, r.randint(1, 200)]) for _ in range(n)]
    kv = list(q) if packed else [max(0, x + r.choice([-2, 0, 5, r.randint(0, 3000)])) for x in q]
    cu = [sum(q[:i]) for i in range(n + 1)]
    units, items, joined, bad = line(exe, r.choice([1, 2, 5, 16, 128]), r.choice([6, 7]), r.choice([0, 0, 1, 60, 1000]), r.choice([1, 3, 8]),
                                     r.choice([1, 7, 148]), 4096, packed, cu[-1] + r.choice([0, 3]), cu, kv, r.choice([0, 1, 2, 5]))
    assert bad == 0 and units >= items


@pytest.mark.parametrize("seed", range(12))
def test_fewer_ctas_where_joins_cost(exe, seed):
    r = random.Random(seed + 50)
    q, kv = [r.randint(1, 200), r.choice([0, 3])], [r.randint(200, 40000), 7]
    args = (r.choice([1, 5, 128]), 7, 0, r.choice([1, 3]), 148, 65536, False, sum(q), [0, q[0], sum(q)], kv, 3)
    assert line(exe, *args, join=r.choice([2, 4, 100]))[:2] == line(exe, *args, join=0)[:2]  # the same work, by fewer


@pytest.mark.parametrize("cu,kv", [([0, 5, 3, 9], [5, 5, 5]), ([-3, 2, 4, 8], [9, 9, 9]), ([0, 100, 200, 300], [400, 400, 400]), ([0, 2, 4, 6], [2, -7, 10 ** 6]),
                                   ([7, 7, 2000000000, -2000000000], [1, 2000000000, -2000000000])])
def test_wrong_arrays_are_forced_into_range(exe, cu, kv):
    assert line(exe, 2, 7, 0, 2, 148, 640, False, 10, cu, kv)[3] == 1


@pytest.mark.parametrize("sizes,want", [
    ((8, 1, 32, 4, 128, 10, 16, 4, 1), "ok"),
    ((8, 1, 32, 4, 128, 0, 0, 0, 0), "ok"),
    ((0, 1, 32, 4, 128, 0, 0, 0, 0), "ok"),
    ((8, 1, 128, 1, 256, 10, 48, 4, 1), "ok"),
    ((8, 0, 32, 4, 128, 0, 0, 0, 0), "invalid"),
    ((8, 1, 0, 4, 128, 0, 0, 0, 0), "invalid"),
    ((8, 1, 32, 0, 128, 0, 0, 0, 0), "invalid"),
    ((8, 1, 30, 4, 128, 0, 0, 0, 0), "invalid"),
    ((8, 1, 32, 4, 128, 10, 0, 4, 1), "invalid"),
    ((8, 1, 32, 4, 128, 10, 16, 4, 0), "invalid"),
    ((8, 1, 32, 4, 128, 10, 65536, 65536, 1), "invalid"),
    ((8, 1, 32, 4, 72, 0, 0, 0, 0), "unsupported"),
    ((8, 1, 32, 4, 272, 0, 0, 0, 0), "unsupported"),
    ((8, 1, 129, 1, 64, 0, 0, 0, 0), "unsupported"),
    ((8, 1, 32, 4, 128, 10, 24, 4, 1), "unsupported"),
    ((8, 20000, 32, 4, 128, 0, 0, 0, 0), "unsupported"),
    ((1 << 23, 1, 32, 4, 128, 0, 0, 0, 0), "unsupported"),
])
def test_sizes(exe, sizes, want):
    out = subprocess.run([exe, "sizes", *map(str, sizes)], capture_output=True, text=True, check=True).stdout
    assert out.split(":")[0].strip() == want, out


@pytest.mark.parametrize("seed", range(30))
def test_rows_that_share_bytes(exe, seed):
    r = random.Random(seed)
    for _ in range(8):
        stride, rows = r.randint(4, 40), r.randint(1, 5)
        wa, wb = r.randint(1, stride), r.randint(1, stride)
        a, b = 1000, 1000 + r.randint(-2 * stride, rows * stride + 3)
        used = lambda at, w: {at + i * stride + j for i in range(rows) for j in range(w)}
        got = subprocess.run([exe, "meet"] + [str(x) for x in (a, wa, stride, b, wb, stride, rows)], capture_output=True, text=True).stdout
        assert got == f"{int(bool(used(a, wa) & used(b, wb)))}\n", (a, wa, stride, b, wb, rows)
    # the parts of wide rows lie between each other; of two strides, spans count
    meet = lambda *x: subprocess.run([exe, "meet"] + [str(i) for i in x], capture_output=True, text=True).stdout == "1\n"
    assert not meet(0, 32, 48, 32, 8, 48, 100) and not meet(0, 32, 48, 40, 8, 48, 100) and meet(0, 32, 48, 28, 8, 48, 100)
    assert meet(0, 32, 48, 32, 8, 44, 100) and not meet(0, 32, 48, 99 * 48 + 32, 8, 44, 100)


@pytest.mark.parametrize("rows,g,pairs,want", [(8, 8, 10 ** 6, 1), (9, 9, 33, 0), (16, 16, 32, 1), (17, 1, 32, 0), (32, 16, 8, 1), (33, 1, 1, 0), (17, 17, 1, 0), (1, 1, 0, 1), (2 ** 40, 4, 1, 0)])
def test_which_kernel(exe, rows, g, pairs, want):
    r = subprocess.run([exe, "few", str(rows), str(g), str(pairs)], capture_output=True, text=True)
    assert r.stdout == f"{want}\n"
