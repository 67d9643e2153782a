"""The entry points around pages of 8 bits and a step's tokens as the other host languages see them: the descriptors' layout, and the C++ mirror."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name,cls", [("infr_cuda_kv_read_desc", "_KvReadDesc"), ("infr_cuda_embed_desc", "_EmbedDesc"), ("infr_cuda_sample_desc", "_SampleDesc")])
def test_descriptors_have_the_same_fields_everywhere(tmp_path, name, cls):
    from moe4all_b200 import backend

    mirror = getattr(backend, cls)
    rust = open(os.path.join(ROOT, "crates", "infr-cuda", "src", "ffi.rs")).read()
    in_rust = re.findall(r"pub (\w+): ([^,]+),", re.search(r"pub struct %s \{(.*?)\n\}" % name, rust, re.S).group(1))
    kinds = {C.c_void_p: ("*const infr_cuda_buf", "*mut infr_cuda_buf"), C.c_uint32: ("u32",), C.c_int32: ("i32",), C.c_float: ("f32",)}
    assert [n for n, _ in in_rust] == [n for n, _ in mirror._fields_]
    assert all(t in kinds[c] for (_, t), (_, c) in zip(in_rust, mirror._fields_))
    src = tmp_path / "offsets.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "infr_cuda.h"\nint main(void) {\n' +
                   "".join('printf("%%zu ", offsetof(%s, %s));\n' % (name, n) for n, _ in mirror._fields_) + 'printf("%%zu", sizeof(%s)); return 0; }\n' % name)
    exe = str(tmp_path / "offsets")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(mirror, n).offset for n, _ in mirror._fields_] + [C.sizeof(mirror)]


def test_every_entry_point_is_in_every_mirror():
    read = lambda *p: open(os.path.join(ROOT, *p)).read()
    header, rust, cpp, py = read("include", "infr_cuda.h"), read("crates", "infr-cuda", "src", "ffi.rs"), read("include", "infr_cuda.hpp"), read("moe4all_b200", "backend.py")
    for name in ("rope_kv_q8", "attention_q8", "kv_read", "embed", "sample"):
        args = [len(re.search(r"infr_cuda_%s\(([^;{]*)\)" % name, t, re.S).group(1).split(",")) for t in (header, rust)]
        assert args[0] == args[1] and "infr_cuda_%s(ctx_" % name in cpp and "infr_cuda_%s(self._ctx" % name in py
    for dt in ("F16", "BF16"):
        value = re.search(r"#define INFR_CUDA_DT_%s (\d+)" % dt, header).group(1)
        assert re.search(r"pub const DT_%s: i32 = %s;" % (dt, value), rust) and "%s = INFR_CUDA_DT_%s" % (dt, dt) in cpp and re.search(r"\b%s = %s\b" % (dt, value), py)


def build_host(tmp_path):
    from moe4all_b200 import build

    libdir = os.path.dirname(build.build())
    exe = str(tmp_path / "host_mirror_tokens")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "host_mirror_tokens.cpp"), "-o", exe,
                    "-L", libdir, "-linfr_cuda", "-Wl,-rpath," + libdir], check=True)
    return exe


def test_cpp_mirror_compiles_and_links(tmp_path):
    assert os.path.exists(build_host(tmp_path))


@pytest.mark.gpu
def test_cpp_mirror_against_the_formula(tmp_path):
    exe = build_host(tmp_path)
    rows, V, hd, page = 37, 50, 64, 16
    rng = np.random.default_rng(3)
    table = (rng.normal(size=(V, 3 * hd)).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)  # bf16 bits
    values = (table.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    ids, u = rng.integers(0, V, rows).astype(np.int32), rng.random(rows).astype(np.float32)
    with open(tmp_path / "in.bin", "wb") as f:
        for a in (np.array([rows, V, hd, page], np.int32), ids, table, u):
            a.tofile(f)
    r = subprocess.run([exe, str(tmp_path / "in.bin"), str(tmp_path / "out.bin")], capture_output=True, text=True)
    assert r.returncode == 0 and "OK" in r.stdout, r.stderr + r.stdout
    raw = open(tmp_path / "out.bin", "rb").read()
    flat, got_ids = np.frombuffer(raw[: 4 * rows * 6 * hd], np.float32), np.frombuffer(raw[4 * rows * 6 * hd :], np.int32)
    x, out, k, v = (a.reshape(rows, -1) for a in np.split(flat, np.cumsum([rows * 3 * hd, rows * hd, rows * hd])))
    assert (x == 2 * values[ids]).all()
    q, kx, vx = np.split(x.astype(np.float64), 3, 1)
    # half a step of 16 values' scale, which is at most 9/8 of what their largest needs of 127 steps
    for got, want in ((k, kx), (v, vx)):
        big = np.abs(want).reshape(rows, hd // 16, 16).max(-1).repeat(16, -1)
        assert (np.abs(got - want) <= big / 127 * 9 / 16).all()
    S, M = np.linalg.norm(q, axis=-1).max() * np.linalg.norm(k, axis=-1).max() * 0.125, np.abs(v).max()
    for i in range(rows):
        s = k[: i + 1].astype(np.float64) @ q[i] * 0.125
        w = np.exp(s - s.max())
        want = (w / w.sum()) @ v[: i + 1].astype(np.float64)
        assert np.abs(out[i] - want).max() <= M * (2.0 ** -18 * (2 * S + 1) + 2.0 ** -14)
    for i in range(rows):
        w = np.exp(out[i].astype(np.float64) - out[i].max())
        c = np.cumsum(w)
        assert got_ids[i] == int((c <= u[i] * c[-1]).sum())
