"""The attention entry points as the other host languages see them: the descriptors' layout, and the C++ mirror."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def fields(text, name, pattern):
    body = re.search(pattern % name, text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/|//[^\n]*", "", body, flags=re.S)
    return body


@pytest.mark.parametrize("name,cls", [("infr_cuda_rope_kv_desc", "_RopeKvDesc"), ("infr_cuda_attention_desc", "_AttentionDesc")])
def test_descriptors_have_the_same_fields_everywhere(tmp_path, name, cls):
    from moe4all_b200 import backend

    mirror = getattr(backend, cls)
    rust = open(os.path.join(ROOT, "crates", "infr-cuda", "src", "ffi.rs")).read()
    body = re.search(r"pub struct %s \{(.*?)\n\}" % name, rust, re.S).group(1)
    in_rust = re.findall(r"pub (\w+): ([^,]+),", body)
    kinds = {C.c_void_p: ("*const infr_cuda_buf", "*mut infr_cuda_buf"), C.c_uint32: ("u32",), C.c_float: ("f32",)}
    assert [n for n, _ in in_rust] == [n for n, _ in mirror._fields_]
    assert all(t in kinds[c] for (_, t), (_, c) in zip(in_rust, mirror._fields_))
    # the header's own offsets
    src = tmp_path / "offsets.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "infr_cuda.h"\nint main(void) {\n' +
                   "".join('printf("%%zu ", offsetof(%s, %s));\n' % (name, n) for n, _ in mirror._fields_) + 'printf("%%zu", sizeof(%s)); return 0; }\n' % name)
    exe = str(tmp_path / "offsets")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(mirror, n).offset for n, _ in mirror._fields_] + [C.sizeof(mirror)]


def build_host(tmp_path):
    from moe4all_b200 import build

    lib = build.build()
    libdir = os.path.dirname(lib)
    exe = str(tmp_path / "host_mirror_attention")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "cpp", "host_mirror_attention.cpp"), "-o", exe,
                    "-L", libdir, "-linfr_cuda", "-Wl,-rpath," + libdir], check=True)
    return exe


def test_cpp_mirror_compiles_and_links(tmp_path):
    assert os.path.exists(build_host(tmp_path))


@pytest.mark.gpu
def test_cpp_mirror_against_the_formula(tmp_path):
    exe = build_host(tmp_path)
    H, K, hd, cu = 4, 2, 64, [0, 13, 40]
    rows = cu[-1]
    rng = np.random.default_rng(3)
    q, k, v = (rng.normal(size=(rows, n, hd)).astype(np.float32) for n in (H, K, K))
    with open(tmp_path / "in.bin", "wb") as f:
        np.array([rows, 2, H, K, hd, *cu], np.int32).tofile(f)
        for a in (q, k, v):
            a.tofile(f)
    r = subprocess.run([exe, str(tmp_path / "in.bin"), str(tmp_path / "out.bin")], capture_output=True, text=True)
    assert r.returncode == 0 and "OK" in r.stdout, r.stderr + r.stdout
    got = np.fromfile(tmp_path / "out.bin", np.float32).reshape(rows, H, hd)
    pos = np.concatenate([np.arange(b - a) for a, b in zip(cu, cu[1:])])
    ang = pos[:, None, None] * 1e4 ** (-np.arange(0, hd, 2) / hd)

    def turn(x):
        a, b = x[..., : hd // 2].astype(np.float64), x[..., hd // 2 :].astype(np.float64)
        return np.concatenate([a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)], -1)

    qr, kr = turn(q), turn(k)
    # the cache holds f16: 2^-11 of a value, of a score of size S twice over in its weights, 2^-11 S of the result's size M
    S, M = np.linalg.norm(qr, axis=-1).max() * np.linalg.norm(kr, axis=-1).max() * 0.125, np.abs(v).max()
    for a, b in zip(cu, cu[1:]):
        for i in range(a, b):
            for h in range(H):
                w = kr[a : i + 1, h // 2] @ qr[i, h] * 0.125
                w = np.exp(w - w.max())
                want = (w / w.sum()) @ v[a : i + 1, h // 2].astype(np.float64)
                assert np.abs(got[i, h] - want).max() <= M * (2.0 ** -11 * (2 * S + 1) + 2.0 ** -14)
