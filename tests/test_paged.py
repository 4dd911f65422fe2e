"""CPU: the paged pool's arithmetic (places in a page, parts of the key axis, pieces
of the rows and their blocks) in a program of its own, and the refusals of
ornith_hip_paged_* that need no device."""
import ctypes as C
import shutil
import subprocess

import pytest

import clibs
import ornithology_amd as oa


def test_arithmetic(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    out = tmp_path / "paged_check"
    r = subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-O1", str(clibs.ROOT / "tests" / "paged_check.cpp"),
                        "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_null_handles_are_refused():
    L = oa.lib()
    b, rows, n, f = oa._Batch(), oa._Rows(), C.c_uint64(7), C.c_int32(0)
    h = C.c_void_p(5)
    cfg = oa.PagedCfg(2, 64, 32, 1, oa.KV_Q8, 0, 1e4, 1, None)
    assert L.ornith_hip_paged_new(None, C.byref(cfg), C.byref(h)) == 2 and not h
    assert b"null" in L.ornith_hip_last_error()
    assert L.ornith_hip_paged_faults(None, C.byref(f)) == 2
    assert L.ornith_hip_paged_append(None, C.byref(b), 0, oa.F32, C.byref(rows), C.byref(rows), None, None, None, None, 0.0, None, 0, None) == 2
    assert L.ornith_hip_paged_read(None, C.byref(b), oa.F32, C.byref(rows), C.byref(rows), None) == 2
    assert L.ornith_hip_paged_attend(None, C.byref(b), 2, oa.F32, C.byref(rows), C.byref(rows), 1.0, None, 0, None) == 2
    assert L.ornith_hip_paged_attend_prefix(None, C.byref(b), 0, None, None, 2, oa.F32, C.byref(rows), C.byref(rows), 1.0, None, 0, None) == 2
    assert L.ornith_hip_paged_workspace(None, C.byref(b), 2, oa.F32, 0, C.byref(n)) == 2 and n.value == 0
    L.ornith_hip_paged_free(None)


def test_lists_on_the_host_are_refused():
    import torch
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="on the GPU"):
        oa.PagedBatch(i, i[:1], i[:1, None], n_rows=1)
