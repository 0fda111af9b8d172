"""The paged key/value cache, as far as it can be checked without a GPU: the division of a batch's
work among workgroups (the kernels' own header, compiled as C++), and the refusals of the two entry
points, which check their arguments before they look for a device."""
import ctypes
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import cachepotato_amd as C
from tests.conftest import ROOT


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_shares_meet_every_unit_once(tmp_path):
    """4000 random batches (empty sequences, rows without keys, windows, broken offsets and lengths)
    against counting tile by tile: tests/paged_sched_main.cc"""
    exe = tmp_path / "sched"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wno-unused-function", "-ftrapv",
                    "-I" + os.path.join(ROOT, "cachepotato_amd", "csrc"),
                    os.path.join(ROOT, "tests", "paged_sched_main.cc"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


BUF = (ctypes.c_uint8 * 4096)()
P = (ctypes.addressof(BUF) + 255) // 256 * 256       # an aligned address; nothing is read from it


def cache(**kw):
    d = dict(KV=4, HD=128, type=C.T_F32, page=16, n_pages=8, page_stride=16 * 512, slot_stride=512,
             head_stride=128, k=P, v=P)
    d.update(kw)
    return C.PagedCache(*[d[f[0]] for f in C.PagedCache._fields_])


def batch(**kw):
    d = dict(S=2, T=3, max_new=2, max_pages=4, pages=P, q_off=P, len=P)
    d.update(kw)
    return C.PagedBatch(*[d[f[0]] for f in C.PagedBatch._fields_])


def rope(**kw):
    d = dict(table=P, max_pos=64, rot=128, pairs=C.ROPE_HALVES, q_norm=P, k_norm=P, eps=1e-6)
    d.update(kw)
    return C.PagedRope(*[d[f[0]] for f in C.PagedRope._fields_])


def refuse(rc, word):
    assert rc == -1
    assert word in C.last_error(), C.last_error()


def call_attn(c=None, b=None, type=C.T_F32, H=32, q=P, ldq=4096, scale=0.0, window=0, out=P, ldo=4096):
    return C.lib().cpg_paged_attn(ctypes.byref(c or cache()), ctypes.byref(b or batch()), type, H, q, ldq,
                                  scale, window, out, ldo, None, None)


def call_append(c=None, b=None, r=None, type=C.T_F32, H=32, q=P, ldq=5120, k=P, ldk=5120, v=P, ldv=5120,
                qo=P, ldqo=4096):
    return C.lib().cpg_paged_append(ctypes.byref(c or cache()), ctypes.byref(b or batch()),
                                    ctypes.byref(r or rope()), type, H, q, ldq, k, ldk, v, ldv, qo, ldqo, None)


@pytest.mark.parametrize("call", [call_attn, call_append])
@pytest.mark.parametrize("kw,word", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(HD=80), "HD=80"), (dict(HD=0), "HD=0"),
    (dict(KV=0), "KV=0"), (dict(page=0), "pages"), (dict(page=24), "pages"), (dict(page=2048), "pages"),
    (dict(n_pages=0), "pages"), (dict(page_stride=16 * 512 + 2), "stride"), (dict(slot_stride=64), "stride"),
    (dict(head_stride=-128), "stride"), (dict(head_stride=0), "stride"), (dict(page_stride=1 << 60), "stride"),
    (dict(k=P + 4), "aligned"), (dict(v=P + 8), "aligned"), (dict(type=5), "type"), (dict(type=-1), "type"),
])
def test_cache_refusals(call, kw, word):
    refuse(call(c=cache(**kw)), word)


@pytest.mark.parametrize("call", [call_attn, call_append])
@pytest.mark.parametrize("kw", [dict(S=-1), dict(T=-1), dict(max_pages=0), dict(pages=None), dict(q_off=None),
                                dict(len=None), dict(T=(1 << 30) + 1)])
def test_batch_refusals(call, kw):
    refuse(call(b=batch(**kw)), "bad batch")


@pytest.mark.parametrize("call", [call_attn, call_append])
@pytest.mark.parametrize("type_,ctype", [(C.T_F16, C.T_F32), (C.T_F16, C.T_BF16), (C.T_BF16, C.T_F16),
                                         (C.T_BF16, C.T_F32), (3, C.T_F32), (-1, C.T_F32)])
def test_type_refusals(call, type_, ctype):
    refuse(call(c=cache(type=ctype), type=type_), "type")


@pytest.mark.parametrize("kw,word", [
    (dict(H=0), "H=0"), (dict(H=30), "H=30"), (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"),
    (dict(scale=math.nan), "scale"), (dict(window=-1), "window"), (dict(q=None), "rows"), (dict(out=None), "rows"),
    (dict(ldq=4095), "rows"), (dict(ldq=4098), "rows"), (dict(ldo=2048), "rows"), (dict(q=P + 4), "rows"),
    (dict(out=P + 8), "rows"),
])
def test_attn_refusals(kw, word):
    refuse(call_attn(**kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(H=-1), "query heads"), (dict(q=None), "rows"), (dict(qo=None), "rows"), (dict(k=None), "rows"),
    (dict(v=P + 4), "rows"), (dict(ldk=511), "rows"), (dict(ldv=514), "rows"), (dict(ldqo=4000), "rows"),
    (dict(r=rope(rot=130)), "rotation"), (dict(r=rope(rot=8)), "rotation"), (dict(r=rope(rot=-16)), "rotation"),
    (dict(r=rope(rot=144)), "rotation"), (dict(r=rope(table=None)), "rotation"), (dict(r=rope(table=P + 8)), "rotation"),
    (dict(r=rope(max_pos=0)), "rotation"), (dict(r=rope(pairs=2)), "rotation"), (dict(r=rope(q_norm=P + 4)), "norm"),
    (dict(r=rope(k_norm=P + 4)), "norm"), (dict(r=rope(eps=-1.0)), "norm"), (dict(r=rope(eps=math.nan)), "norm"),
])
def test_append_refusals(kw, word):
    refuse(call_append(**kw), word)


def test_null_and_workspace_refusals():
    L = C.lib()
    refuse(L.cpg_paged_attn(None, ctypes.byref(batch()), 0, 32, P, 4096, 0.0, 0, P, 4096, None, None), "null")
    refuse(L.cpg_paged_attn(ctypes.byref(cache()), None, 0, 32, P, 4096, 0.0, 0, P, 4096, None, None), "null")
    refuse(call_attn(), "workspace")                 # everything else is right, the workspace is NULL
    refuse(call_append(), "workspace")
    refuse(call_append(H=0, q=None, qo=None), "workspace")
    refuse(L.cpg_paged_append(ctypes.byref(cache()), ctypes.byref(batch()), None, 0, 32, P, 5120, P, 5120, P,
                              5120, P, 4096, None), "workspace")
    if L.cpg_current_device() < 0:
        assert L.cpg_paged_ws_create(32, 4, 128) is None and "cpg_init" in C.last_error()
        assert L.cpg_paged_ws_status(None) == -7
    L.cpg_paged_ws_destroy(None)


def test_mode_refusals():
    for mode in (-1, 3):
        refuse(C.lib().cpg_paged_attn_mode(mode), "mode")
    for mode in (C.PAGED_FEW, C.PAGED_MANY, C.PAGED_AUTO):
        assert C.lib().cpg_paged_attn_mode(mode) == 0


def test_no_gpu_no_call():
    """right arguments without a context: -7, as from the library's other calls"""
    if C.lib().cpg_current_device() >= 0:
        pytest.skip("a context is there")
    x = np.zeros(4, np.float32)
    assert C.lib().cpg_rmsnorm(x.ctypes.data, x.ctypes.data, 1, 4, 1e-6, x.ctypes.data) == -7
