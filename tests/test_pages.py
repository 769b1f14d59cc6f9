"""The paged KV cache without a GPU: argument checks that need no device, and
rotary frequencies."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import ferry_amd as F

GEO = dict(n_layers=2, kv_heads=4, head_dim=128, block_tokens=16, dtype=F.BF16, n_pages=100,
           n_lanes=8, max_pages=16, device=0)


def desc(**kw):
    return F.PagesDesc(**{**GEO, **kw})


def last_error():
    return F.lib.ferry_last_error().decode()


@pytest.mark.parametrize("bad", [
    dict(dtype=4), dict(dtype=-1), dict(head_dim=64), dict(block_tokens=32), dict(n_layers=0),
    dict(kv_heads=0), dict(n_pages=0), dict(n_lanes=0), dict(max_pages=0), dict(n_lanes=65537),
    dict(max_pages=(1 << 20) + 1), dict(kv_heads=5000),
])
def test_geometry_is_checked(bad):
    n = C.c_uint64()
    assert F.lib.ferry_pages_work_bytes(C.byref(desc()), C.byref(n)) == 0 and n.value > 0
    assert F.lib.ferry_pages_work_bytes(C.byref(desc(**bad)), C.byref(n)) == -1
    assert F.lib.ferry_pages_compact(C.byref(desc(**bad)), None, None) == -1
    assert last_error()


def test_null_arguments():
    n = C.c_uint64()
    assert F.lib.ferry_pages_work_bytes(None, C.byref(n)) == -1
    assert F.lib.ferry_pages_work_bytes(C.byref(desc()), None) == -1
    assert F.lib.ferry_pages_append(C.byref(desc()), 0, None, None) == -1
    assert F.lib.ferry_pages_attend(C.byref(desc()), 0, None, None) == -1
    # null and pageable buffers are refused before anything is launched
    assert F.lib.ferry_pages_reserve(C.byref(desc()), None, None, 1, None) == -1
    host = np.zeros(4096, np.uint8)
    d = desc(pool=host.ctypes.data, table=host.ctypes.data, len=host.ctypes.data,
             error=host.ctypes.data, refs=host.ctypes.data, work=host.ctypes.data, work_bytes=4096)
    assert F.lib.ferry_pages_trim(C.byref(d), host.ctypes.data, None, 1, None) == -1
    assert "pool is not device-accessible" in last_error()


@pytest.mark.parametrize("bad,text", [
    (dict(x_dtype=3), "x_dtype"), (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=130), "rot_dim"),
    (dict(rot_dim=63), "rot_dim"), (dict(q=None, k=None, v=None), "neither"), (dict(v=None), "together"),
    (dict(q_out_dtype=3), "q_out_dtype"), (dict(q_heads=0), "q_heads"), (dict(n_tokens=-1), "n_tokens"),
])
def test_append_arguments(bad, text):
    a = dict(n_tokens=1, q_heads=8, x_dtype=F.BF16, q_out_dtype=F.BF16, rot_dim=128, q=16, k=16, v=16)
    assert F.lib.ferry_pages_append(C.byref(desc()), 0, C.byref(F.AppendArgs(**{**a, **bad})), None) == -1
    assert text in last_error()
    assert F.lib.ferry_pages_append(C.byref(desc()), 2, C.byref(F.AppendArgs(**a)), None) == -1
    assert "layer" in last_error()


@pytest.mark.parametrize("bad,text", [
    (dict(q_heads=6), "q_heads"), (dict(q_heads=0), "q_heads"), (dict(n_req=-1), "n_req"),
    (dict(n_groups=3), "n_groups"), (dict(n_tokens=5), "one token"),
])
def test_attend_arguments(bad, text):
    a = F.AttendArgs(**{**dict(n_req=2, n_tokens=2, q_heads=8), **bad})
    n = C.c_uint64()
    assert F.lib.ferry_pages_attend(C.byref(desc()), 0, C.byref(a), None) == -1
    assert text in last_error()
    assert F.lib.ferry_pages_attend_work_bytes(C.byref(desc()), C.byref(a), C.byref(n)) == -1


def test_host_tensors_are_refused():
    x = torch.zeros((1, 4, 2, 2, 16, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        F.Pages(x, torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_rope_frequencies():
    i = np.arange(0, 64, 2)
    plain = 10000.0 ** (-i / 64)
    assert np.allclose(F.rope_freqs(F.ROPE_PLAIN, 64), plain, rtol=1e-14)
    assert np.allclose(F.rope_freqs(F.ROPE_LINEAR, 64, stretch=4.0), plain / 4, rtol=1e-14)
    assert np.allclose(F.rope_freqs(F.ROPE_BASE, 64, stretch=4.0),
                       (10000.0 * 4.0 ** (64 / 62)) ** (-i / 64), rtol=1e-13)
    got = F.rope_freqs(F.ROPE_PARTS, 64, stretch=8.0, trained_ctx=4096, slow=1.0, fast=32.0)
    turns = 4096 * plain / (2 * math.pi)
    keep = np.clip((turns - 1.0) / 31.0, 0.0, 1.0)
    assert np.allclose(got, plain * keep + plain / 8 * (1 - keep), rtol=1e-14)
    assert got[0] == plain[0] and np.isclose(got[-1], plain[-1] / 8, rtol=1e-14)


@pytest.mark.parametrize("args", [
    (9, 64, 1e4, 1.0, 0.0, 1.0, 32.0), (F.ROPE_PLAIN, 3, 1e4, 1.0, 0.0, 1.0, 32.0),
    (F.ROPE_PLAIN, 64, 0.0, 1.0, 0.0, 1.0, 32.0), (F.ROPE_LINEAR, 64, 1e4, 0.0, 0.0, 1.0, 32.0),
    (F.ROPE_BASE, 2, 1e4, 2.0, 0.0, 1.0, 32.0), (F.ROPE_PARTS, 64, 1e4, 2.0, 0.0, 1.0, 32.0),
    (F.ROPE_PARTS, 64, 1e4, 2.0, 8192.0, 2.0, 2.0), (F.ROPE_LINEAR, 64, 1e4, math.nan, 0.0, 1.0, 32.0),
])
def test_rope_refusals(args):
    with pytest.raises(F.FerryError):
        F.rope_freqs(*args)


@pytest.mark.parametrize("args", [(math.inf, 1.0, 32.0), (8192.0, -math.inf, 32.0), (8192.0, 1.0, math.inf)])
def test_frequencies_in_parts_that_are_not_finite_are_refused(args):
    with pytest.raises(F.FerryError, match="all finite"):
        F.rope_freqs(F.ROPE_PARTS, 64, 1e4, 2.0, *args)
