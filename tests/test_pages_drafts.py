"""Windows, trees of drafts and rotary axes over the paged KV cache without a GPU:
argument checks that need no device."""
import ctypes as C

import numpy as np
import pytest

import ferry_amd as F

from test_pages import desc, last_error

SMALL = dict(n_req=2, n_tokens=2)


@pytest.mark.parametrize("bad,text", [
    (dict(window=-1), "negative"), (dict(window=4, sinks=-1), "negative"), (dict(sinks=1), "go with a window"),
    (dict(tree_words=65, tree=64), "tree_words"), (dict(tree_words=-1), "tree_words"), (dict(tree_words=1), "together"),
    (dict(tree=64), "together"), (dict(tree_words=1, tree=12), "aligned"),
])
def test_what_rows_see(bad, text):
    a = F.AttendArgs(**SMALL, q_heads=8)
    assert F.lib.ferry_pages_attend_seen(C.byref(desc()), 0, C.byref(a), C.byref(F.SeenArgs(**bad)), None) == -1
    assert text in last_error()


def test_a_window_goes_with_no_groups():
    a = F.AttendArgs(**SMALL, q_heads=8, n_groups=1)
    s = F.SeenArgs(window=5)
    assert F.lib.ferry_pages_attend_seen(C.byref(desc()), 0, C.byref(a), C.byref(s), None) == -1
    assert "no groups" in last_error()
    # the causal call's own checks come with it
    a = F.AttendArgs(**SMALL, q_heads=6)
    assert F.lib.ferry_pages_attend_seen(C.byref(desc()), 0, C.byref(a), C.byref(s), None) == -1
    assert "q_heads" in last_error()
    assert F.lib.ferry_pages_attend_seen(C.byref(desc()), 0, None, C.byref(s), None) == -1


@pytest.mark.parametrize("bad,text", [(dict(n_axes=0), "n_axes"), (dict(n_axes=5, axis=16), "n_axes"),
                                      (dict(n_axes=2), "several axes")])
def test_axes(bad, text):
    a = F.AppendArgs(n_tokens=1, q_heads=8, x_dtype=F.BF16, q_out_dtype=F.BF16, rot_dim=128, q=16, k=16, v=16)
    assert F.lib.ferry_pages_append_axes(C.byref(desc()), 0, C.byref(a), C.byref(F.AxesArgs(**bad)), None) == -1
    assert text in last_error()


@pytest.mark.parametrize("bad,text", [
    (dict(n_req=-1), "negative"), (dict(n_tokens=-1), "negative"), (dict(n_tokens=5), "one token"),
    (dict(tree_words=0), "tree_words"), (dict(tree_words=65), "tree_words"),
])
def test_trees(bad, text):
    a = F.TreeArgs(**{**SMALL, "tree_words": 1, **bad})
    assert F.lib.ferry_pages_tree(C.byref(desc()), C.byref(a), None) == -1
    assert text in last_error()
    assert F.lib.ferry_pages_tree(C.byref(desc()), None, None) == -1


@pytest.mark.parametrize("bad,text", [
    (dict(n_tokens=-1), "negative"), (dict(n_tokens=5), "one token"), (dict(n_req=9, n_tokens=9), "n_lanes"),
    (dict(n_req=-1, n_tokens=-1), "negative"),
])
def test_accept(bad, text):
    a = F.AcceptArgs(**{**SMALL, **bad})
    assert F.lib.ferry_pages_accept(C.byref(desc()), C.byref(a), None) == -1
    assert text in last_error()
    assert F.lib.ferry_pages_accept(C.byref(desc()), None, None) == -1


def test_pageable_buffers_are_refused():
    host = np.zeros(4096, np.uint8)
    at = host.ctypes.data
    d = desc(pool=at, table=at, len=at, error=at, refs=at, work=at, work_bytes=4096)
    a = F.AcceptArgs(**SMALL, lanes=at, draft=at, chosen=at, path=at, kept=at, next=at)
    assert F.lib.ferry_pages_accept(C.byref(d), C.byref(a), None) == -1
    assert "pool is not device-accessible" in last_error()
    t = F.TreeArgs(**SMALL, tree_words=1, lanes=at, parent=at, tree=at)
    assert F.lib.ferry_pages_tree(C.byref(d), C.byref(t), None) == -1
    assert "pool is not device-accessible" in last_error()
