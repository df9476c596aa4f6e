"""The paged cache's C entry points without a device: argument checks come
before the first CUDA call, ctypes and Rust structs match the header; and the
64-bit oracle's own properties."""
import ctypes
import os
import re

import numpy as np
import pytest

import paged_oracle as po
from mxmoe import _lib
from test_rust_binding import header_struct, rust_struct

HEADER = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mxmoe.h")).read()
STRUCTS = {"mxmqa_paged_config": _lib.PagedConfig, "mxmqa_paged_buffers": _lib.PagedBuffers,
           "mxmqa_paged_append_args": _lib.PagedAppendArgs, "mxmqa_paged_decode_args": _lib.PagedDecodeArgs,
           "mxmqa_paged_evict_args": _lib.PagedEvictArgs, "mxmqa_rotary_config": _lib.RotaryTableConfig,
           "mxmqa_rotary_args": _lib.RotaryArgs}


def fields(name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    return [(t.replace(" ", ""), n) for t, n in re.findall(r"((?:const\s+)?\w+\s*\*?)\s*(\w+);", body)]


@pytest.mark.parametrize("name", STRUCTS)
def test_structs_match_the_header(name):
    ctype = {"uint32_t": ctypes.c_uint32, "int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float}
    rust = {"uint32_t": "u32", "int32_t": "i32", "int64_t": "i64", "float": "f32", "void": "c_void"}
    want = fields(name)
    assert [n for _, n in want] == [n for n, _ in STRUCTS[name]._fields_]
    for (t, n), (_, c) in zip(want, STRUCTS[name]._fields_):
        assert c is (ctypes.c_void_p if "*" in t else ctype[t]), n
    sys_rs = open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "rust", "burn-extended-cuda-sys", "src",
                               "lib.rs")).read()
    body = re.search(r"pub struct %s \{(.*?)\}" % name, sys_rs, re.S).group(1)
    got = re.findall(r"pub (\w+): ([^,]+),", body)
    assert [n for _, n in want] == [n for n, _ in got]
    for (t, n), (_, r) in zip(want, got):
        base = rust[t.replace("const", "").replace("*", "")]
        assert r == (base if "*" not in t else ("*const " if "const" in t else "*mut ") + base), n


def fake(n=1 << 12):
    """16-byte aligned memory that no check reads."""
    raw = ctypes.create_string_buffer(n + 16)
    return raw, (ctypes.addressof(raw) + 15) // 16 * 16


def refused(code, rc, word):
    assert rc == code and word in _lib.last_error(), (rc, _lib.last_error())


def test_create_refuses():
    L, h = _lib.lib(), ctypes.c_void_p()
    keep, p = fake()

    def create(cfg=(4, 16, 8, 2, 64, 1, 0), buf=(p, p, None, None, None, None)):
        return L.mxmqa_paged_create(ctypes.byref(_lib.PagedConfig(*cfg)), ctypes.byref(_lib.PagedBuffers(*buf)),
                                    ctypes.byref(h))

    refused(1, L.mxmqa_paged_create(None, None, ctypes.byref(h)), "null")
    for i in range(5):
        cfg = [4, 16, 8, 2, 64, 1, 0]
        cfg[i] = 0
        refused(1, create(cfg), "zero")
    refused(1, create((4, 16, 9, 2, 64, 1, 0)), "divisible")
    refused(1, create((4, 16, 8, 2, 64, 7, 0)), "dtype")
    refused(5, create((4, 16, 8, 2, 60, 1, 0)), "head_dim")
    refused(5, create((4, 16, 8, 2, 264, 1, 0)), "head_dim")
    refused(5, create((4, 16, 8, 2, 24, 2, 0)), "head_dim")
    refused(5, create((4, 65537, 8, 2, 64, 1, 0)), "page_size")
    refused(1, create(buf=(None, p, None, None, None, None)), "null k")
    refused(1, create(buf=(p + 8, p, None, None, None, None)), "16-byte")
    refused(1, create(buf=(p, p, p, None, None, None)), "8-bit")
    refused(1, create(buf=(p, p, None, None, p + 2, None)), "4-byte")
    assert not h.value
    assert L.mxmqa_paged_destroy(None) == 0
    refused(1, L.mxmqa_paged_status(None, None), "null")
    for f in (L.mxmqa_paged_append, L.mxmqa_paged_decode, L.mxmqa_paged_evict):
        refused(1, f(None, None, None), "null")


def test_rotary_refuses():
    L = _lib.lib()
    keep, p = fake()

    def table(rot=64, scaling=0, theta=1e4, s=1.0, first=4096.0, alpha=1.0, beta=32.0, at=0, n=4, cos=p):
        c = _lib.RotaryTableConfig(rot, scaling, theta, s, first, alpha, beta)
        return L.mxmqa_rotary_table(ctypes.byref(c), at, n, cos, p, 0, None)

    refused(1, table(rot=63), "rot_dim")
    refused(1, table(rot=0), "rot_dim")
    refused(1, table(rot=258), "rot_dim")
    refused(1, table(scaling=5), "scaling")
    refused(1, table(theta=0.0), "theta")
    refused(1, table(theta=float("inf")), "theta")
    refused(1, table(scaling=1, s=0.0), "scaling_factor")
    refused(1, table(scaling=3, s=8.0, first=0.0), "initial_context")
    refused(1, table(scaling=4, s=8.0, first=1.0), "out of range")
    refused(1, table(at=0xFFFFFFFF), "positions")
    refused(1, table(cos=None), "null")
    assert table(n=0) == 0

    def turn(x=p, out=p, dtype=0, tokens=2, heads=2, hd=64, pos=p, cos=p, rot=64, n=8):
        a = _lib.RotaryArgs(x, 128, 64, out, 128, 64, dtype, tokens, heads, hd, pos, cos, p, rot, n, 0, 0, 0)
        return L.mxmqa_rotary(ctypes.byref(a), None)

    refused(1, turn(dtype=2), "dtype")
    refused(1, turn(x=None), "null")
    refused(1, turn(pos=None), "null")
    refused(1, turn(x=p + 2), "misaligned")
    refused(1, turn(cos=p + 4), "16-byte")
    refused(1, turn(cos=None), "table")
    refused(1, turn(rot=66), "rot_dim")
    refused(1, turn(rot=33), "rot_dim")
    refused(1, turn(n=0), "empty")
    assert turn(tokens=0) == 0 and turn(heads=0) == 0


def test_oracle_turns_back_and_keeps_inner_products():
    rng = np.random.default_rng(0)
    x, y = rng.standard_normal((2, 6, 3, 32))
    inv, f = po.frequencies(20)
    for il in (False, True):
        pos = np.arange(6) * 11
        a = po.rotate(x, pos, inv, f, il)
        assert np.allclose(po.rotate(a, pos, inv, f, il, inverse=True), x)
        # <x at m, y at n> depends on m - n alone
        b = po.rotate(y, pos + 5, inv, f, il)
        c = po.rotate(x, pos + 100, inv, f, il), po.rotate(y, pos + 105, inv, f, il)
        assert np.allclose((a * b).sum(-1), (c[0] * c[1]).sum(-1))
        # the gradient against differences
        up = rng.standard_normal(x.shape)
        grad = po.rotate(up, pos, inv, f, il, inverse=True)
        e = np.zeros_like(x)
        e[2, 1, 7] = 1e-3
        num = ((po.rotate(x + e, pos, inv, f, il) - po.rotate(x - e, pos, inv, f, il)) * up).sum() / 2e-3
        assert abs(num - grad[2, 1, 7]) < 1e-9


def test_oracle_decode_is_plain_attention_and_evict_keeps_the_heaviest():
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((2, 5, 2, 4, 8))
    tab = np.array([[3, 0], [1, 4]])
    q = rng.standard_normal((2, 4, 8))
    w = np.zeros((5, 2, 4))
    out, lse = po.decode(q, k, v, tab, [7, 3], 0.3, weight=w)
    kk = np.concatenate([k[3, 1], k[0, 1]])[:7]
    vv = np.concatenate([v[3, 1], v[0, 1]])[:7]
    e = np.exp(kk @ q[0, 2] * 0.3)
    assert np.allclose(out[0, 2], e @ vv / e.sum()) and np.isclose(lse[0, 2], np.log(e.sum()))
    assert np.isclose(w.sum(), 2 * 4)  # one for every row and query head
    pos = np.zeros((5, 2, 4), np.int32)
    for r in range(2):
        for n in range(8):
            pos[tab[r, n // 4], :, n % 4] = n
    old = np.concatenate([w[3, 0], w[0, 0]])[:7].copy()
    assert po.evict(k, v, w, pos, tab, [7, 3], [7, 3], 4, 1, 1).tolist() == [4, 3]
    assert {0, 6} <= set(pos[3, 0].tolist())
    middle = sorted(range(1, 6), key=lambda i: -old[i])[:2]
    assert set(pos[3, 0].tolist()) == {0, 6, *middle}
