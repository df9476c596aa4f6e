"""The paged cache's host side against a CUDA runtime without a device
(fake_cudart.c, preloaded): what a call has waited for when it returns, what it
refuses, how much it launches."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
PRELUDE = """
import ctypes, importlib.util, sys
spec = importlib.util.spec_from_file_location("_lib", sys.argv[1])
_lib = importlib.util.module_from_spec(spec)
spec.loader.exec_module(_lib)
L, fake = _lib.lib(), ctypes.CDLL(sys.argv[2])
keep = ctypes.create_string_buffer(4112)
P = (ctypes.addressof(keep) + 15) // 16 * 16  # 16-byte aligned memory that no check reads

def create(n_pages=4, page=16, heads=8, kv_heads=2, hd=64, dtype=1, weight=None, position=None):
    h = ctypes.c_void_p()
    rc = L.mxmqa_paged_create(ctypes.byref(_lib.PagedConfig(n_pages, page, heads, kv_heads, hd, dtype, 0)),
                              ctypes.byref(_lib.PagedBuffers(P, P, None, None, weight, position)), ctypes.byref(h))
    assert rc == 0, _lib.last_error()
    return h
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("fake") / "libfake_cudart.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-w", "-fexceptions", os.path.join(HERE, "fake_cudart.c"), "-o", out, "-ldl"], check=True)
    return out


def run(fake, body):
    lib = os.path.join(os.path.dirname(HERE), "burn-extended_b200", "mxmoe", "_lib.py")
    r = subprocess.run([sys.executable, "-c", PRELUDE + body, lib, fake], env=dict(os.environ, LD_PRELOAD=fake),
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)


def test_create_has_zeroed_its_counters_when_it_returns(fake):
    """Streams that do not wait for the legacy one may use the cache at once."""
    run(fake, """
h = create(weight=P, position=P)
assert fake.fake_pending() == 0
""")


DECODE = """
def decode(h, rows=1, max_pages=4, window=0, dtype=1, stride=0):
    a = _lib.PagedDecodeArgs(P, 64, 64, P, 64, 64, None, dtype, dtype, rows, max_pages, P, stride, P, 0.125, window,
                             None, None, 0, 0, 0, 0, 0)
    return L.mxmqa_paged_decode(h, ctypes.byref(a), None)
"""


def test_decode_under_the_widest_tables(fake):
    """Tiles of a launch are numbered in 32 bits: a table one page too wide for one row is refused, and the widest that
    is not takes one launch for its row."""
    run(fake, DECODE + """
h = create(page=16, heads=64, kv_heads=64, hd=128)  # tiles of 16 keys
for window in (0, 16):
    n = fake.fake_launches()
    assert decode(h, max_pages=(1 << 25) - 1, window=window) == 5 and "max_pages" in _lib.last_error()
    assert fake.fake_launches() == n
    assert decode(h, max_pages=(1 << 25) - 2, window=window) == 0
    assert fake.fake_launches() - n <= 2  # the attention, the join of its parts
h = create(page=1, heads=1024, kv_heads=1024, hd=128)
assert decode(h, max_pages=33554431, window=16) == 5
""")


def test_cache_indexes_stay_a_stride_below_2_to_the_31(fake):
    """The kernels walk a row in strides of up to 1024 cache indexes, held in 32 bits."""
    run(fake, DECODE + """
h = create(page=1, heads=2, kv_heads=2, weight=P, position=P)

def append(max_pages):
    a = _lib.PagedAppendArgs(None, P, P, 0, 0, 128, 64, 128, 64, None, 0, 0, None, 0, 0, 1, 1, P, 0, 1, max_pages,
                             None, P, None, None, None, 0, 0, 0)
    return L.mxmqa_paged_append(h, ctypes.byref(a), None)

def evict(max_pages):
    a = _lib.PagedEvictArgs(P, 0, 1, max_pages, P, P, P + 4, 8, 0, 0)
    return L.mxmqa_paged_evict(h, ctypes.byref(a), None)

for f in (append, lambda n: decode(h, max_pages=n), evict):
    for n in (2 ** 31 - 1, 2 ** 31 - 1023):
        assert f(n) == 1 and "max_pages" in _lib.last_error()
    assert f(2 ** 31 - 1024) == 0, _lib.last_error()
""")


def test_rotary_refuses_more_pairs_than_it_can_number(fake):
    """The kernel for any stride numbers the pairs and passing columns of a token in 32 bits, 256 at a step."""
    run(fake, """
def turn(heads, hd, rot):
    a = _lib.RotaryArgs(P, heads * hd, hd, P, heads * hd, hd, 1, 1, heads, hd, P, P, P, rot, 8, 0, 0, 0)
    return L.mxmqa_rotary(ctypes.byref(a), None)

for heads, hd, rot in ((65535, 65536, 65536), (65535, 65536, 0), (32768, 65536, 2), (65535, 32768, 0)):
    n = fake.fake_launches()
    rc = turn(heads, hd, rot)
    if heads * (hd - rot // 2) > 2 ** 31 - 257:
        assert rc == 5 and "heads" in _lib.last_error() and fake.fake_launches() == n, (heads, hd, rot)
    else:
        assert rc == 0 and fake.fake_launches() == n + 1, (heads, hd, rot)
assert turn(32769, 65535, 0) == 5 and turn(32767, 65536, 0) == 0
""")


def test_evict_writes_lengths_over_others_last(fake):
    """new_lens may be lens or lie over seen: a launch of its own writes it after the one that reads those.  Askew over
    lens it would be read and written by that launch: refused."""
    run(fake, """
h = create(weight=P, position=P)

def evict(new, lens=P + 64, seen=P + 128, rows=8):
    a = _lib.PagedEvictArgs(P, 4, rows, 4, lens, seen, new, 8, 0, 0)
    n = fake.fake_launches()
    rc = L.mxmqa_paged_evict(h, ctypes.byref(a), None)
    return (rc, fake.fake_launches() - n)

for new in (P + 68, P + 36, P + 92):
    assert evict(new) == (1, 0) and "new_lens" in _lib.last_error(), new - P
for new in (P + 32, P + 96, P + 160):
    assert evict(new) == (0, 1), _lib.last_error()
for new in (P + 64, P + 100, P + 128, P + 132, P + 156):
    assert evict(new) == (0, 2), (new - P, _lib.last_error())
assert evict(P + 64, seen=P + 64) == (0, 2)
""")


def test_no_exception_leaves_an_entry_point(fake):
    """Where the host has no memory left, create and a kernel's first launch return an error."""
    run(fake, DECODE + """
h, dead = create(weight=P, position=P), ctypes.c_void_p()
fake.fake_no_memory(1)
rc = L.mxmqa_paged_create(ctypes.byref(_lib.PagedConfig(4, 16, 8, 2, 64, 1, 0)),
                          ctypes.byref(_lib.PagedBuffers(P, P, None, None, None, None)), ctypes.byref(dead))
assert rc == 4 and not dead.value
assert decode(h) == 3
a = _lib.PagedEvictArgs(P, 0, 1, 4, P, P, P + 64, 8, 0, 0)
assert L.mxmqa_paged_evict(h, ctypes.byref(a), None) == 3
fake.fake_no_memory(0)
assert decode(h) == 0 and L.mxmqa_paged_evict(h, ctypes.byref(a), None) == 0
""")
