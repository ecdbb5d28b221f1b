"""The table that says which kernels have had their shared-memory limit raised, without a GPU."""
import ctypes
import os
import subprocess

import pytest


@pytest.fixture
def seen(tmp_path):
    here = os.path.dirname(os.path.abspath(__file__))
    so = str(tmp_path / "libseen_probe.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", so, os.path.join(here, "csrc", "seen_probe.cpp")], check=True)
    lib = ctypes.CDLL(so)
    ull = ctypes.c_ulonglong
    lib.seen_has.argtypes = lib.seen_add.argtypes = [ull, ctypes.c_int, ctypes.c_int]
    lib.seen_add.restype = None
    return lib


def test_several_hundred_kernels_on_eight_devices_are_kept(seen):
    keys = [(0x7f0000001000 + 16 * i, dev) for i in range(380) for dev in range(8)]
    for i, (fn, dev) in enumerate(keys):
        assert not seen.seen_has(fn, dev, 1)
        seen.seen_add(fn, dev, 1000 + i)
    for i, (fn, dev) in enumerate(keys):
        assert seen.seen_has(fn, dev, 1000 + i) and seen.seen_has(fn, dev, 5) and not seen.seen_has(fn, dev, 1001 + i)
    seen.seen_add(*keys[3], 9000)
    seen.seen_add(*keys[3], 100)   # (a smaller limit is not a smaller one)
    assert seen.seen_has(*keys[3], 9000) and not seen.seen_has(*keys[3], 9001)


def test_more_than_it_holds(seen):
    """It starts anew: the newest are known, whatever is known was added, and every search ends."""
    for i in range(20000):
        fn = 0x1000 + 64 * i
        assert not seen.seen_has(fn, i % 3, 1)
        seen.seen_add(fn, i % 3, i + 1)
        assert seen.seen_has(fn, i % 3, i + 1) and not seen.seen_has(fn, i % 3, i + 2) and not seen.seen_has(fn, (i + 1) % 3, 1)
