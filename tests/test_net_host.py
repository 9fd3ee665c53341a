"""The host side of the projection (psgpu_proj.hip) on a runtime of two devices that only writes its calls down (tests/hostsim/fake_hip.cc): a
load waits for the device of its weights, and no other load and no run comes in between its first wait and its last."""
import ctypes as C
import os
import shutil
import subprocess
import threading

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
pytestmark = pytest.mark.skipif(not (os.path.exists(HIPCC) or shutil.which("hipcc")), reason="hipcc not installed")


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    lib = str(tmp_path_factory.mktemp("fake") / "libproj_fake.so")
    flags = ["-O1", "-std=c++17", "-fPIC", "-I" + os.path.join(ROOT, "include")]
    hipcc = HIPCC if os.path.exists(HIPCC) else shutil.which("hipcc")
    rocm = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(hipcc))), "include")
    for cmd in ([hipcc, "--cuda-host-only", "--offload-arch=gfx950", "-fuse-cuid=none"] + flags + ["-c", os.path.join(ROOT, "pocketsphinx_amd", "csrc", "psgpu_proj.hip"), "-o", lib + ".proj.o"],
                ["g++", "-D__HIP_PLATFORM_AMD__", "-I" + rocm] + flags + ["-c", os.path.join(ROOT, "tests", "hostsim", "fake_hip.cc"), "-o", lib + ".fake.o"],
                ["g++", "-shared", "-pthread", "-o", lib, lib + ".proj.o", lib + ".fake.o"]):
        p = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
        assert p.returncode == 0, p.stderr[-3000:]
    L = C.CDLL(lib)
    vp, i32, i64 = C.c_void_p, C.c_int32, C.c_int64
    L.psgpu_proj_create.argtypes = [C.POINTER(vp), i32, i32, i32, vp, vp, i32, i32]
    L.psgpu_proj_set_adapter.argtypes = [vp, i32, i32, vp, vp, C.c_float]
    L.psgpu_proj_run_dev.argtypes = [vp, vp, i64, vp, vp, i32, i32, vp, i64, i32, vp, C.c_size_t, vp]
    L.psgpu_proj_free.argtypes = [vp]
    L.fake_place.argtypes = [vp, C.c_size_t, C.c_int]
    L.fake_log.argtypes = [vp, C.c_size_t]
    L.fake_log.restype = C.c_size_t
    return L


def _log(L):
    buf = C.create_string_buffer(1 << 22)
    n = L.fake_log(buf, 1 << 22)
    return [tuple(line.split()) for line in buf.raw[:n].decode().splitlines()]


def _matrix(*shape):
    return np.ones(shape, np.float32)


def _at(a):
    return a.ctypes.data_as(C.c_void_p)


def _object(L, weight, bias=None, adapters=2):
    h = C.c_void_p()
    assert L.psgpu_proj_create(C.byref(h), 0, 8, 12, _at(weight), None if bias is None else _at(bias), adapters, 4) == 0
    return h


@pytest.mark.parametrize("which", ["weight", "bias", "a", "b"])
def test_weights_on_another_device_are_waited_for(fake, which):
    m = dict(weight=_matrix(12, 8), bias=_matrix(12), a=_matrix(3, 8), b=_matrix(12, 3))
    fake.fake_place(_at(m[which]), m[which].nbytes, 1)
    _log(fake)
    h = _object(fake, m["weight"], m["bias"])
    assert fake.psgpu_proj_set_adapter(h, 0, 3, _at(m["a"]), _at(m["b"]), 1.0) == 0
    calls = [c[1:] for c in _log(fake)]
    assert ("copy", "1") in calls, "the other device's weights are copied"
    assert ("sync", "1") in calls[:calls.index(("copy", "1"))], "and were not waited for: %r" % (calls,)
    assert ("sync", "0") in calls[:calls.index(("copy", "1"))]
    d = C.c_int(-1)
    assert fake.hipGetDevice(C.byref(d)) == 0 and d.value == 0, "the current device is what it was"
    fake.psgpu_proj_free(h)
    fake.fake_place(_at(m[which]), 0, -1)


def test_loads_and_runs_of_several_threads_take_turns(fake):
    h = _object(fake, _matrix(12, 8))
    a, b = [_matrix(3, 8), _matrix(4, 8)], [_matrix(12, 3), _matrix(12, 4)]
    x, y = _matrix(40, 8), _matrix(40, 12)
    off, slot, work = np.array([0, 40], np.int32), np.zeros(1, np.int32), np.zeros(1 << 16, np.uint8)
    at_work = work.ctypes.data + 15 & ~15
    _log(fake)
    bad = []

    def load(k):
        fake.fake_name(1 + k)
        for _ in range(10):
            if fake.psgpu_proj_set_adapter(h, k, 3 + k, _at(a[k]), _at(b[k]), 1.0):
                bad.append(k)

    def run():
        fake.fake_name(3)
        for _ in range(20):
            if fake.psgpu_proj_run_dev(h, _at(x), 8, _at(off), _at(slot), 1, 40, _at(y), 12, 0, at_work, 1 << 15, None):
                bad.append("run")

    threads = [threading.Thread(target=load, args=(k,)) for k in range(2)] + [threading.Thread(target=run)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    calls = _log(fake)
    assert not bad
    assert sum(c[1] == "launch" for c in calls if c[0] == "3") == 40 and {c[0] for c in calls} == {"1", "2", "3"}
    at = 0
    while at < len(calls):          # a load: wait, launch (the slot is empty), two copies, two layouts, the slot's; wait.  A run: two launches
        who = calls[at][0]
        turn = ["launch"] * 2 if who == "3" else ["sync", "launch", "copy", "copy", "launch", "launch", "launch", "sync"]
        assert [c[:2] for c in calls[at:at + len(turn)]] == [(who, what) for what in turn], "call %d on: %r" % (at, calls[at:at + 12])
        at += len(turn)
    fake.psgpu_proj_free(h)
