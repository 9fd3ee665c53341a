"""What the acoustic-network operators refuse before they touch a device: the C entry points' checks of sizes, strides, types and
overlaps (none of the addresses below is ever read), and the wrappers' checks of tensors."""
import ctypes as C

import numpy as np
import pytest
import torch

import pocketsphinx_amd as P
from pocketsphinx_amd import capi

EINVAL, ENODEV = -2, -1
X, Y, W = C.c_void_p(1 << 20), C.c_void_p(1 << 30), C.c_void_p(1 << 40)


def _gn(dtype=0, x=X, xs=12, off=W, n_utt=1, rows=4, chan=12, groups=3, eps=1e-5, act=0, y=Y, ys=12, work=W, wb=1 << 30):
    return capi.lib().psgpu_group_norm_dev(dtype, x, xs, off, n_utt, rows, chan, groups, None, None, eps, act, y, ys, work, wb, None)


def _ns(dtype=0, z=X, zs=12, rows=4, n_sen=12, scale=1.0, base=1.0001, y=Y, ys=12):
    return capi.lib().psgpu_senone_scores_dev(dtype, z, zs, rows, n_sen, None, scale, base, y, ys, None, None)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(n_utt=-1), dict(n_utt=65536), dict(rows=-1), dict(chan=0), dict(groups=0), dict(groups=5),
                                dict(groups=-3), dict(xs=11), dict(ys=11), dict(act=4), dict(act=-1), dict(eps=-1e-9), dict(eps=float("nan")),
                                dict(eps=float("inf")), dict(x=None), dict(y=None), dict(off=None), dict(y=C.c_void_p((1 << 20) + 48)),
                                dict(y=X, ys=13)])
def test_group_norm_refuses(kw):
    assert _gn(**kw) == EINVAL and b"psgpu_group_norm_dev" in capi.lib().psgpu_last_error()


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(rows=-1), dict(n_sen=0), dict(zs=11), dict(ys=11), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(base=1.0), dict(base=float("inf")), dict(z=None), dict(y=None), dict(y=X), dict(y=C.c_void_p((1 << 20) + 40))])
def test_senone_scores_refuse(kw):
    assert _ns(**kw) == EINVAL and b"psgpu_senone_scores_dev" in capi.lib().psgpu_last_error()


def test_projection_refuses():
    L = capi.lib()
    h = C.c_void_p()
    w = np.zeros((4, 4), np.float32).ctypes.data_as(C.c_void_p)
    for a in ((3, 4, 4, w, None, 0, 0), (0, 0, 4, w, None, 0, 0), (0, 4, 0, w, None, 0, 0), (0, 4, (1 << 20) + 1, w, None, 0, 0), (0, 4, 4, None, None, 0, 0),
              (0, 4, 4, w, None, -1, 4), (0, 4, 4, w, None, 65537, 4), (0, 4, 4, w, None, 1, 0), (0, 4, 4, w, None, 1, 129)):
        assert L.psgpu_proj_create(C.byref(h), *a) == EINVAL and not h.value
    assert L.psgpu_proj_create(None, 0, 4, 4, w, None, 0, 0) == EINVAL
    assert L.psgpu_proj_set_adapter(None, 0, 1, w, w, 1.0) == EINVAL
    assert L.psgpu_proj_run_dev(None, X, 4, None, None, 0, 1, Y, 4, 0, None, 0, None) == EINVAL
    assert L.psgpu_proj_work_bytes(None, 10) == 0
    L.psgpu_proj_free(None)


def test_nothing_to_do_is_no_error():
    assert _gn(rows=0, x=None, y=None) == 0 and _gn(n_utt=0) == 0 and _ns(rows=0, z=None, y=None) == 0


def test_capability_and_version():
    L = capi.lib()
    L.psgpu_capabilities.restype = C.c_uint64
    assert L.psgpu_capabilities() >> 15 & 1 and L.psgpu_abi_version() == (1 << 16 | 7)


def test_tensors_on_the_host_are_refused():
    off = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError):
        P.group_norm(torch.zeros(4, 6), off, 2)
    with pytest.raises(ValueError):
        P.senone_scores(torch.zeros(4, 6))
    with pytest.raises(ValueError):
        P.senone_scores(np.zeros((4, 6), np.float32))


def test_no_cpu_fallback():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    assert _gn() == ENODEV and _ns() == ENODEV
    with pytest.raises(P.PsgpuError):
        P.AdaptedProjection(torch.zeros(4, 4))


def test_vectors_with_a_tangent_are_refused():
    import torch.autograd.forward_ad as forward
    from pocketsphinx_amd import net
    v = torch.ones(6)
    with forward.dual_level():
        dual = forward.make_dual(v, torch.ones(6))
        for no_grad in (False, True):               # (which leaves forward mode as it is)
            with torch.set_grad_enabled(not no_grad), pytest.raises(ValueError, match="tangent"):
                net._vector(dual, "weight", 6, torch.float32, v.device)
        assert net._vector(v, "weight", 6, torch.float32, v.device) is v and net._vector(dual.detach(), "weight", 6, torch.float32, v.device).shape == (6,)
    assert net._vector(v, "weight", 6, torch.float32, v.device) is v


@pytest.mark.parametrize("v", [1 << 32, (1 << 32) + 3, 1 << 31, -(1 << 31) - 1, 3.5, "3", float("nan")])
def test_whole_numbers_of_32_bits(v):
    """what C would cut to another number: a slot of 2^32 is not slot 0"""
    from pocketsphinx_amd import net
    with pytest.raises(ValueError):
        net._int32(v, "slot")
    for kw in (dict(max_adapters=v), dict(max_adapters=1, max_rank=v)):
        with pytest.raises(ValueError):
            P.AdaptedProjection(torch.zeros(4, 4), **kw)
    assert net._int32(np.int64(7), "slot") == 7 and net._int32(32.0, "slot") == 32 and net._int32(-(1 << 31), "slot") == -(1 << 31) and net._int32((1 << 31) - 1, "slot") == (1 << 31) - 1
