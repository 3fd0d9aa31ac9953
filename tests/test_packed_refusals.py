"""Packed sequences and paged caches: every refusal of the C entry points and of
the Python calls, before any launch.  No GPU needed (made-up device addresses, so
only where no GPU is visible)."""
import ctypes
from pathlib import Path

import pytest
import torch

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -4
P = ctypes.c_void_p(1 << 20)

no_device = pytest.mark.skipif(Path("/dev/kfd").exists(),
                               reason="passes made-up device pointers; runs only where no GPU is visible")


def view(pkg, N=10, H=4, D=64, **kw):
    L = pkg.WaveLayout(1, H, N, D, 0, D, H * D)
    for k, v in kw.items():
        setattr(L, k, v)
    return L


def packed(pkg, bwd=False, **kw):
    a = dict(q=view(pkg), k=view(pkg, H=2), v=view(pkg, H=2), o=view(pkg), n=3, dtype=1, scale=0.125, p=P, cu=P,
             ws=P, ws_bytes=1 << 30)
    a.update(kw)
    lay = [ctypes.byref(x) if x is not None else None for x in (a["q"], a["k"], a["v"], a["o"])]
    if bwd:
        return pkg.lib().wha_packed_bwd(P, P, P, P, P, P, P, P, a["p"], a["cu"], a["n"], a["dtype"], a["ws"],
                                        a["ws_bytes"], *lay, a["scale"], None)
    return pkg.lib().wha_packed_fwd(P, P, P, a["p"], None, a["cu"], a["n"], a["dtype"], *lay, a["scale"], None)


@no_device
@pytest.mark.parametrize("bwd", [False, True])
def test_packed_refusals(pkg, bwd):
    def refused(code, word, **kw):
        assert packed(pkg, bwd, **kw) == code
        assert word in pkg.lib().wha_last_error()
    refused(INVALID, b"NULL", q=None)
    refused(INVALID, b"k_layout", k=view(pkg, H=2, stride_t=64))
    refused(INVALID, b"overlap", o=view(pkg, stride_t=128))
    refused(UNSUPPORTED, b"128", q=view(pkg, D=129))
    refused(INVALID, b"B = 1", v=view(pkg, H=2, N=11))
    refused(INVALID, b"B = 1", k=view(pkg, H=2, D=32))
    refused(INVALID, b"heads", k=view(pkg, H=3), v=view(pkg, H=3))
    refused(INVALID, b"heads", v=view(pkg, H=4))
    refused(INVALID, b"heads", o=view(pkg, H=2))
    refused(UNSUPPORTED, b"128 query heads", q=view(pkg, H=129), o=view(pkg, H=129), k=view(pkg, H=1), v=view(pkg, H=1))
    refused(INVALID, b"dtype", dtype=3)
    refused(INVALID, b"dtype", dtype=-1)
    for s in (0.0, -1.0, float("nan"), float("inf")):
        refused(INVALID, b"scale", scale=s)
    refused(INVALID, b"n_seq", n=0)
    refused(INVALID, b"cu_seqlens", cu=None)
    refused(INVALID, b"non-NULL", p=None)
    big = dict(q=view(pkg, N=1 << 27, H=16), o=view(pkg, N=1 << 27, H=16), k=view(pkg, N=1 << 27, H=1),
               v=view(pkg, N=1 << 27, H=1))
    refused(UNSUPPORTED, b"too large", **big)
    if bwd:
        refused(UNSUPPORTED, b"fp16", dtype=2)
        refused(WORKSPACE, b"workspace", ws_bytes=10 * 4 * 8 - 1)
        refused(INVALID, b"aligned", ws=ctypes.c_void_p((1 << 20) + 4))


@no_device
def test_rows_too_far_apart_are_refused(pkg):
    """A tile is loaded with 31-bit byte offsets from one base: 128 rows of k and v, in the backward
    64 rows of q and o with the heads of a group."""
    for size, dtype in ((2, 1), (4, 0)):
        far = (1 << 31) // (128 * size)
        for name in "kv":
            for bwd in (False, True):
                assert packed(pkg, bwd, dtype=dtype, **{name: view(pkg, H=2, stride_t=far)}) == UNSUPPORTED
                assert b"2 GiB" in pkg.lib().wha_last_error()
        for name in "qo":
            for lay in (view(pkg, stride_t=2 * far), view(pkg, stride_h=64 * far, stride_t=64)):
                assert packed(pkg, True, dtype=dtype, **{name: lay}) == UNSUPPORTED
                assert b"2 GiB" in pkg.lib().wha_last_error()


def test_workspace_sizes(pkg):
    L = pkg.lib()
    assert L.wha_packed_bwd_workspace_size(ctypes.byref(view(pkg, N=1000, H=3))) >= 1000 * 3 * 8
    assert L.wha_packed_bwd_workspace_size(None) == 0
    q = pkg.WaveLayout(2, 8, 1, 64, 512, 64, 512)
    size = L.wha_paged_decode_workspace_size
    assert size(ctypes.byref(q), 2, 16, 4) == 0  # one split
    splits = size(ctypes.byref(q), 2, 16, 4096) // (2 * 8 * 66 * 4)
    assert 2 <= splits <= 256
    assert size(None, 2, 16, 4) == 0 and size(ctypes.byref(q), 3, 16, 4) == 0 and size(ctypes.byref(q), 2, 16, 0) == 0


def rows(pkg, read=False, **kw):
    a = dict(k=view(pkg, H=2), v=view(pkg, H=2), dtype=1, cdtype=3, pages=8, P=16, ks=P, slots=P, kc=P, kp=P)
    a.update(kw)
    lay = [ctypes.byref(x) if x is not None else None for x in (a["k"], a["v"])]
    if read:
        return pkg.lib().wha_paged_kv_read(a["kc"], P, a["ks"], P, a["slots"], a["kp"], P, a["dtype"], a["cdtype"],
                                           a["pages"], a["P"], *lay, None)
    return pkg.lib().wha_paged_kv_write(a["kp"], P, a["slots"], a["kc"], P, a["ks"], P, a["dtype"], a["cdtype"],
                                        a["pages"], a["P"], *lay, None)


def decode(pkg, **kw):
    q = pkg.WaveLayout(2, 8, 1, 64, 512, 64, 512)
    a = dict(q=q, o=q, dtype=1, cdtype=3, pages=8, P=16, ks=P, kc=P, table=P, ts=4096, per=4096, HK=2, scale=0.1, ws=P,
             ws_bytes=1 << 30, lens=P, out=P)
    a.update(kw)
    return pkg.lib().wha_paged_decode(P, a["kc"], P, a["ks"], P, a["table"], a["ts"], a["per"], a["lens"], a["out"],
                                      None, a["ws"], a["ws_bytes"], a["dtype"], a["cdtype"], a["pages"], a["P"],
                                      a["HK"], ctypes.byref(a["q"]), ctypes.byref(a["o"]), a["scale"], None)


@no_device
@pytest.mark.parametrize("call", ["write", "read", "decode"])
def test_paged_refusals(pkg, call):
    def refused(code, word, **kw):
        rc = decode(pkg, **kw) if call == "decode" else rows(pkg, call == "read", **kw)
        assert rc == code, kw
        assert word in pkg.lib().wha_last_error()
    for p in (0, -16, 3, 24, 8192):
        refused(INVALID, b"power of two", P=p)
    refused(INVALID, b"n_pages", pages=0)
    refused(INVALID, b"n_pages", pages=(1 << 31) + 1)
    refused(INVALID, b"k_cache", kc=None)
    refused(INVALID, b"k_scale", ks=None)
    refused(INVALID, b"cache_dtype", cdtype=2)
    refused(INVALID, b"dtype", dtype=3)
    if call != "decode":
        refused(INVALID, b"slots", slots=None)
        refused(INVALID, b"non-NULL", kp=None)
        refused(INVALID, b"NULL", k=None)
        refused(INVALID, b"same rows", v=view(pkg, H=3))
        refused(INVALID, b"same rows", v=view(pkg, H=2, N=9))
        return
    refused(INVALID, b"lengths", lens=None)
    refused(INVALID, b"lengths", table=None)
    refused(INVALID, b"lengths", out=None)
    refused(INVALID, b"max_pages", per=0)
    refused(INVALID, b"table_stride", ts=4095)
    refused(INVALID, b"heads", HK=3)
    refused(INVALID, b"heads", HK=0)
    refused(INVALID, b"scale", scale=0.0)
    refused(INVALID, b"T = 1", q=pkg.WaveLayout(2, 8, 2, 64, 1024, 64, 512))
    refused(INVALID, b"T = 1", o=pkg.WaveLayout(2, 4, 1, 64, 512, 64, 512))
    refused(UNSUPPORTED, b"2^30", P=4096, per=1 << 19, ts=1 << 19)
    refused(WORKSPACE, b"workspace", ws_bytes=1000)


def test_python_refusals(pkg):
    """Checks of the Python calls that come before the device."""
    q, k = torch.zeros(4, 4, 64), torch.zeros(4, 2, 64)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        pkg.packed_fwd(q, k, k, cu)
    with pytest.raises(ValueError, match="3-D"):
        pkg.packed_fwd(q[0], k, k, cu)
    with pytest.raises(ValueError, match="device"):
        pkg.paged_kv_write(k, k, cu.long(), k[None], k[None])
    with pytest.raises(ValueError, match="device"):
        pkg.paged_decode_fwd(q, k[None], k[None], cu[None], cu)
    with pytest.raises(TypeError, match="int8"):
        pkg._dtype_code(torch.float64, "k_cache", cache=True)
    with pytest.raises(TypeError):
        pkg._dtype_code(torch.int8, "q")
