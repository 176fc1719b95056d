"""CPU-side checks of dense decode attention, the paged cache's forks and moves, and the rotation on several axes: refusals
and host bookkeeping (no kernel is launched here)."""
import ctypes
import os

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nsa_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from nsa_amd import build
        build.build()
    return _lib.load()


def test_dense_decode_argument_errors_do_not_launch(lib):
    """every call is refused before a launch (the pointers are not device memory)"""
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    names = ["q", "k", "v", "table", "max_pages", "num_pages", "lens", "out", "lse", "batch", "hq", "hkv", "dk", "dv", "cap",
             "window", "scale", "dtype", "ws", "ws_bytes", "stream"]
    good = dict(q=p, k=p, v=p, table=p, max_pages=64, num_pages=8, lens=p, out=p, lse=None, batch=2, hq=16, hkv=2, dk=64, dv=64,
                cap=0, window=0, scale=0.1, dtype=0, ws=p, ws_bytes=1 << 40, stream=None)

    def call(**kw):
        return lib.nsa_dense_decode_step(*[dict(good, **kw)[n] for n in names])

    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(lens=None), dict(out=None), dict(dtype=7), dict(batch=0),
                dict(hq=15), dict(hkv=0), dict(window=-1), dict(max_pages=0), dict(num_pages=0), dict(max_pages=1 << 30),
                dict(table=None, cap=0), dict(table=None, cap=100), dict(scale=float("inf")), dict(scale=float("nan")),
                dict(q=p + 2), dict(out=p + 8), dict(ws=None), dict(ws=p + 4), dict(ws_bytes=100),
                dict(batch=1 << 30, max_pages=1 << 20)):
        assert call(**bad) == -1, bad
        assert lib.nsa_last_error_string()
    for bad in (dict(dk=128), dict(dk=96, dv=96), dict(dk=192, dv=192)):
        assert call(**bad) == -2, bad
    assert lib.nsa_dense_decode_workspace_bytes(2, 16, 2, 64, 64, 128, 0, 0) == 0          # one unit per sequence
    assert lib.nsa_dense_decode_workspace_bytes(2, 16, 2, 64, 64, 4096, 64, 0) == 0        # a window of two pages at most
    assert lib.nsa_dense_decode_workspace_bytes(2, 16, 2, 64, 64, 4096, 0, 0) > 0
    assert lib.nsa_dense_decode_workspace_bytes(2, 15, 2, 64, 64, 4096, 0, 0) == -1
    assert lib.nsa_dense_decode_workspace_bytes(2, 16, 2, 64, 64, 100, 0, 0) == -1


def test_dense_decode_python_checks():
    from nsa_amd.decode import NSAPagedDecodeCache, dense_decode_step
    c = NSAPagedDecodeCache(2, 4, 128, 2, 64, 64, device="cpu")
    with pytest.raises(RuntimeError, match="GPU only"):
        dense_decode_step(torch.zeros(2, 4, 64, dtype=torch.bfloat16), c)
