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


def test_rope_axes_argument_errors_do_not_launch(lib):
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    names = ["packed", "q", "k", "v", "gates", "inv", "pos", "axes", "pair_axis", "total", "ld", "q_off", "k_off", "v_off",
             "g_off", "hq", "hkv", "dk", "dv", "rope_off", "rope_dim", "interleaved", "pack", "dtype", "stream"]
    pairs = lambda *a: (ctypes.c_int32 * 128)(*a)                                       # noqa: E731
    good = dict(packed=p, q=p, k=p, v=p, gates=p, inv=p, pos=p, axes=3, pair_axis=pairs(0, 1, 2), total=4, ld=416, q_off=0,
                k_off=256, v_off=320, g_off=384, hq=4, hkv=1, dk=64, dv=64, rope_off=0, rope_dim=32, interleaved=0, pack=0,
                dtype=0, stream=None)

    def call(**kw):
        return lib.nsa_qkv_rope_axes(*[dict(good, **kw)[n] for n in names])

    for bad in (dict(packed=None), dict(q=None), dict(inv=None), dict(pos=None), dict(pair_axis=None), dict(dtype=3),
                dict(total=0), dict(dk=60), dict(ld=412), dict(k_off=252), dict(v_off=400), dict(g_off=405), dict(q_off=-8),
                dict(rope_dim=24), dict(rope_dim=0), dict(rope_off=40), dict(rope_off=4), dict(axes=0), dict(axes=5),
                dict(axes=2), dict(pair_axis=pairs(-1)), dict(packed=p + 4), dict(hq=1 << 26)):
        assert call(**bad) == -1, bad
        assert lib.nsa_last_error_string()
    assert call(dk=512, rope_dim=512, ld=8192, k_off=2048, v_off=4096, g_off=6000) == -2


def test_rope_pair_axes_and_the_layers_checks():
    from nsa_amd.layer import NSAAttentionLayer, rope_pair_axes
    assert rope_pair_axes((2, 3, 1)) == (0, 0, 1, 1, 1, 2)
    assert rope_pair_axes((2, 3, 1), "turns") == (0, 1, 2, 0, 1, 1)
    assert rope_pair_axes((4,)) == (0, 0, 0, 0) and rope_pair_axes((0, 2)) == (1, 1)
    for bad in (((), "blocks"), ((1,) * 5, "blocks"), ((-1, 2), "blocks"), ((1, 2), "rows")):
        with pytest.raises(ValueError):
            rope_pair_axes(*bad)
    for bad in (dict(rope_axes=(4, 6, 5)), dict(rope_axes=(4, 6, 6), rope_axes_spectrum="half"),
                dict(rope_axes=(4, 6, 6), rope_axes_layout="rows")):
        with pytest.raises(ValueError):
            NSAAttentionLayer(64, 2, 1, 64, rope_dim=32, **bad)
    with pytest.raises(ValueError):
        NSAAttentionLayer(64, 2, 1, 64, rope_dim=0, rope_axes=(0,))
    plain, own = (NSAAttentionLayer(64, 2, 1, 64, rope_dim=32, rope_axes=(4, 6, 6), rope_axes_spectrum=s)
                  for s in ("shared", "own"))
    assert torch.equal(plain.inv_freq, NSAAttentionLayer(64, 2, 1, 64, rope_dim=32).inv_freq)
    for lo, n in ((0, 4), (4, 6), (10, 6)):
        assert torch.allclose(own.inv_freq[lo:lo + n], 10000.0 ** -(torch.arange(n) / n), rtol=1e-6)
    cu = torch.tensor([0, 3, 3, 7], dtype=torch.int32)
    assert plain._axis_positions(None, 7, cu).tolist() == [[0, 1, 2, 0, 1, 2, 3]] * 3
    ids = torch.arange(42).view(3, 2, 7)
    assert torch.equal(plain._axis_positions(ids, 14, None), ids.reshape(3, 14))
    for bad in (torch.zeros(14), torch.zeros(2, 14), torch.zeros(3, 13)):
        with pytest.raises(ValueError, match="position_ids"):
            plain._axis_positions(bad, 14, None)


def test_rope_axes_python_checks(monkeypatch):
    """refusals of the tensor-level wrapper, on CPU tensors with the device check out of the way"""
    from nsa_amd import ops
    x = torch.zeros(3, 416, dtype=torch.bfloat16)
    args = (4, 1, 64, 64, (0, 256, 320, 384))
    good = dict(inv_freq=torch.zeros(16), positions=torch.zeros(3, 3, dtype=torch.int32), rope_off=0, rope_dim=32,
                pair_axis=[0, 1] * 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.qkv_rope_split(x, *args, **good)
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    for bad, err in ((dict(inv_freq=None), ValueError), (dict(positions=None), ValueError),
                     (dict(inv_freq=torch.zeros(8)), ValueError), (dict(pair_axis=[0] * 15), ValueError),
                     (dict(pair_axis=[3] * 16), ValueError), (dict(pair_axis=[-1] * 16), ValueError),
                     (dict(positions=torch.zeros(3, dtype=torch.int32)), ValueError),
                     (dict(positions=torch.zeros(3, 4, dtype=torch.int32)), ValueError),
                     (dict(positions=torch.zeros(5, 3, dtype=torch.int32)), ValueError),
                     (dict(positions=torch.zeros(3, 3)), TypeError)):
        with pytest.raises(err):
            ops.qkv_rope_split(x, *args, **dict(good, **bad))
    dq, dk, dv, dg = (torch.zeros(3, h, d, dtype=torch.bfloat16) for h, d in ((4, 64), (1, 64), (1, 64), (4, 3)))
    for bad in ((dq, dk[:2], dv, dg), (dq, dk, dv, dg.float()), (dq, dk[:, :, :32].contiguous(), dv, dg)):
        with pytest.raises(ValueError, match="agree"):
            ops.qkv_rope_pack(*bad, 416, args[4], **good)
