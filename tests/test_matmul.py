"""Products with packed weights: what the entry points refuse.  No device is touched -- every check precedes the launch."""
import ctypes

import numpy as np
import pytest

P = 1 << 20          # a non-null address that is never used


def mv(lib, ty=12, rows=4, cols=256, w=P, xt=0, x=P, xs=256, tokens=1, yt=0, y=P, ys=4):
    return lib.ggq_matvec_device(ty, rows, cols, w, xt, x, xs, tokens, yt, y, ys, None)


def gr(lib, ty=12, rows=4, cols=256, w=P, it=27, ids=P, n=2, yt=0, y=P, ys=256):
    return lib.ggq_get_rows_device(ty, rows, cols, w, it, ids, n, yt, y, ys, None)


def test_matvec_refusals():
    from gguf_amd import _lib as L
    lib = L.lib
    for bad in (0, 4, 16, 24, 31, 99):
        assert mv(lib, ty=bad) == L.UNSUPPORTED
    assert mv(lib, xt=12) == mv(lib, yt=28) == mv(lib, xt=26) == L.UNSUPPORTED
    assert mv(lib, cols=255) == mv(lib, ty=2, cols=33) == L.INDIVISIBLE
    assert mv(lib, tokens=2, ys=3) == L.INVALID                      # overlapping outputs
    assert mv(lib, w=None) == mv(lib, x=None) == mv(lib, y=None) == L.INVALID
    assert mv(lib, rows=1 << 31) == mv(lib, tokens=1 << 31, ys=1 << 12) == mv(lib, cols=1 << 31) == L.INVALID
    assert mv(lib, xs=1 << 40) == mv(lib, ys=1 << 40) == L.INVALID
    assert mv(lib, x=P + 2) == mv(lib, y=P + 2) == mv(lib, xt=1, x=P + 1) == mv(lib, yt=30, y=P + 1) == L.MISALIGNED
    assert mv(lib, rows=0, w=None) == mv(lib, tokens=0, x=None, y=None) == L.OK        # nothing to do


def test_get_rows_refusals():
    from gguf_amd import _lib as L
    lib = L.lib
    assert gr(lib, ty=0) == gr(lib, it=24) == gr(lib, it=0) == gr(lib, yt=12) == L.UNSUPPORTED
    assert gr(lib, cols=128) == L.INDIVISIBLE
    assert gr(lib, ys=255) == gr(lib, w=None) == gr(lib, ids=None) == gr(lib, y=None) == gr(lib, n=1 << 31) == L.INVALID
    assert gr(lib, ids=P + 4) == gr(lib, it=26, ids=P + 2) == gr(lib, y=P + 1) == L.MISALIGNED
    assert gr(lib, n=0, y=None) == gr(lib, cols=0, ys=0) == L.OK


def moe_desc(**kw):
    from gguf_amd import _lib as L
    f = dict(router_type=0, up_type=12, down_type=14, reserved=0, d_router=P, d_gate=P, d_up=P, d_down=P, hidden=512, ff=256, experts=8,
             top_k=2, gating=0, normalize=1, activation=0, scale=1.0)
    f.update(kw)
    return L.ggq_moe(*[f[n] for n, _ in L.ggq_moe._fields_])


def test_moe_refusals():
    from gguf_amd import _lib as L
    lib = L.lib
    size = ctypes.c_size_t()

    def ws(tokens=1, **kw):
        return lib.ggq_moe_workspace_bytes(ctypes.byref(moe_desc(**kw)), tokens, ctypes.byref(size))

    assert ws() == L.OK and 0 < size.value < 1 << 20
    one = size.value
    assert ws(64) == L.OK and size.value > one
    assert ws(65) == L.TOO_LARGE
    assert ws(0) == L.OK and size.value == 0
    assert ws(router_type=12) == ws(up_type=0) == ws(down_type=16) == L.UNSUPPORTED
    assert ws(hidden=511) == ws(ff=255) == L.INDIVISIBLE
    for bad in (dict(experts=0), dict(experts=513), dict(top_k=0), dict(top_k=9), dict(experts=64, top_k=33), dict(gating=2), dict(normalize=2),
                dict(activation=2), dict(reserved=1), dict(hidden=0), dict(ff=0), dict(hidden=1 << 31)):
        assert ws(**bad) == L.INVALID, bad
    assert lib.ggq_moe_workspace_bytes(None, 1, ctypes.byref(size)) == L.INVALID
    assert lib.ggq_moe_workspace_bytes(ctypes.byref(moe_desc()), 1, None) == L.INVALID

    def run(tokens=2, xt=0, x=P, xs=512, yt=0, y=P, ys=512, ids=P, weights=P, space=P, room=1 << 30, **kw):
        return lib.ggq_moe_device(ctypes.byref(moe_desc(**kw)), xt, x, xs, tokens, yt, y, ys, ids, weights, space, room, None)

    assert run(tokens=65) == L.TOO_LARGE
    assert run(xt=2) == run(yt=28) == L.UNSUPPORTED
    assert run(ys=511) == run(x=None) == run(y=None) == run(space=None) == run(d_router=None) == run(d_down=None) == L.INVALID
    assert run(room=one) == run(room=0) == L.INVALID
    assert run(space=P + 128) == run(x=P + 1) == run(y=P + 2) == run(ids=P + 2) == run(weights=P + 1) == run(d_router=P + 2) == L.MISALIGNED
    assert run(tokens=0, x=None, y=None, space=None, room=0) == L.OK


def test_python_refusals():
    """The Python layer's own checks, in front of the library's."""
    import torch
    import gguf_amd as g
    w = torch.zeros(4 * 144, dtype=torch.uint8)
    x, y = torch.zeros(2, 256), torch.zeros(2, 4)
    with pytest.raises(ValueError):
        g.matvec(12, y, w, x)                                    # host tensors
    with pytest.raises(g.LengthMismatch):
        g.matvec(12, y[:1], w, x)                                # as many outputs as tokens
    with pytest.raises(g.LengthMismatch):
        g.matvec(12, y, w[:-1], x)
    with pytest.raises(g.Indivisible):
        g.matvec(12, y, w, torch.zeros(2, 255))
    with pytest.raises(g.Unsupported):
        g.matvec(g.GGmlType.IQ2XXS, y, w, x)
    with pytest.raises(TypeError):
        g.Q4K.get_rows(torch.zeros(2, 256), w, torch.zeros(2, dtype=torch.int16))
    with pytest.raises(ValueError):
        g.matvec(12, y, w, torch.zeros(256, 2).t())              # rows of x not contiguous
    with pytest.raises(g.LengthMismatch):
        g.get_rows(12, torch.zeros(3, 256), w, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(g.Unsupported):
        g.MoeLayer(torch.zeros(2, 256), (12, w), (2, w), (12, w), hidden=256, ff=256, top_k=1)
    with pytest.raises(g.LengthMismatch):
        g.MoeLayer(torch.zeros(2, 256), (12, w), (12, w), (12, w), hidden=256, ff=256, top_k=1)
    with pytest.raises(ValueError):
        g.MoeLayer(torch.zeros(2, 256), (12, w), (12, w), (12, w), hidden=256, ff=256, top_k=1, gating="tanh")


def test_reference_bounds_notice_mistakes(oracle):
    """The tolerance of the GPU tests is tight enough: one wrong word of codes in a row of 4096
    elements is outside it."""
    import matmul_ref as ref
    from gguf_amd import synth
    rng = np.random.default_rng(3)
    for ty in (2, 12, 14, 8):
        cols = 4096
        p = synth.random_blocks(ty, 4 * cols // oracle.block_elems(ty), 5)
        x = rng.standard_normal((1, cols)).astype(np.float32).astype(np.float64)
        w, w0 = ref.decode(oracle, ty, p, 4, cols)
        y, b = ref.product(w, w0, x)
        q = p.copy()
        q[ref.CODES[ty][0] + 4:ref.CODES[ty][0] + 8] ^= 0x55
        w2, _ = ref.decode(oracle, ty, q, 4, cols)
        assert ref.outside((x @ w2.T)[:, :1], y[:, :1], b[:, :1], "f32") == 1
        assert ref.outside(y.astype(np.float32), y, b, "f32") == 0
