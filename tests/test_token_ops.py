"""What the token operators refuse (no GPU needed), and the oracle that their device tests go by."""
import ctypes as C
import math

import pytest
import torch

from sleap_amd import _lib, ops
from tests import token_oracle as oracle


def refused(rc, text):
    assert rc < 0 and text.encode() in _lib.lib().sa_last_error(), (rc, _lib.lib().sa_last_error())


def i64(*v):
    return (C.c_int64 * len(v))(*v)


def test_rotary_entry_point_refuses():
    h = _lib.lib()

    def call(dtype=0, B=1, T=1, H=1, D=8, pos=0, axes=1, sections=(2,), theta=1e4, interleaved=0, x=256, xs=(8, 8, 8)):
        return h.sa_rotary_axes(x, dtype, B, T, H, D, i64(*xs), 256, pos, i64(0, 1, 1), axes, (C.c_int * len(sections))(*sections), theta, 0, interleaved, 0, 256, None)

    refused(call(dtype=3), "bad dtype")
    refused(call(B=-1), "bad shape")
    refused(call(D=7), "bad shape")
    refused(call(H=5000), "4096 heads")
    refused(call(pos=3), "position type")
    refused(call(axes=0), "axes")
    refused(call(axes=9, sections=(1,) * 9), "axes")
    refused(call(sections=(-1,)), "bad section")
    refused(call(sections=(0,)), "pairs in heads")
    refused(call(sections=(5,)), "pairs in heads")
    refused(call(D=600, sections=(129,)), "bad section")
    refused(call(theta=0.0), "theta")
    refused(call(theta=math.inf), "theta")
    refused(call(interleaved=1, x=260), "interleaved")
    refused(call(x=None), "null address")
    refused(call(interleaved=1, T=2, xs=(8, 9, 8)), "interleaved")
    assert call(B=0) == 0 and call(T=0) == 0


def test_attention_entry_points_refuse():
    h = _lib.lib()

    def call(dtype=1, B=1, Tq=4, Tk=8, H=2, K=2, D=32, strides=(64, 64, 32) * 3, scale=1.0, q=256, k=256, out=256, ws=0, backward=False, so=(64, 64, 32), mask=None, wsp=256):
        args = (q, k, 256, dtype, B, Tq, Tk, H, K, D, i64(*strides), None, mask, None, scale)
        if backward:
            return h.sa_cross_attention_backward(*args, out, None, 256, 256, i64(*so), 256, 256, 256, wsp, ws, None)
        return h.sa_cross_attention(*args, out, None, None, wsp, ws, None)

    for backward in (False, True):
        def no(text, **kw):
            refused(call(backward=backward, **kw), text)

        no("16-bit types", dtype=0)
        no("16-bit types", dtype=3)
        no("bad shape", B=-1)
        no("bad shape", H=3)
        no("bad shape", K=0)
        no("head size", D=20)
        no("head size", D=136)
        no("head size", D=0)
        no("scale", scale=0.0)
        no("scale", scale=-1.0)
        no("scale", scale=math.inf)
        no("scale", scale=math.nan)
        no("strides", strides=(64, 64, 32, 64, 60, 32, 64, 64, 32))
        no("strides", strides=(64, -64, 32, 64, 64, 32, 64, 64, 32))
        no("token strides", strides=(64, 64, 32, 64, 1 << 23, 32, 64, 64, 32))
        no("addresses", q=264)
        no("addresses", out=264)
        no("null address", q=None)
        no("null address", k=None)
        no("null address", out=None)
        no("strides", mask=256)
    assert call(B=0) == 0 and call(Tq=0) == 0
    refused(call(Tq=1, Tk=100000), "workspace")
    refused(call(Tq=1, Tk=100000, ws=1 << 40, wsp=None), "workspace")
    refused(call(backward=True, ws=1 << 40, wsp=None), "workspace")
    refused(call(backward=True), "workspace")
    refused(call(backward=True, so=(64, 60, 32)), "strides")
    refused(call(backward=True, so=(64, 1 << 24, 32), ws=1 << 40), "span")
    assert h.sa_cross_attention_workspace(1, 1, 100000, 2, 2, 32) > 0
    assert h.sa_cross_attention_workspace(0, 1, 1, 1, 1, 8) == 0 and h.sa_cross_attention_workspace(1, 4, 8, 3, 2, 8) == 0


def test_attention_gradients_are_asked_for_in_pairs():
    h = _lib.lib()

    def call(dq, dk, dv, ws=0):
        return h.sa_cross_attention_backward(256, 256, 256, 1, 1, 4, 8, 2, 2, 32, i64(*(64, 64, 32) * 3), None, None, None, 1.0, 256, None, 256, 256, i64(64, 64, 32), dq, dk, dv, 256, ws, None)

    refused(call(256, 256, None), "null address")
    refused(call(None, None, 256), "null address")
    assert call(None, None, None) == 0  # nothing asked for
    for asked in ((256, None, None), (None, 256, 256), (256, 256, 256)):
        refused(call(*asked), "workspace")


def test_adamw_entry_point_refuses():
    h = _lib.lib()
    row = i64(256, 256, 256, 256, 0, 10)

    def call(n=1, table=row, dtype=0, ams=0, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1):
        return h.sa_adamw_step(table, n, dtype, ams, lr, None, b1, b2, eps, wd, step, None, None)

    refused(call(n=-1), "list")
    refused(call(table=None), "list")
    refused(call(dtype=7), "dtype")
    refused(call(b1=1.0), "betas")
    refused(call(b2=-0.1), "betas")
    refused(call(eps=-1.0), "negative")
    refused(call(wd=-1.0), "negative")
    refused(call(lr=-1.0), "negative")
    refused(call(lr=math.nan), "negative")
    refused(call(step=0), "first step")
    refused(call(ams=1), "null address")
    refused(call(table=i64(0, 256, 256, 256, 0, 10)), "null address")
    refused(call(table=i64(256, 256, 256, 256, 0, -1)), "negative size")
    assert call(n=0, table=None) == 0 and call(table=i64(0, 0, 0, 0, 0, 0)) == 0


def test_sizes_beyond_64_bits_are_refused():
    """Counts and strides whose products do not fit 64 bits are not taken for small ones."""
    h = _lib.lib()
    refused(h.sa_adamw_step(i64(256, 256, 256, 256, 0, 2 ** 63 - 1), 1, 0, 0, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, 1, None, None), "2^36")
    near, far = (64, 64, 32), (64, 1 << 58, 32)  # 64 tokens of 2^58 elements: 2^64
    for q, dout in ((far, near), (near, far), ((64, 64, 1 << 62), near), (near, (64, 64, 1 << 62))):
        refused(h.sa_cross_attention_backward(256, 256, 256, 1, 1, 4, 8, 8, 2, 32, i64(*q, *near, *near), None, None, None, 1.0, 256, None, 256, 256, i64(*dout), 256, 256, 256, 256,
                                              1 << 40, None), "span")


def test_null_host_arrays_are_refused():
    h = _lib.lib()
    xs, ps, sections, strides = i64(8, 8, 8), i64(0, 1, 1), (C.c_int * 1)(2), i64(*(64, 64, 32) * 3)
    for a, b, c in ((None, ps, sections), (xs, None, sections), (xs, ps, None)):
        refused(h.sa_rotary_axes(256, 0, 1, 1, 1, 8, a, 256, 0, b, 1, c, 1e4, 0, 0, 0, 256, None), "null")
    refused(h.sa_cross_attention(256, 256, 256, 1, 1, 4, 8, 2, 2, 32, None, None, None, None, 1.0, 256, None, None, 256, 0, None), "null")
    for a, b in ((None, xs), (strides, None)):
        refused(h.sa_cross_attention_backward(256, 256, 256, 1, 1, 4, 8, 2, 2, 32, a, None, None, None, 1.0, 256, None, 256, 256, b, 256, 256, 256, 256, 1 << 40, None), "null")


def test_host_tensors_are_refused():
    x = torch.zeros((1, 2, 1, 8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.rotary_axes(x, torch.zeros((2, 1)), (2,))
    with pytest.raises(ValueError, match="CUDA"):
        ops.cross_attention(x.half(), x.half(), x.half())
    with pytest.raises(ValueError, match="GPU"):
        ops.adamw_step([x], [x], [x], [x], step=1, lr=1e-3)
    with pytest.raises(ValueError, match="lists"):
        ops.adamw_step([x], [x, x], [x], [x], step=1, lr=1e-3)
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.adamw_step([None], [x], [x], [x], step=1, lr=1e-3)
    from sleap_amd.nn.optim import AdamW

    with pytest.raises(ValueError, match="CUDA"):
        AdamW([torch.nn.Parameter(x)])
    with pytest.raises(ValueError, match="lr"):
        AdamW([], lr=-1.0)


def test_tangents_are_refused():
    """Forward-mode derivatives would be dropped silently; refused ahead of the device."""
    import torch.autograd.forward_ad as fw

    x, p = torch.zeros((1, 2, 1, 8)), torch.zeros((2, 1))
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))

        h = x.half()
        for call in (lambda: ops.rotary_axes(dual(x), p, (2,)), lambda: ops.rotary_axes(x, dual(p), (2,)), lambda: ops.cross_attention(dual(h), h, h),
                     lambda: ops.cross_attention(h, dual(h), h), lambda: ops.cross_attention(h, h, dual(h)), lambda: ops.adamw_step([dual(x)], [x], [x], [x], step=1, lr=1e-3),
                     lambda: ops.adamw_step([x], [x], [x], [x], step=1, lr=dual(torch.ones(1)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_oracle_gradients_against_differences():
    """The formulas of the attention oracle by central differences in 64 bits."""
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(s, generator=g).half() for s in ((2, 3, 4, 8), (2, 7, 2, 8), (2, 7, 2, 8), (2, 3, 4, 8)))
    lengths, mask = torch.tensor([7, 4]), torch.rand((2, 7), generator=g) < 0.7

    class Any64(dict):  # the oracle asks a tensor's type for its unit only
        def __missing__(self, _):
            return 0.0

    keep = oracle.UNIT, oracle.TINY
    oracle.UNIT, oracle.TINY = Any64(), Any64()
    try:
        x = [t.double() for t in (q, k, v)]
        want = oracle.attention(*x, lengths, mask, dout=do.double())
        for i, name in enumerate(("dq", "dk", "dv")):
            d, h = torch.randn(x[i].shape, generator=g, dtype=torch.float64), 1e-5
            loss = []
            for s in (1, -1):
                y = list(x)
                y[i] = y[i] + s * h * d
                loss.append((oracle.attention(*y, lengths, mask)["out"][0] * do.double()).sum())
            assert abs((loss[0] - loss[1]) / (2 * h) - (want[name][0] * d).sum()) < 1e-7
    finally:
        oracle.UNIT, oracle.TINY = keep
