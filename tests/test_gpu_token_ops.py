"""Rotary positions, cross attention and AdamW on the device against their 64-bit definitions (tests/token_oracle.py)."""
import math

import pytest
import torch

from tests import token_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=torch.float16, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


# --------------------------------------------------------------------------------------------------
# rotary positions
# --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,D,sections,ladder", [
    (1, 1, 1, 2, (1,), "axis"), (1, 52, 8, 64, (16, 16), "axis"), (2, 333, 3, 80, (8, 15, 13), "shared"), (3, 17, 5, 34, (4, 0, 3), "axis"),
    (2, 100, 2, 128, (24, 20, 20), "axis"), (1, 2050, 1, 50, (2, 3, 5), "shared"), (2, 65, 7, 256, (128,), "axis"), (1, 31, 4, 300, (1, 1, 1, 1), "axis")])
def test_rotary_matches_its_definition(dtype, interleaved, B, T, H, D, sections, ladder):
    from sleap_amd import ops

    g = rng(T * D)
    x = normal(g, B, T, H, D, dtype=dtype)
    for positions in (torch.randint(-50, 2_000_000, (T, len(sections)), generator=g, device=DEV, dtype=torch.int32),
                      torch.randint(0, 100_000_000, (B, T, len(sections)), generator=g, device=DEV),
                      torch.rand((B, T, len(sections)), generator=g, device=DEV) * 1024):
        y = ops.rotary_axes(x, positions, sections, ladder=ladder, interleaved=interleaved)
        assert y.dtype == dtype and y.is_contiguous()
        assert oracle.worst(y, oracle.rotary(x, positions, sections, ladder=ladder, interleaved=interleaved)) <= 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_takes_any_layout(dtype, interleaved):
    from sleap_amd import ops

    g = rng(3)
    B, T, H, D, sections = 2, 37, 4, 48, (8, 8)
    p = torch.rand((T, 2, 2), generator=g, device=DEV)[..., 1] * 300  # strided positions
    base = normal(g, B, H, T + 3, D + 9, dtype=dtype)
    for x in (base[..., :T, :D].transpose(1, 2), base[..., 3:, 9:].transpose(1, 2), base[..., 1:T + 1, 1:D + 1].transpose(1, 2),
              base[..., :T, :D].transpose(1, 2)[:, :, :1].expand(B, T, H, D), base[:1, :, :T, :D].transpose(1, 2).expand(B, T, H, D),
              normal(g, B, T, D, H, dtype=dtype).transpose(2, 3), normal(g, B * T * H * D + 1, dtype=dtype)[1:].view(B, T, H, D)):
        y = ops.rotary_axes(x, p, sections, theta=500.0, interleaved=interleaved)
        assert oracle.worst(y, oracle.rotary(x, p, sections, 500.0, interleaved=interleaved)) <= 1


def test_rotary_gradient_is_the_inverse_turn():
    from sleap_amd import ops

    g = rng(4)
    x = normal(g, 2, 45, 3, 40, dtype=torch.float32).requires_grad_(True)
    p = torch.randint(0, 5000, (2, 45, 3), generator=g, device=DEV)
    dy = normal(g, 2, 45, 3, 40, dtype=torch.float32)
    y = ops.rotary_axes(x, p, (5, 6, 4))
    (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    assert oracle.worst(dx, oracle.rotary(dy, p, (5, 6, 4), inverse=True)) <= 1
    back = ops.rotary_axes(y.detach(), p, (5, 6, 4), inverse=True)
    assert torch.allclose(back, x, atol=4e-6)  # two turns of 1e-6 (|a| + |b|)
    # differences: <dx, d> against (y(x + h d) - y(x - h d)) . dy / 2h in 64 bits; linear in x, so any h does
    d = normal(g, *x.shape, dtype=torch.float32)
    plus, minus = (oracle.rotary(x.detach() + s * d, p, (5, 6, 4))[0] for s in (1, -1))
    want = ((plus - minus) * dy.double()).sum() / 2
    assert abs((dx.double() * d.double()).sum() - want) <= 2e-6 * (dy.double().abs() * d.double().abs()).sum() * 2
    # a second gradient: d/d(dy) of <dx, d>
    dy2 = dy.clone().requires_grad_(True)
    (dx2,) = torch.autograd.grad(ops.rotary_axes(x, p, (5, 6, 4)), x, dy2, create_graph=True)
    (again,) = torch.autograd.grad((dx2 * d).sum(), dy2)
    assert oracle.worst(again, oracle.rotary(d, p, (5, 6, 4))) <= 1


def test_rotary_refusals():
    from sleap_amd import ops

    x, p = normal(rng(6), 2, 5, 2, 16, dtype=torch.float32), torch.zeros((5, 2), device=DEV)
    for bad, kind, text in ((dict(x=x[0]), ValueError, "x must be"), (dict(x=x[..., :15]), ValueError, "even"), (dict(x=x.double()), TypeError, "float32"),
                            (dict(positions=p.double()), TypeError, "positions"), (dict(positions=p[:4]), ValueError, "positions"),
                            (dict(positions=p[:, :1]), ValueError, "positions"), (dict(positions=p.expand(3, 5, 2)), ValueError, "positions"),
                            (dict(positions=p.clone().requires_grad_(True)), ValueError, "gradient"), (dict(sections=(4, 5)), ValueError, "sections"),
                            (dict(sections=(0, 0)), ValueError, "sections"), (dict(sections=()), ValueError, "sections"), (dict(sections=(-1, 2)), ValueError, "sections"),
                            (dict(sections=(1,) * 9), ValueError, "sections"), (dict(ladder="none"), ValueError, "ladder"), (dict(theta=0.0), ValueError, "theta"),
                            (dict(theta=math.nan), ValueError, "theta"), (dict(positions=p.cpu()), ValueError, "CUDA")):
        with pytest.raises(kind, match=text):
            ops.rotary_axes(**{**dict(x=x, positions=p, sections=(4, 4)), **bad})


def test_rotary_reads_negated_views():
    """The imaginary part of a conjugated tensor is a float view that torch holds with the other sign."""
    from sleap_amd import ops

    z = torch.randn((7, 2), generator=rng(43), device=DEV, dtype=torch.complex64) * 50
    p = z.conj().imag
    assert p.is_neg()
    x = normal(rng(44), 1, 7, 2, 16, dtype=torch.float32)
    assert oracle.worst(ops.rotary_axes(x, p, (4, 4)), oracle.rotary(x, p.resolve_neg(), (4, 4))) <= 1


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fw

    from sleap_amd import ops

    x, p = normal(rng(45), 1, 5, 2, 16, dtype=torch.float32), torch.zeros((5, 2), device=DEV)
    q, k, v, _, _, _ = make(rng(46), 1, 5, 9, 2, 2, 16, torch.float16)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.rotary_axes(dual(x), p, (4, 4)), lambda: ops.rotary_axes(x, dual(p), (4, 4)), lambda: ops.cross_attention(dual(q), k, v),
                     lambda: ops.cross_attention(q, dual(k), v), lambda: ops.cross_attention(q, k, dual(v))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        one = [torch.ones(3, device=DEV) for _ in range(4)]
        for j in range(4):
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.adamw_step(*[[dual(t) if i == j else t] for i, t in enumerate(one)], step=1, lr=1e-3)
        ops.rotary_axes(x, p, (4, 4))  # without a tangent: as ever


def test_rotary_of_positions_that_are_learned_elsewhere():
    from sleap_amd import ops

    x, p = normal(rng(48), 1, 5, 2, 16, dtype=torch.float32), torch.rand((5, 2), device=DEV)
    want = ops.rotary_axes(x, p, (4, 4))
    with torch.no_grad():
        assert torch.equal(ops.rotary_axes(x, p.requires_grad_(True), (4, 4)), want)


def test_rotary_of_more_workgroups_than_a_grid_row():
    """2^24 single tokens: more threads than one dimension of a launch has."""
    from sleap_amd import ops

    g, B = rng(54), (1 << 24) + 5
    x, p = normal(g, B, 1, 1, 4, dtype=torch.float16), torch.rand((B, 1, 1), generator=g, device=DEV) * 100
    assert oracle.worst(ops.rotary_axes(x, p, (2,)), oracle.rotary(x, p, (2,))) <= 1


def test_attention_refusals():
    from sleap_amd import ops

    q, k, v, _, _, _ = make(rng(7), 2, 5, 9, 4, 2, 16, torch.float16)
    lengths, mask = torch.ones(2, dtype=torch.int32, device=DEV), torch.ones((2, 9), dtype=torch.bool, device=DEV)
    for bad, kind, text in ((dict(q=q[0]), ValueError, "q \\(B"), (dict(k=k[:1]), ValueError, "q \\(B"), (dict(v=v[:, :8]), ValueError, "q \\(B"),
                            (dict(q=q.float()), TypeError, "float16"), (dict(q=q.bfloat16()), TypeError, "float16"),
                            (dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), ValueError, "head size"), (dict(q=q[:, :, :3]), ValueError, "share"),
                            (dict(k=k[:, :, :0], v=v[:, :, :0]), ValueError, "share"), (dict(scale=0.0), ValueError, "scale"), (dict(scale=-1.0), ValueError, "scale"),
                            (dict(scale=math.inf), ValueError, "scale"), (dict(key_lengths=lengths[:1]), ValueError, "key_lengths"),
                            (dict(key_lengths=lengths.float()), ValueError, "key_lengths"), (dict(key_mask=mask[:, :8]), ValueError, "key_mask"),
                            (dict(key_mask=mask.float()), ValueError, "key_mask"), (dict(key_mask=mask.cpu()), ValueError, "CUDA")):
        with pytest.raises(kind, match=text):
            ops.cross_attention(**{**dict(q=q, k=k, v=v), **bad})


@pytest.mark.parametrize("B,T", [(0, 5), (3, 0)])
def test_rotary_of_nothing(B, T):
    from sleap_amd import ops

    assert ops.rotary_axes(torch.empty((B, T, 2, 8), device=DEV), torch.empty((T, 1), device=DEV), (4,)).shape == (B, T, 2, 8)


def test_rotary_of_a_bad_position_stays_in_its_token():
    from sleap_amd import ops

    x = normal(rng(5), 1, 9, 2, 16, dtype=torch.float32)
    p = torch.arange(9, device=DEV, dtype=torch.float32)[:, None].clone()
    p[4] = float("nan")
    y = ops.rotary_axes(x, p, (4,))
    assert torch.isnan(y[:, 4, :, :8]).all() and torch.equal(y[:, 4, :, 8:], x[:, 4, :, 8:])
    assert torch.isfinite(y[:, [0, 1, 2, 3, 5, 6, 7, 8]]).all()


# --------------------------------------------------------------------------------------------------
# cross attention
# --------------------------------------------------------------------------------------------------
def make(g, B, Tq, Tk, H, K, D, dtype, ragged="none", scale=1.0):
    q, k, v, dout = (normal(g, B, n, h, D, dtype=dtype, scale=s) for n, h, s in ((Tq, H, scale), (Tk, K, 1.0), (Tk, K, 1.0), (Tq, H, 1.0)))
    lengths = mask = None
    if "lengths" in ragged:
        lengths = torch.randint(0, Tk + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
        lengths[:1] = Tk + 5  # counts as Tk
        if B > 1:
            lengths[1] = -3  # counts as 0
    if "mask" in ragged:
        mask = torch.rand((B, Tk), generator=g, device=DEV) < 0.6
        if B > 2:
            mask[2] = False
    hidden = ~oracle.visible(B, Tk, lengths, mask, DEV)[:, :, None, None]
    k.masked_fill_(hidden, float("nan"))
    v.masked_fill_(hidden, float("inf"))
    return q, k, v, dout, lengths, mask


def check(q, k, v, dout, lengths=None, mask=None, scale=None):
    from sleap_amd import ops

    want = oracle.attention(q, k, v, lengths, mask, scale, dout)
    out, lse = ops.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask, scale=scale, return_lse=True)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    far = {"out": oracle.worst(out, want["out"]), "lse": oracle.worst(lse, want["lse"])}
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    again = ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask, scale=scale)
    far["out, differentiated"] = oracle.worst(again.detach(), want["out"])  # (over few keys with two-term weights: other bits)
    grads = torch.autograd.grad(again, leaves, dout)
    for name, x in zip(("dq", "dk", "dv"), grads):
        assert x.dtype == q.dtype
        far[name] = oracle.worst(x, want[name])
    assert max(far.values()) <= 1, far
    return out, grads


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 64, 2, 2, 16), (1, 7, 63, 4, 1, 24), (2, 33, 65, 3, 3, 32), (3, 64, 129, 2, 1, 40), (1, 65, 200, 6, 2, 64),
          (2, 130, 97, 4, 4, 72), (1, 257, 300, 2, 2, 96), (2, 100, 130, 8, 2, 104), (1, 140, 333, 2, 1, 128), (3, 1, 1029, 8, 2, 128),
          (1, 5, 2500, 2, 2, 64), (1, 1500, 40, 1, 1, 56), (4, 31, 31, 5, 5, 120), (2, 1, 0, 2, 2, 32), (2, 0, 9, 2, 2, 32), (0, 4, 9, 2, 2, 32)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ragged", ["none", "lengths", "mask", "lengths+mask"])
@pytest.mark.parametrize("B,Tq,Tk,H,K,D", SHAPES)
def test_attention_matches_its_definition(dtype, ragged, B, Tq, Tk, H, K, D):
    check(*make(rng(B + Tq * Tk + D), B, Tq, Tk, H, K, D, dtype, ragged))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Tq,Tk,H,K,D", [(2, 1000, 1100, 4, 2, 64), (1, 300, 5000, 2, 2, 128), (1, 3000, 320, 4, 1, 80), (16, 1, 4096, 8, 1, 128)])
def test_attention_of_many_tiles(dtype, B, Tq, Tk, H, K, D):
    check(*make(rng(7), B, Tq, Tk, H, K, D, dtype, "lengths+mask"))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ragged", ["none", "lengths+mask"])
@pytest.mark.parametrize("B,Tq,Tk,H,K,D", [(2300, 30, 31, 8, 8, 40), (600, 60, 64, 8, 8, 64), (2, 1100, 1300, 8, 8, 64), (4, 1100, 1300, 8, 8, 48), (1, 1700, 1701, 4, 4, 96),
                                           (3, 900, 1001, 8, 4, 72), (1, 1500, 1501, 4, 4, 128), (2, 2500, 999, 4, 1, 104)])
def test_gradients_multiplied_once(dtype, ragged, B, Tq, Tk, H, K, D):
    """Just above 2^30 multiply-adds a product: the kernels of long training calls, in all their widths, with one, two and four waves."""
    assert B * H * Tq * Tk * -(-D // 32) * 32 > 2 ** 30
    check(*make(rng(B + Tq * Tk + D), B, Tq, Tk, H, K, D, dtype, ragged))



@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ragged", ["none", "lengths+mask"])
@pytest.mark.parametrize("B,Tq,Tk,H,K,D", [(13, 130, 8000, 20, 20, 64), (13, 300, 500, 20, 20, 64), (3, 1500, 2100, 24, 12, 128), (9, 1100, 2300, 8, 8, 24)])
def test_more_workgroups_than_places(dtype, ragged, B, Tq, Tk, H, K, D):
    """More than 512 workgroups of 128 rows, where runs of keys even out the last round and where they do not pay."""
    assert B * K * -(-Tq * (H // K) // 128) > 512
    check(*make(rng(B + Tq * Tk + D), B, Tq, Tk, H, K, D, dtype, ragged))



def test_layouts_that_span_too_far_are_copied():
    """Tokens of q, k, v and dout so far apart that the kernels' 32-bit offsets do not reach over a tile; and keys that they just reach over."""
    g = rng(41)
    for step in (1 << 24, (1 << 23) - 8):
        held = torch.empty((72, step), dtype=torch.bfloat16, device=DEV)
        held[:, :256] = normal(g, 72, 256, dtype=torch.bfloat16)
        q, k, v, dout = (held[:n, a:a + 64].view(1, n, 2, 32) for n, a in ((40, 0), (70, 64), (70, 128), (40, 192)))
        check(q, k, v, dout)



def test_gradients_of_keys_beyond_32_bit_offsets():
    """Keys 128 Ki elements apart: the last lie 4.3 GB behind the first. (The copies are contiguous, the order of sums is the same.)"""
    from sleap_amd import ops

    g, Tk, step = rng(42), 16500, 1 << 17
    held = torch.empty((Tk, step), dtype=torch.bfloat16, device=DEV)
    held[:, :64] = normal(g, Tk, 64, dtype=torch.bfloat16)
    far = [held[:, :32].view(1, Tk, 1, 32), held[:, 32:64].view(1, Tk, 1, 32)]
    q, dout = normal(g, 1, 3, 2, 32, dtype=torch.bfloat16), normal(g, 1, 3, 2, 32, dtype=torch.bfloat16)
    got = []
    for k, v in (far, [t.contiguous() for t in far]):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        got.append(torch.autograd.grad(ops.cross_attention(*leaves), leaves, dout))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ragged", ["none", "lengths+mask"])
@pytest.mark.parametrize("B,Tq,Tk,H,K,D", [(1, 52, 1024, 8, 8, 32), (3, 33, 129, 2, 1, 8), (3, 20, 192, 4, 4, 64), (2, 1, 193, 2, 2, 40), (1, 800, 1537, 8, 8, 64), (3, 410, 1500, 8, 8, 32),
                                           (16, 500, 320, 1, 1, 32), (16, 513, 320, 1, 1, 32), (8, 1000, 500, 1, 1, 48), (8, 1025, 500, 1, 1, 48)])
def test_attention_of_waves_along_the_keys(dtype, ragged, B, Tq, Tk, H, K, D):
    """Few rows on few keys, four waves a workgroup along the keys: waves whose run is short, empty or hidden, and the last sizes that are cut so."""
    check(*make(rng(B + Tq * Tk + D), B, Tq, Tk, H, K, D, dtype, ragged))


def test_waves_whose_keys_are_hidden():
    """Of four runs of 128 keys, each alone visible, and each alone hidden."""
    q, k, v, dout, _, _ = make(rng(40), 1, 40, 512, 2, 2, 32, torch.float16)
    for run in range(4):
        mask = torch.zeros((1, 512), dtype=torch.bool, device=DEV)
        mask[:, 128 * run:128 * run + 128] = True
        for seen in (mask, ~mask):
            hidden = ~seen[:, :, None, None]
            check(q, k.masked_fill(hidden, float("nan")), v.masked_fill(hidden, float("inf")), dout, None, seen)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.0, 8.0, 40.0])
def test_attention_of_flat_and_of_steep_scores(dtype, spread):
    """From uniform weights to a weight of one; the largest score comes first, last and in the middle of the keys."""
    g = rng(8)
    q, k, v, dout, _, _ = make(g, 1, 70, 700, 2, 2, 64, dtype, scale=spread)
    check(q, k, v, dout)
    at = torch.linspace(-1, 1, 700, device=DEV)[None, :, None, None]
    for slope in (at, -at, 1 - at.abs()):
        check(q, (k * 0.1 + slope).to(dtype), v, dout, scale=0.3)


def test_half_precision_gradients_of_far_sizes():
    """fp16 gradients of outputs scaled by 2^-14 and by 2^12, and of values that are large: ds leaves fp16's range both ways."""
    q, k, v, dout, lengths, mask = make(rng(9), 2, 90, 1200, 4, 2, 64, torch.float16, "lengths")
    for scale in (2.0 ** -10, 1.0, 2.0 ** 9):
        check(q, k, v, (dout * scale).to(torch.float16), lengths, mask)
    rows = torch.logspace(-4, 3, 90, device=DEV)[None, :, None, None]
    check(q, k, v, (dout * rows).to(torch.float16), lengths, mask)
    check(q, k, v, (dout * rows.flip(1)).to(torch.float16), lengths, mask)


def test_attention_takes_any_layout():
    g = rng(10)
    B, Tq, Tk, H, K, D = 2, 50, 90, 4, 2, 40
    dtype = torch.bfloat16
    packed = normal(g, B, Tk, 2, K, D, dtype=dtype)
    q = normal(g, B, H, Tq, D, dtype=dtype).transpose(1, 2)  # heads first
    dout = normal(g, B, 1, H, D, dtype=dtype).expand(B, Tq, H, D)
    check(q, packed[:, :, 0], packed[:, :, 1], dout)
    wide = normal(g, B, Tk, K, D + 3, dtype=dtype)
    check(q, wide[..., 3:], wide[..., :D], dout)                                # addresses and strides of odd values
    check(q, packed[:1, :, 0].expand(B, Tk, K, D), packed[:, :1, 1].expand(B, Tk, K, D), dout)  # one image for all, one value for all
    last = normal(g, B, Tk, D, K, dtype=dtype).transpose(2, 3)
    check(normal(g, B, Tq, D, H, dtype=dtype).transpose(2, 3), last, last, dout)
    mask = torch.rand((Tk, 2, B), generator=g, device=DEV) < 0.5
    check(q, packed[:, :, 0], packed[:, :, 1], dout, mask=mask[:, 0].T)          # a strided mask
    check(q, packed[:, :, 0], packed[:, :, 1], dout, mask=mask[:, 1, :1].T)      # one mask for all
    check(q, packed[:, :, 0], packed[:, :, 1], dout, lengths=torch.tensor([[90, 1], [17, 1]], device=DEV)[:, 0])  # int64, strided


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_of_empty_views(dtype):
    """No keys, and no queries, cut from a layout whose strides the kernels do not take."""
    g = rng(47)
    q, wide = normal(g, 2, 4, 3, 8, dtype=dtype), normal(g, 2, 5, 3, 9, dtype=dtype)
    none = wide[..., :8][:, :0]
    check(q, none, none, q)
    check(none, q, q, none)


def test_gradients_of_broadcast_inputs_are_summed():
    from sleap_amd import ops

    g = rng(11)
    q, k, v, dout, _, _ = make(g, 3, 20, 40, 2, 2, 32, torch.bfloat16)
    one = k[:1].clone().requires_grad_(True)
    (d,) = torch.autograd.grad(ops.cross_attention(q, one.expand(3, -1, -1, -1), v), one, dout)
    whole = k[:1].expand(3, -1, -1, -1).contiguous().requires_grad_(True)
    (e,) = torch.autograd.grad(ops.cross_attention(q, whole, v), whole, dout)
    assert torch.equal(d, e.sum(0, keepdim=True))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ragged", ["none", "lengths+mask"])
@pytest.mark.parametrize("B,Tq,Tk,H,K,D", [(2, 1, 64, 2, 2, 16), (3, 31, 700, 4, 2, 40), (1, 1100, 50, 2, 1, 64), (2, 190, 2300, 2, 2, 128), (1, 12, 9000, 1, 1, 72),
                                           (2, 0, 9, 2, 2, 32), (2, 9, 0, 2, 2, 32)])
def test_only_the_gradients_asked_for(dtype, ragged, B, Tq, Tk, H, K, D):
    """A frozen map (q alone), given queries (k, v), and each of the three alone: cut otherwise than all together, as right."""
    from sleap_amd import ops

    q, k, v, dout, lengths, mask = make(rng(B + Tq * Tk + D), B, Tq, Tk, H, K, D, dtype, ragged)
    want = oracle.attention(q, k, v, lengths, mask, None, dout)
    for asked in ("q", "k", "v", "kv", "qv"):
        inputs = {n: t.detach().requires_grad_(n in asked) for n, t in zip("qkv", (q, k, v))}
        out = ops.cross_attention(*inputs.values(), key_lengths=lengths, key_mask=mask)
        for n, x in zip(asked, torch.autograd.grad(out, [inputs[n] for n in asked], dout)):
            assert x.shape == inputs[n].shape and oracle.worst(x, want["d" + n]) <= 1, (asked, n)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("by", ["lengths", "mask", "lengths+mask"])
@pytest.mark.parametrize("n", [2, 3, 40])
def test_few_visible_keys_of_many(dtype, by, n):
    """Gradients over n visible keys of 5000 are as exact as over n keys alone: the arithmetic is the same but for the float32 sums of the
    runs (2^-24 beside 2^-11 at least), so their errors' norms differ by less than a fifth."""
    from sleap_amd import ops

    g = rng(38 + n)
    q, k, v, dout, _, _ = make(g, 2, 150, n, 2, 2, 32, dtype)
    want = oracle.attention(q, k, v, None, None, None, dout)
    many = [torch.full((2, 5000, 2, 32), float("nan"), device=DEV, dtype=dtype) for _ in range(2)]
    at = torch.arange(n, device=DEV) if by == "lengths" else torch.randperm(5000, generator=g, device=DEV)[:n].sort()[0]
    for x, y in zip(many, (k, v)):
        x[:, at] = y
    mask = torch.zeros((1, 5000), dtype=torch.bool, device=DEV)
    mask[:, at] = True
    args = dict(key_lengths=torch.full((2,), n if by == "lengths" else 5000, device=DEV) if "lengths" in by else None, key_mask=mask if "mask" in by else None)

    def errors(q, k, v, **args):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        grads = torch.autograd.grad(ops.cross_attention(*leaves, **args), leaves, dout)
        grads = [grads[0], *(x[:, at] if args else x for x in grads[1:])]
        return [(x.double() - want[name][0]).norm().item() for name, x in zip(("dq", "dk", "dv"), grads)]

    for e, alone in zip(errors(q, *many, **args), errors(q, k, v)):
        assert e <= 1.2 * alone


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Tq,Tk,n", [(2, 150, 20000, 2000), (1, 30, 3000, 700), (1, 5, 40000, 600)])
def test_visible_keys_that_lie_together(dtype, B, Tq, Tk, n):
    """As above, for keys that one run or wave has all of."""
    from sleap_amd import ops

    g = rng(51 + n)
    q, k, v, dout, _, _ = make(g, B, Tq, n, 2, 2, 32, dtype, scale=0.3)
    want = oracle.attention(q, k, v, None, None, None, dout)
    for start in (0, 64 * 11, Tk - n):
        many = [torch.full((B, Tk, 2, 32), float("nan"), device=DEV, dtype=dtype) for _ in range(2)]
        for x, y in zip(many, (k, v)):
            x[:, start:start + n] = y
        mask = torch.zeros((1, Tk), dtype=torch.bool, device=DEV)
        mask[:, start:start + n] = True

        def errors(k, v, mask=None):
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
            out = ops.cross_attention(*leaves, key_mask=mask)
            grads = torch.autograd.grad(out, leaves, dout)
            if mask is not None:
                grads = [grads[0], *(x[:, start:start + n] for x in grads[1:])]
            return [(x.double() - want[name][0]).norm().item() for name, x in zip(("out", "dq", "dk", "dv"), [out.detach(), *grads])]

        a, b = errors(*many, mask), errors(k, v)
        print(dtype, B, Tq, Tk, n, start, ["%.3f" % (x / y) for x, y in zip(a, b)], flush=True)
        assert all(x <= 1.2 * y for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ragged", ["none", "lengths+mask"])
@pytest.mark.parametrize("B,Tq,Tk,H,K,D", [(3, 1, 11, 2, 1, 48), (2, 18, 2, 1, 1, 72), (5, 2, 282, 8, 8, 16), (1, 300, 900, 4, 2, 128), (3, 400, 1500, 4, 2, 40), (4, 2000, 2000, 4, 4, 16)])
def test_gradients_as_exact_as_their_type(dtype, ragged, B, Tq, Tk, H, K, D):
    """Over up to 2048 keys, weights of the gradients multiplied in two terms (dq alone in the last of the sizes): what is left are terms of
    2^-16 (bf16) and 2^-22 (fp16) beside the gradients' own rounding of 2^-8 and 2^-11, a tenth of it in the norm at most, and the float32
    sums of dw and delta: a row that sees one key has dw = delta, dq = 0, and both sums are off by D 2^-24 of their terms."""
    from sleap_amd import ops

    q, k, v, dout, lengths, mask = make(rng(B + Tq * Tk + D), B, Tq, Tk, H, K, D, dtype, ragged, scale=1.5)
    want = oracle.attention(q, k, v, lengths, mask, None, dout)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask), leaves, dout)
    for name, x in zip(("dq", "dk", "dv"), grads):
        if name == "dq" or Tq < 2000:
            w = want[name][0]
            sums = {"dq": want["sums"][0], "dk": want["sums"][1], "dv": torch.zeros(1)}[name]
            assert (x.double() - w).norm() <= 1.1 * (w.to(dtype).double() - w).norm() + 1e-6 * w.norm() + sums.norm().item(), name


def test_gradients_against_differences():
    """The 64-bit loss along a direction, by central differences, against the kernels' gradients along it."""
    from sleap_amd import ops

    g = rng(12)
    q, k, v, dout, lengths, mask = make(g, 2, 40, 100, 4, 2, 48, torch.float16, "lengths+mask")
    k, v = (t.nan_to_num(0, 0, 0) for t in (k, v))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask), leaves, dout)
    want = oracle.attention(q, k, v, lengths, mask, dout=dout)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(leaves[i].shape, generator=g, device=DEV, dtype=torch.float64)
        h, loss = 1e-4, []
        for s in (1, -1):
            x = [t.detach().double() for t in (q, k, v)]
            x[i] = x[i] + s * h * d
            y = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
            seen = oracle.visible(2, 100, lengths, mask, DEV)
            for b in range(2):
                at = seen[b].nonzero()[:, 0]
                for n in range(4 if len(at) else 0):
                    y[b, :, n] = torch.softmax(x[0][b, :, n] @ x[1][b, at, n // 2].T / math.sqrt(48), -1) @ x[2][b, at, n // 2]
            loss.append((y * dout.double()).sum())
        slope = (loss[0] - loss[1]) / (2 * h)
        assert abs((grads[i].double() * d).sum() - slope) <= (want[name][1] * d.abs()).sum() + 1e-5 * abs(slope)


def test_what_a_visible_key_holds_is_seen():
    """A NaN value reaches its head's outputs and no other's; an infinite key its rows."""
    from sleap_amd import ops

    q, k, v, _, _, _ = make(rng(13), 2, 40, 100, 4, 2, 32, torch.bfloat16)
    v[1, 70, 1, 5] = float("nan")
    out = ops.cross_attention(q, k, v)
    bad = torch.isnan(out)
    assert bad[1, :, 2:, 5].all() and bad.sum() == 40 * 2
    k[0, 3, 0] = float("nan")
    out, lse = ops.cross_attention(q, k, v, return_lse=True)
    assert torch.isnan(out[0, :, :2]).all() and torch.isfinite(out[0, :, 2:]).all() and torch.isnan(lse[0, :2]).all()


def test_rows_without_a_visible_key():
    from sleap_amd import ops

    q, k, v, dout, _, _ = make(rng(14), 3, 17, 130, 2, 1, 64, torch.float16)
    lengths = torch.tensor([0, 130, 0], dtype=torch.int32, device=DEV)
    k[0], v[0], k[2], v[2] = (float("nan"),) * 4
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out, lse = ops.cross_attention(*leaves, key_lengths=lengths, return_lse=True)
    assert (out[[0, 2]] == 0).all() and (lse[[0, 2]] == -math.inf).all() and not lse.requires_grad
    dout[0] = float("inf")
    for x in torch.autograd.grad(out, leaves, dout):
        assert (x[[0, 2]] == 0).all() and torch.isfinite(x).all() and x[1].abs().sum() > 0


def test_the_same_call_gives_the_same_bits():
    from sleap_amd import ops

    for shape in ((1, 5, 9000, 2, 2, 64), (1, 9000, 70, 4, 1, 64)):  # runs of keys and of rows, joined
        q, k, v, dout, _, _ = make(rng(15), *shape, torch.bfloat16)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        first = None
        for _ in range(3):
            out = ops.cross_attention(*leaves)
            got = [out, *torch.autograd.grad(out, leaves, dout)]
            assert first is None or all(torch.equal(a, b) for a, b in zip(first, got))
            first = got


def test_keys_beyond_32_bit_offsets():
    """Keys 128 Ki elements apart: the last lie 4.3 GB behind the first."""
    from sleap_amd import ops

    g, Tk, step = rng(16), 16500, 1 << 17
    held = torch.empty((Tk, step), dtype=torch.bfloat16, device=DEV)
    held[:, :64] = normal(g, Tk, 64, dtype=torch.bfloat16)
    k = held[:, :32].view(1, Tk, 1, 32)
    v = held[:, 32:64].view(1, Tk, 1, 32)
    q = normal(g, 1, 3, 2, 32, dtype=torch.bfloat16)
    near = ops.cross_attention(q, k.contiguous(), v.contiguous())
    far = ops.cross_attention(q, k, v)
    assert torch.equal(near, far)


@pytest.mark.parametrize("B,Tq", [((1 << 26) + 9, 1), (1, (1 << 28) + 17)])
def test_attention_of_more_workgroups_than_a_grid_row(B, Tq):
    """2^26 images of one query, and 2^28 queries (row statistics have 16 threads each), on two keys of equal weight and small whole values:
    all results are exact. With the gradients of whichever side is as large."""
    from sleap_amd import ops

    def whole(*shape, step=1):
        return (torch.randint(-2, 3, shape, generator=rng(sum(shape)), device=DEV, dtype=torch.int8) * step).half()

    q, k, v, dout = torch.zeros((B, Tq, 1, 8), device=DEV, dtype=torch.float16), whole(B, 2, 1, 8), whole(B, 2, 1, 8, step=2), whole(B, Tq, 1, 8)
    leaves = [q.requires_grad_(True), k.requires_grad_(B > 1), v.requires_grad_(B > 1)]
    out = ops.cross_attention(*leaves, scale=1.0)
    grads = torch.autograd.grad(out, leaves if B > 1 else leaves[:1], dout)
    with torch.no_grad():
        for rows in torch.arange(max(B, Tq), device=DEV).split(1 << 24):
            b, t = (slice(int(rows[0]), int(rows[-1]) + 1), slice(None)) if B > 1 else (slice(None), slice(int(rows[0]), int(rows[-1]) + 1))
            kk, vv, do = k[b].float(), v[b].float(), dout[b, t].float()
            mean = vv.mean(1, keepdim=True)
            assert torch.equal(out[b, t].float(), mean.expand(do.shape))
            ds = 0.5 * (do * (vv[:, :1] - mean)).sum(-1, keepdim=True)  # of the first key; the second has the opposite
            assert torch.equal(grads[0][b, t].float(), ds * (kk[:, :1] - kk[:, 1:]))
            if B > 1:
                assert (grads[1][b] == 0).all() and torch.equal(grads[2][b].float(), (0.5 * do).expand(vv.shape))


def test_attention_on_another_stream():
    from sleap_amd import ops

    q, k, v, dout, lengths, mask = make(rng(17), 2, 30, 700, 4, 2, 64, torch.float16, "lengths+mask")
    want = oracle.attention(q, k, v, lengths, mask, dout=dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        out = ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask)
        got = [out, *torch.autograd.grad(out, leaves, dout)]
    torch.cuda.current_stream().wait_stream(side)
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        assert oracle.worst(x.detach(), want[name]) <= 1


def test_captured_calls_follow_their_inputs():
    """Forward and backward in a graph each, replayed on new inputs with eager work between; each graph has its own scratch."""
    from sleap_amd import ops

    graphs = []
    for seed, shape in ((18, (2, 24, 1300, 4, 2, 64)), (19, (1, 150, 2600, 2, 2, 128))):
        q, k, v, dout, _, _ = make(rng(seed), *shape, torch.bfloat16)
        p = torch.randint(0, 1000, (shape[1], 2), generator=rng(seed), device=DEV)

        def step(q=q, k=k, v=v, dout=dout, p=p):
            leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
            out = ops.cross_attention(ops.rotary_axes(leaves[0], p, (16, 16)), leaves[1], leaves[2])
            return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held, step, (q, k, v, dout)))
    for turn in range(3):
        for graph, held, step, inputs in graphs:
            for t in inputs:
                t.copy_(torch.randn(t.shape, generator=rng(100 + turn), device=DEV).to(t.dtype))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, held, step, _ in graphs:
            for a, b in zip(held, step()):
                assert torch.equal(a, b)


def test_second_gradients_are_refused():
    from sleap_amd import ops

    q, k, v, dout, _, _ = make(rng(30), 1, 4, 6, 1, 1, 16, torch.float16)
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(ops.cross_attention(q, k, v), q, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="first gradients only"):
        dq.sum().backward()


def test_a_changed_input_is_noticed():
    from sleap_amd import ops

    q, k, v, dout, lengths, _ = make(rng(31), 2, 4, 6, 1, 1, 16, torch.float16, "lengths")
    for t in (k, lengths):
        leaf = q.clone().requires_grad_(True)
        out = ops.cross_attention(leaf, k, v, key_lengths=lengths)
        t.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            out.backward(dout)


def test_a_capture_beside_a_living_graph_of_its_leaves_is_refused():
    from sleap_amd import ops

    q, k, v, dout, _, _ = make(rng(32), 1, 4, 6, 1, 1, 16, torch.float16)
    q.requires_grad_(True)
    x = normal(rng(33), 1, 4, 1, 16, dtype=torch.float32).requires_grad_(True)
    p = torch.zeros((4, 1), device=DEV)
    eager = [ops.cross_attention(q, k, v), ops.rotary_axes(x, p, (4,))]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device=DEV)
        with pytest.raises(RuntimeError, match="holds the same leaf"):
            ops.cross_attention(q, k, v)
        with pytest.raises(RuntimeError, match="holds the same leaf"):
            ops.rotary_axes(x, p, (4,))
        held = ops.cross_attention(q.detach(), k, v)  # without a gradient: nothing to refuse
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, ops.cross_attention(q.detach(), k, v))
    eager[0].backward(dout)  # the eager graphs are whole
    eager[1].sum().backward()
    assert q.grad is not None and x.grad is not None


def test_a_capture_on_top_of_a_living_graph_is_refused():
    """As above where the held leaf, or a node from outside of the capture, is not an input itself but what an input hangs on."""
    from sleap_amd import ops

    q, k, v, dout, _, _ = make(rng(34), 1, 4, 6, 1, 1, 16, torch.float16)
    q.requires_grad_(True)
    twice = q * 2
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device=DEV)
        for call in (lambda: ops.cross_attention(twice, k, v), lambda: ops.cross_attention(q * 3, k, v), lambda: ops.cross_attention(k, (q * 3)[:, :1].expand(1, 6, 1, 16), v),
                     lambda: ops.rotary_axes(twice, torch.zeros((4, 1), device=DEV), (4,))):
            with pytest.raises(RuntimeError, match="holds the same leaf"):
                call()
    twice.backward(dout)  # the eager graph is whole
    assert torch.equal(q.grad, dout * 2)
    del twice
    leaf = q.detach().requires_grad_(True)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        ops.cross_attention(leaf * 3, k, v)  # built in the capture altogether


def test_a_capture_over_two_streams():
    """What an input hangs on may come from another stream of the same capture."""
    from sleap_amd import ops

    q, k, v, _, _, _ = make(rng(39), 1, 4, 6, 1, 1, 16, torch.float16)
    leaf, side, graph = q.detach().requires_grad_(True), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    want = ops.cross_attention(q * 3, k, v)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            thrice = leaf * 3
        torch.cuda.current_stream().wait_stream(side)
        out = ops.cross_attention(thrice, k, v).detach()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        # weights in one term (off by 2^-11 of v at most) and in two, both results rounded (2^-11 each)
        assert (out.float() - want.float()).abs().max() <= 2.0 ** -11 * (v.float().abs().max() + 2 * want.float().abs().max()) * 1.01


def test_callables_graphed_by_torch():
    """torch's own capture of a function and its gradients, which keeps its warm-up's graph (on a stream of its own) while it captures."""
    from sleap_amd import ops

    p = torch.rand((30, 2), generator=rng(57), device=DEV) * 50

    def data(seed):
        g = rng(seed)
        return [normal(g, 2, n, 4, 32).requires_grad_(True) for n in (30, 700, 700)]

    def step(q, k, v):
        return ops.cross_attention(ops.rotary_axes(q, p, (8, 8)), k, v)

    graphed = torch.cuda.make_graphed_callables(step, tuple(data(58)))
    for seed in (59, 60, 61):
        one, two, dout = data(seed), data(seed), normal(rng(seed + 10), 2, 30, 4, 32)
        got, want = (f(*x) for f, x in ((graphed, one), (step, two)))
        for a, b in zip((got, *torch.autograd.grad(got, one, dout)), (want, *torch.autograd.grad(want, two, dout))):
            assert torch.equal(a, b)


def test_a_captured_fit_after_a_warm_up_that_lives():
    """Warm-up on a side stream whose graph is still held, then forward, backward and optimizer step in one graph; replayed on new inputs against
    the same steps made one by one."""
    from sleap_amd import ops

    g = rng(62)
    q0, w0 = normal(g, 1, 20, 2, 32, dtype=torch.float32), normal(g, 64, 64, dtype=torch.float32, scale=0.1)
    x, target = normal(g, 3, 500, 64, dtype=torch.float32), normal(g, 3, 20, 2, 32, dtype=torch.float32)
    place = torch.rand((20, 2), generator=g, device=DEV) * 9

    def make_fit():
        leaves = [t.clone().requires_grad_(True) for t in (q0, w0)]
        states = [[torch.zeros_like(t) for t in leaves] for _ in range(2)]
        count, rate = torch.zeros(1, dtype=torch.int64, device=DEV), torch.full((1,), 1e-2, device=DEV)

        def fit(update=True):
            for t in leaves:
                t.grad = None
            kv = (x @ leaves[1]).half().view(3, 500, 2, 32)
            q = ops.rotary_axes(leaves[0].half().expand(3, 20, 2, 32), place, (8, 8))
            loss = ((ops.cross_attention(q, kv, kv).float() - target) ** 2).mean()
            loss.backward()
            if update:
                with torch.no_grad():
                    count.add_(1)
                    ops.adamw_step(leaves, [t.grad for t in leaves], *states, step=count, lr=rate)
            return loss

        return leaves, fit

    (leaves, fit), (twins, twin) = make_fit(), make_fit()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = fit(update=False)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = fit()
    for turn in range(3):
        x.copy_(normal(rng(70 + turn), 3, 500, 64, dtype=torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        want = twin()
        assert torch.equal(loss.detach(), want.detach())
        for a, b in zip(leaves, twins):
            assert torch.equal(a.grad, b.grad) and torch.equal(a, b)
    assert torch.isfinite(held)


def test_two_calls_at_once_on_two_streams():
    """Calls with scratch, from two threads on streams of their own, do not meet."""
    import threading

    from sleap_amd import ops

    sets = [make(rng(34 + i), 2, 9, 3000 + 500 * i, 4, 2, 64, torch.bfloat16) for i in range(2)]
    want = []
    for q, k, v, dout, _, _ in sets:
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = ops.cross_attention(*leaves)
        want.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
    torch.cuda.synchronize()
    bad = []

    def work(i):
        q, k, v, dout, _, _ = sets[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
                out = ops.cross_attention(*leaves)
                got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


NAN_SHAPES = [(2, 40, 100, 4, 2, 32), (1, 52, 1024, 2, 2, 32), (1, 3, 9000, 2, 2, 64), (2, 300, 900, 2, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", NAN_SHAPES)
def test_a_nan_goes_where_it_is_used(dtype, shape):
    """In q: its row, and through it the keys of its head; in a visible key: all rows of its heads; in a value: its place in them; in dout: its
    row's dq and its head's keys. Workgroups along rows, along keys, and runs that are joined."""
    from sleap_amd import ops

    B, Tq, Tk, H, K, D = shape
    G = H // K
    for what in ("q", "k", "v", "dout"):
        q, k, v, dout, _, _ = make(rng(49), *shape, dtype)
        t = {"q": q, "k": k, "v": v, "dout": dout}[what]
        at = (B - 1, t.shape[1] - 2, t.shape[2] - 1, 5)
        t[at] = float("nan")
        leaves = [x.requires_grad_(True) for x in (q, k, v)]
        out, lse = ops.cross_attention(*leaves, return_lse=True)
        dq, dk, dv = torch.autograd.grad(out, leaves, dout)
        plain = ops.cross_attention(*(x.detach() for x in leaves))
        want = {n: torch.zeros_like(x, dtype=torch.bool) for n, x in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv))}
        b, row, h, d = at
        heads = slice(h * G, h * G + G) if what in "kv" else h
        key = h if what in "kv" else h // G
        if what == "q":
            want["out"][b, row, h], want["lse"][b, h, row], want["dq"][b, row, h], want["dk"][b, :, key], want["dv"][b, :, key] = (True,) * 5
        if what == "k":
            want["out"][b, :, heads], want["lse"][b, heads], want["dq"][b, :, heads], want["dk"][b, :, key], want["dv"][b, :, key] = (True,) * 5
        if what == "v":
            want["out"][b, :, heads, d], want["dq"][b, :, heads], want["dk"][b, :, key] = (True,) * 3
        if what == "dout":
            want["dq"][b, row, h], want["dk"][b, :, key], want["dv"][b, :, key, d] = (True,) * 3
        for n, x in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
            assert torch.equal(torch.isnan(x), want[n]), (what, n)
        assert torch.equal(torch.isnan(plain), want["out"]), what


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", NAN_SHAPES)
def test_scores_of_minus_infinity(dtype, shape):
    """A visible key that scores -inf has no weight; where all that a query sees do, its softmax is undefined: NaN, not the zeros of a query without a
    key. The one visible key with a finite score comes first, last, and in a run of its own."""
    from sleap_amd import ops

    B, Tq, Tk, H, K, D = shape
    q, k, v, dout, _, _ = make(rng(50), *shape, dtype)
    q[..., 0] = q[..., 0].abs() + 0.25
    low = k.clone()
    low[..., 0] = float("-inf")
    for at in (0, Tk // 2, Tk - 1):
        kk = low.clone()
        kk[0, at] = k[0, at]
        for grad in (False, True):
            out, lse = ops.cross_attention(q.clone().requires_grad_(grad), kk, v, return_lse=True)
            want = v[:1, at].repeat_interleave(H // K, 1)[:, None].expand(1, Tq, H, D)
            assert torch.equal(out[:1], want) and torch.isfinite(lse[:1]).all()
            if B > 1:
                assert torch.isnan(out[1:]).all() and torch.isnan(lse[1:]).all()
    leaves = [t.requires_grad_(True) for t in (q, low, v)]
    out, lse = ops.cross_attention(*leaves, return_lse=True)
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    assert all(torch.isnan(x).all() for x in torch.autograd.grad(out, leaves, dout))
    out, lse = ops.cross_attention(q, low, v, key_lengths=torch.zeros(B, dtype=torch.int32, device=DEV), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


# --------------------------------------------------------------------------------------------------
# AdamW
# --------------------------------------------------------------------------------------------------
def tensors(g, sizes, dtype, amsgrad, offset=0):
    def some(scale, kind=torch.float32):
        return [normal(g, n + offset, dtype=kind, scale=scale)[offset:] for n in sizes]

    p, gr, m = some(0.05, dtype), some(1e-2, dtype), some(2e-3)
    v = [t.square() for t in some(1e-2)]
    return p, gr, m, v, [t * 1.5 for t in v] if amsgrad else None


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("amsgrad", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw_matches_its_definition(dtype, amsgrad, offset):
    from sleap_amd import ops

    sizes = [1, 3, 4096, 4097, 0, 12289, 16, 5000] + [7 * i + 1 for i in range(130)]
    p, gr, m, v, w = tensors(rng(20), sizes, dtype, amsgrad, offset)
    if amsgrad:
        w = [t * f for t, f in zip(w, torch.rand(len(w)).tolist())]
    gr[5][17], v[3][0] = float("nan"), float("inf")
    how = dict(step=7, lr=3e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    want = [oracle.adamw(*[x[i] for x in (p, gr, m, v)], w[i] if amsgrad else None, **how) for i in range(len(sizes))]
    ops.adamw_step(p, gr, m, v, max_exp_avg_sqs=w, **how)
    for i, o in enumerate(want):
        for name, got in (("param", p), ("exp_avg", m), ("exp_avg_sq", v), ("max_exp_avg_sq", w)):
            if name in o:
                assert oracle.worst(got[i], o[name]) <= 1, (i, name)


def test_adamw_of_mixed_types_and_of_its_corners():
    from sleap_amd import ops

    g = rng(21)
    sets = [tensors(g, [100, 5000], dtype, False) for dtype in (torch.float32, torch.bfloat16, torch.float16)]
    p, gr, m, v = ([t for s in sets for t in s[j]] for j in range(4))
    for t in gr + m + v:
        t.zero_()  # no gradient so far: only the decay moves
    before = [t.double() for t in p]
    ops.adamw_step(p, gr, m, v, step=1, lr=0.5, weight_decay=0.5)
    for a, b in zip(p, before):
        assert oracle.worst(a, (b * 0.75, b.abs() * 1.01 * oracle.UNIT[a.dtype] + oracle.TINY[a.dtype])) <= 1
    ops.adamw_step([], [], [], [], step=1, lr=1.0)


def test_adamw_refuses_gradients_in_what_it_writes():
    from sleap_amd import ops

    p, gr, m, v, _ = tensors(rng(35), [40, 40], torch.float32, False)
    pool = torch.zeros(100, device=DEV)
    for lists in (([p[0]], [p[1]], [m[0]], [p[1]]), (p, [gr[0], p[0]], m, v), (p, [m[1], gr[1]], m, v), (p, [gr[0], v[1]], m, v), ([pool[:40], p[1]], [gr[0], pool[39:79]], m, v),
                  ([pool[40:80], p[1]], [gr[0], pool[1:41]], m, v)):
        with pytest.raises(ValueError, match="a gradient overlaps"):
            ops.adamw_step(*lists, step=1, lr=1e-3)
    # two parameters of one gradient, neighbours in memory, and a parameter that is its own gradient, are whole
    pool = normal(rng(36), 120, dtype=torch.float32)
    args = ([pool[:40], pool[80:], p[0]], [pool[40:80], pool[40:80], p[0]], [*m, torch.zeros_like(m[0])], [*v, torch.zeros_like(v[0])])
    alone = [[t.clone() for t in x] for x in args]
    ops.adamw_step(*args, step=1, lr=1e-3)
    ops.adamw_step(*alone, step=1, lr=1e-3)
    assert all(torch.equal(a, b) for j in (0, 2, 3) for a, b in zip(args[j], alone[j]))


def test_adamw_refuses_what_it_would_write_twice():
    from sleap_amd import ops

    p, gr, m, v, _ = tensors(rng(26), [40, 40], torch.float32, False)
    for lists in (([p[0], p[0]], gr, m, v), ([p[0][:30], p[0][20:]], [gr[0][:30], gr[0][20:]], [m[0][:30], m[1][:20]], [v[0][:30], v[1][:20]]),
                  (p, gr, [m[0], m[0]], v), (p, gr, m, [m[0], v[1]]), (p, gr, [p[1], m[1]], v)):
        with pytest.raises(ValueError, match="twice"):
            ops.adamw_step(*lists, step=1, lr=1e-3)
    with pytest.raises(ValueError, match="contiguous"):
        ops.adamw_step([p[0][::2]], [gr[0][::2]], [m[0][::2]], [v[0][::2]], step=1, lr=1e-3)
    with pytest.raises(ValueError, match="size"):
        ops.adamw_step(p, [gr[0], gr[1][:7]], m, v, step=1, lr=1e-3)
    with pytest.raises(TypeError, match="one type"):
        ops.adamw_step(p, [t.half() for t in gr], m, v, step=1, lr=1e-3)
    with pytest.raises(TypeError, match="float32"):
        ops.adamw_step(p, gr, [t.half() for t in m], v, step=1, lr=1e-3)
    with pytest.raises(ValueError, match="step"):
        ops.adamw_step(p, gr, m, v, step=0, lr=1e-3)


def test_adamw_refuses_negated_views():
    from sleap_amd import ops

    z = torch.ones((1,), device=DEV, dtype=torch.complex64)
    neg = z.conj().imag
    assert neg.is_neg() and neg.is_contiguous()
    one = [torch.ones(1, device=DEV) for _ in range(4)]
    for j in range(4):
        with pytest.raises(ValueError, match="negated"):
            ops.adamw_step(*[[neg if i == j else t] for i, t in enumerate(one)], step=1, lr=1e-3)
    with pytest.raises(ValueError, match="negated"):
        ops.adamw_step(*[[t] for t in one], step=1, lr=neg)


def test_adamw_refuses_to_cut_a_graph():
    from sleap_amd import ops

    def sets():
        return [torch.ones(4, device=DEV) for _ in range(4)]

    for j in range(4):
        one = sets()
        one[j] = one[j].requires_grad_(True) * 2
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.adamw_step(*[[t] for t in one], step=1, lr=1e-3)
        with torch.no_grad():
            ops.adamw_step(*[[t] for t in one], step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.adamw_step(*[[t] for t in sets()], step=1, lr=torch.ones(1, device=DEV).requires_grad_(True))


def test_an_adamw_step_is_noticed_by_graphs():
    from sleap_amd import ops

    w = normal(rng(27), 8, dtype=torch.float32).requires_grad_(True)
    loss = (w * w).sum()
    states = [torch.zeros(8, device=DEV) for _ in range(2)]
    ops.adamw_step([w], [torch.ones(8, device=DEV)], states[:1], states[1:], step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_a_captured_adamw_step_counts_on():
    from sleap_amd import ops

    p, gr, m, v, _ = tensors(rng(22), [300, 70], torch.float32, False)
    q, mm, vv = ([t.clone() for t in x] for x in (p, m, v))
    step, lr = torch.zeros(1, dtype=torch.int64, device=DEV), torch.full((1,), 1e-2, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.add_(1)
        ops.adamw_step(p, gr, m, v, step=step, lr=lr)
        with pytest.raises(RuntimeError, match="count as a tensor"):
            ops.adamw_step(p, gr, m, v, step=1, lr=lr)
    for t in range(1, 4):
        lr.fill_(1e-2 / t)
        graph.replay()
        ops.adamw_step(q, gr, mm, vv, step=t, lr=1e-2 / t)
        torch.cuda.synchronize()
        for a, b in zip(p + m + v, q + mm + vv):
            assert torch.allclose(a, b, rtol=4 * oracle.F32, atol=1e-9)  # lr and its decay once rounded more


def test_the_optimizer_follows_the_definition_over_steps():
    """Eight steps with a schedule against the 64-bit step, allowances added up; a state that was saved and loaded goes on."""
    from sleap_amd.nn.optim import AdamW

    g = rng(23)
    start = [normal(g, *s, dtype=torch.float32, scale=0.1) for s in ((16, 3, 3, 3), (16,), (33, 16), (7,))]
    params = [torch.nn.Parameter(t.clone()) for t in start]
    opt = AdamW([dict(params=params[:2], lr=1e-2), dict(params=params[2:], weight_decay=0.0)], lr=3e-3, amsgrad=True)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda t: 1 / (1 + t))
    state = [[t.double(), torch.zeros_like(t).double(), torch.zeros_like(t).double(), torch.zeros_like(t).double(), torch.zeros_like(t).double()] for t in start]
    for t in range(1, 9):
        for i, p in enumerate(params):
            p.grad = None if i == 3 else normal(g, *p.shape, dtype=torch.float32, scale=10.0 ** (i - 2))
            if i == 3:
                continue
            group = opt.param_groups[i // 2]
            x, m, v, w, e = state[i]
            o = oracle.adamw(x.float(), p.grad, m, v, w, step=t, lr=group["lr"], weight_decay=group["weight_decay"])
            moved = x - x.float().double()
            state[i] = [o["param"][0] + moved, o["exp_avg"][0], o["exp_avg_sq"][0], o["max_exp_avg_sq"][0], e + o["param"][1] * 4 * t]
        opt.step()
        sched.step()
        if t == 4:
            saved = opt.state_dict()
            opt = AdamW([dict(params=params[:2]), dict(params=params[2:])], amsgrad=True)
            opt.load_state_dict(saved)
            sched.optimizer = opt
            assert all(s["exp_avg"].dtype == torch.float32 for s in opt.state.values())
    for p, (x, *_, e) in zip(params, state):
        assert oracle.worst(p.detach(), (x, e + 1e-30)) <= 1
    assert torch.equal(params[3].detach(), start[3])


def test_the_optimizer_keeps_float32_states_of_16_bit_parameters():
    from sleap_amd.nn.optim import AdamW

    p = torch.nn.Parameter(normal(rng(24), 50, dtype=torch.bfloat16))
    p.grad = torch.full_like(p, 1e-3)
    opt = AdamW([p], lr=1e-2)
    opt.step()
    saved = opt.state_dict()
    m = opt.state[p]["exp_avg"].clone()
    opt.load_state_dict(saved)
    assert opt.state[p]["exp_avg"].dtype == torch.float32 and torch.equal(opt.state[p]["exp_avg"], m)
    opt.step()
    assert opt.state[p]["step"] == 2
    p.grad = torch.ones((5, 10), device=DEV, dtype=torch.bfloat16).T.reshape(50)  # any layout of gradient
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device=DEV)
        with pytest.raises(RuntimeError, match="counts on the host"):
            opt.step()


def test_the_optimizer_reads_negated_gradients():
    """What the backward pass of a conjugation may leave: a view that torch holds with the other sign."""
    from sleap_amd.nn.optim import AdamW

    for n in (1, 5):
        z = torch.randn(n, generator=rng(55), device=DEV, dtype=torch.complex64)
        params = [torch.nn.Parameter(torch.ones(n, device=DEV)) for _ in range(2)]
        params[0].grad, params[1].grad = z.conj().imag, -z.imag
        assert params[0].grad.is_neg()
        AdamW(params).step()
        assert torch.equal(*params)


def test_what_the_fitting_commands_step_with():
    from sleap_amd.nn.optim import AdamW, adam

    kernel = normal(rng(56), 8, 4, 3, 3, dtype=torch.float32)
    for p, kind in ((kernel, AdamW), (kernel.to(memory_format=torch.channels_last), torch.optim.Adam), (kernel.double(), torch.optim.Adam), (kernel.cpu(), torch.optim.Adam)):
        p = torch.nn.Parameter(p)
        p.grad = torch.ones_like(p)
        opt = adam([p], 1e-2)
        assert type(opt) is kind
        opt.step()


def test_the_optimizer_goes_on_from_a_state_of_torch():
    """What torch's AdamW saved (a float32 tensor as step) continues: a step from it is `ops.adamw_step` with the next count; what this
    optimizer would do otherwise is refused."""
    from sleap_amd import ops
    from sleap_amd.nn.optim import AdamW

    g = rng(37)
    p = torch.nn.Parameter(normal(g, 70, dtype=torch.float32))
    theirs = torch.optim.AdamW([p], lr=1e-2, amsgrad=True)
    for _ in range(3):
        p.grad = normal(g, 70, dtype=torch.float32)
        theirs.step()
    saved = theirs.state_dict()
    q, *states = (t.detach().clone() for t in (p, *(theirs.state[p][k] for k in ("exp_avg", "exp_avg_sq", "max_exp_avg_sq"))))
    opt = AdamW([p])
    opt.load_state_dict(saved)
    opt.step()
    assert opt.state[p]["step"] == 4 and isinstance(opt.state[p]["step"], int)
    ops.adamw_step([q], [p.grad], *([t] for t in states[:2]), max_exp_avg_sqs=states[2:], step=4, lr=1e-2)
    assert torch.equal(p.detach(), q) and all(torch.equal(opt.state[p][k], t) for k, t in zip(("exp_avg", "exp_avg_sq", "max_exp_avg_sq"), states))
    for other, what in ((torch.optim.AdamW([p], maximize=True), "maximize"), (torch.optim.Adam([p], weight_decay=0.1), "decoupled")):
        before = opt.state_dict()["param_groups"]
        with pytest.raises(ValueError, match=what):
            opt.load_state_dict(other.state_dict())
        assert opt.state_dict()["param_groups"] == before
    opt.load_state_dict(torch.optim.Adam([p]).state_dict())  # without decay both are one


def test_the_optimizer_refuses_states_of_unknown_decay():
    from sleap_amd.nn.optim import AdamW

    p = torch.nn.Parameter(normal(rng(52), 9, dtype=torch.float32))
    old = torch.optim.Adam([p], weight_decay=0.1).state_dict()
    del old["param_groups"][0]["decoupled_weight_decay"]
    opt = AdamW([p])
    with pytest.raises(ValueError, match="decoupled"):
        opt.load_state_dict(old)
    opt.load_state_dict(AdamW([p], weight_decay=0.3).state_dict())
    assert opt.param_groups[0]["weight_decay"] == 0.3
    opt.load_state_dict(torch.optim.Adam([p]).state_dict())
    opt.param_groups[0]["weight_decay"] = 0.2
    AdamW([p]).load_state_dict(opt.state_dict())  # decays decoupled from here on, and says so
    torch.optim.AdamW([p]).load_state_dict(opt.state_dict())


def test_the_optimizer_refuses_groups_that_it_would_step_otherwise():
    from sleap_amd.nn.optim import AdamW

    p = torch.nn.Parameter(normal(rng(52), 9, dtype=torch.float32))
    for more, what in ((dict(maximize=True), "maximize"), (dict(decoupled_weight_decay=False, weight_decay=0.1), "decoupled")):
        with pytest.raises(ValueError, match=what):
            AdamW([dict(params=[p], **more)])


def test_the_optimizer_loads_what_hooks_leave():
    """A hook that changes the state ahead of its loading is heard, one that looks at what was loaded sees float32."""
    from sleap_amd.nn.optim import AdamW

    p = torch.nn.Parameter(normal(rng(53), 9, dtype=torch.bfloat16))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    opt.step()

    def half(_, saved):
        return {**saved, "state": {i: {n: x / 2 if torch.is_tensor(x) else x for n, x in s.items()} for i, s in saved["state"].items()}}

    twin, seen = AdamW([p]), []
    twin.register_load_state_dict_pre_hook(half)
    twin.register_load_state_dict_post_hook(lambda o: seen.append(o.state[p]["exp_avg"].dtype))
    twin.load_state_dict(opt.state_dict())
    assert torch.equal(twin.state[p]["exp_avg"], opt.state[p]["exp_avg"] / 2) and seen == [torch.float32]


def test_the_fitting_commands_step_on_the_gpu():
    """tools/train_benchmark_model.py as it is started, three small steps of it: the fit runs and its losses stay finite."""
    import os
    import subprocess
    import sys
    import tempfile

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as d:
        run = subprocess.run([sys.executable, os.path.join(root, "tools", "train_benchmark_model.py"), "--steps", "3", "--batch", "2", "--crop", "128", "--pool", "1",
                              "--out", os.path.join(d, "w.npz")], capture_output=True, text=True, timeout=110)
        assert run.returncode == 0 and os.path.exists(os.path.join(d, "w.npz")), run.stderr[-2000:]
    losses = [float(line.split("loss")[1].split()[0]) for line in run.stdout.splitlines() if line.startswith("step")]
    assert len(losses) == 2 and all(math.isfinite(v) for v in losses) and "on cuda" in run.stdout


# --------------------------------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------------------------------
def test_keypoint_queries_read_a_padded_clip_and_are_fitted():
    """Queries with sub-pixel places read the tokens of clips of different lengths: rotary -> attention -> loss -> gradients -> AdamW,
    three steps of a whole model, each step's gradients against the same graph in 64 bits."""
    from sleap_amd import ops
    from sleap_amd.nn.optim import AdamW

    g = rng(25)
    B, frames, side, N, H, D = 3, 3, 7, 26, 4, 32
    Tk = frames * side * side
    feats = normal(g, B, Tk, H * D, dtype=torch.bfloat16)
    grid = torch.stack(torch.meshgrid(torch.arange(frames, device=DEV), torch.arange(side, device=DEV), torch.arange(side, device=DEV), indexing="ij"), -1).reshape(Tk, 3)
    places = torch.rand((B, N, 3), generator=g, device=DEV) * side
    lengths = torch.tensor([Tk, 2 * side * side, 0], dtype=torch.int32, device=DEV)
    target = normal(g, B, N, 2, dtype=torch.float32)
    params = [torch.nn.Parameter(normal(g, *s, dtype=torch.float32, scale=0.2)) for s in ((N, H * D), (H * D, H * D), (H * D, H * D), (H * D, 2))]
    opt = AdamW(params, lr=1e-3)

    def loss_of(ps, rotary, attend, kind):
        q0, wk, wv, wo = ps
        q = rotary(q0.to(kind).expand(B, N, H * D).reshape(B, N, H, D), places)
        k = rotary((feats.to(kind) @ wk.to(kind)).reshape(B, Tk, H, D), grid)
        v = (feats.to(kind) @ wv.to(kind)).reshape(B, Tk, H, D)
        y = attend(q, k, v).reshape(B, N, H * D).to(wo.dtype) @ wo
        return ((y - target.to(y.dtype)) ** 2).mean()

    def rotary64(x, p):
        axis = [0] * 4 + [1] * 6 + [2] * 6
        f = torch.tensor([10000.0 ** -(i / n) for n in (4, 6, 6) for i in range(n)], device=DEV, dtype=torch.float64)
        a = p.double()[..., axis] * f
        c, s = a.cos()[..., None, :], a.sin()[..., None, :]
        u, w = x[..., :16], x[..., 16:]
        return torch.cat([u * c - w * s, w * c + u * s], -1)

    def attend64(q, k, v):
        s = (q.transpose(1, 2) @ k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(D)
        s = s.masked_fill((torch.arange(Tk, device=DEV)[None] >= lengths[:, None])[:, None, None], -1e300)
        w = torch.softmax(s, -1) * (lengths > 0)[:, None, None, None]
        return (w @ v.transpose(1, 2).contiguous()).transpose(1, 2)

    for _ in range(3):
        opt.zero_grad()
        loss = loss_of(params, lambda x, p: ops.rotary_axes(x, p, (4, 6, 6)), lambda q, k, v: ops.cross_attention(q, k, v, key_lengths=lengths), torch.bfloat16)
        loss.backward()
        twins = [p.detach().double().requires_grad_(True) for p in params]
        wants = torch.autograd.grad(loss_of(twins, rotary64, attend64, torch.float64), twins)
        for p, want in zip(params, wants):
            # bf16 along the way: inputs, products, turns, weights and outputs are rounded, about ten roundings of 2^-9 each that
            # add up along sums of hundreds of terms of either sign; held to ten of them over the whole gradient
            assert (p.grad.double() - want).norm() <= 10 * 2.0 ** -8 * want.norm()
        opt.step()
    assert all(torch.isfinite(p).all() for p in params)
