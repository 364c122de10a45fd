"""GPU: rotary positions from token positions and frequencies against the 64-bit formula."""
import math

import pytest
import torch

from oracle import text as ot

pytestmark = pytest.mark.gpu


def _bound(ref, x, dtype, magnitude):
    """One rounding to the type (eps / 2 of the value; half of the least step near zero), and
    the fp32 steps before it: sine and cosine to 2^-22, products and sum three roundings of
    at most 2 |x| magnitude."""
    u = torch.finfo(dtype).eps / 2
    big = x.double().abs().amax(-1, keepdim=True) * magnitude
    return u * ref.abs() + 2.0 ** -20 * big + torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def _check(x, y, positions, f, layout, magnitude=1.0, inverse=False):
    ref = ot.rotary(x, positions, f, layout, magnitude, inverse)
    err = (y.double() - ref).abs()
    tol = _bound(ref, x, x.dtype, magnitude)
    assert (err <= tol).all(), (err / tol).max().item()
    r = 2 * f.numel()
    assert torch.equal(y[..., r:], x[..., r:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 2, 2), (2, 1, 24, 8, 128, 128), (3, 77, 5, 5, 96, 32), (1, 1003, 3, 1, 64, 64),
                                   (2, 19, 4, 2, 80, 20), (1, 33, 2, 1, 7, 6), (1, 5, 1, 1, 1024, 1024)])
def test_rotary_matches_formula(cuda, dtype, layout, shape):
    from quantfun2_b200 import kernels as K

    B, S, H, Hk, D, r = shape
    g = torch.Generator(device=cuda).manual_seed(S)
    q = torch.randn(B, S, H, D, device=cuda, generator=g).to(dtype)
    k = torch.randn(B, S, Hk, D, device=cuda, generator=g).to(dtype)
    pos = torch.randint(0, 100000, (B, S), device=cuda, generator=g)
    f = K.rotary_inv_freq(r, device=cuda)
    q0, k0 = q.clone(), k.clone()
    yq, yk = K.rotary_apply(q, k, pos, f, layout=layout, magnitude=1.25)
    _check(q, yq, pos, f, layout, 1.25)
    _check(k, yk, pos, f, layout, 1.25)
    assert torch.equal(q, q0) and torch.equal(k, k0)
    # in place gives the same bits; int32 positions too
    a, b = K.rotary_apply_(q, k, pos.int(), f, layout=layout, magnitude=1.25)
    assert a is q and b is k and torch.equal(q, yq) and torch.equal(k, yk)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_and_negative_positions(cuda, layout):
    from quantfun2_b200 import kernels as K

    pos = torch.tensor([0, 1, -1, 131071, 10 ** 6 + 7, 2 ** 31 - 1, -2 ** 31], device=cuda)
    x = torch.randn(1, 7, 2, 128, device=cuda)
    f = K.rotary_inv_freq(128, scaling="by_parts", factor=8.0, device=cuda)
    y, none = K.rotary_apply(x, None, pos, f, layout=layout)
    assert none is None
    _check(x, y, pos, f, layout)


def test_strided_views_and_broadcast_positions(cuda):
    from quantfun2_b200 import kernels as K

    f = K.rotary_inv_freq(64, device=cuda)
    pos = torch.arange(50, device=cuda)
    buf = torch.randn(2, 6, 50, 64 + 4, device=cuda).bfloat16()
    for off in (0, 1):                                      # rows off the 16-byte alignment
        x = buf[..., off:off + 64].transpose(1, 2)          # [B, S, H, D] view of [B, H, S, D + 4]
        y, _ = K.rotary_apply(x, None, pos, f)
        _check(x, y, pos, f, "half")
        z, _ = K.rotary_apply(x, None, pos[None], f)
        assert torch.equal(y, z)
    joint = torch.randn(2, 50, 8, 64, device=cuda).half()   # q and k slices of one buffer, in place
    ref = joint.clone()
    K.rotary_apply_(joint[:, :, :5], joint[:, :, 5:7], pos, f, layout="interleaved")
    _check(ref[:, :, :7], joint[:, :, :7], pos, f, "interleaved")
    assert torch.equal(joint[:, :, 7], ref[:, :, 7])


def test_inverse_turns_back(cuda):
    from quantfun2_b200 import kernels as K

    x = torch.randn(1, 40, 3, 96, device=cuda)
    pos = torch.arange(40, device=cuda) * 977
    f = K.rotary_inv_freq(48, device=cuda)
    for layout in ("half", "interleaved"):
        y, _ = K.rotary_apply(x, None, pos, f, layout=layout)
        z, _ = K.rotary_apply(y, None, pos, f, layout=layout, inverse=True)
        _check(y, z, pos, f, layout, inverse=True)
        # two passes, each to 2^-20 of the row's greatest
        assert ((z - x).abs() <= 2.0 ** -18 * x.abs().amax(-1, keepdim=True)).all()


def test_empty_and_graph(cuda):
    from quantfun2_b200 import kernels as K

    f = K.rotary_inv_freq(32, device=cuda)
    y, _ = K.rotary_apply(torch.empty(0, 3, 2, 64, device=cuda), None, torch.arange(3, device=cuda), f)
    assert y.shape == (0, 3, 2, 64)
    x = torch.randn(2, 9, 4, 64, device=cuda).bfloat16()
    pos = torch.arange(9, device=cuda)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.rotary_apply(x, None, pos, f)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        y, _ = K.rotary_apply(x, None, pos, f)
    x.copy_(torch.randn_like(x))
    pos += 5
    graph.replay()
    torch.cuda.synchronize()
    _check(x, y, pos, f, "half")


def test_refusals(cuda):
    from quantfun2_b200 import kernels as K

    x = torch.randn(2, 4, 3, 64, device=cuda).bfloat16()
    pos, f = torch.arange(4, device=cuda), K.rotary_inv_freq(64, device=cuda)
    bad = [
        (x[0], None, pos, f), (x.double(), None, pos, f), (x, x[:, :3], pos, f), (x, x.half(), pos, f),
        (x, None, pos.float(), f), (x, None, pos[:3], f), (x, None, pos.cpu(), f), (x, None, pos, f.float()),
        (x, None, pos, f.cpu()), (x, None, pos, K.rotary_inv_freq(66, device=cuda)), (x.transpose(2, 3), None, pos, f),
        (x.float().requires_grad_(), None, pos, f), (x.cpu(), None, pos, f),
    ]
    for args in bad:
        with pytest.raises(K.QF2Error):
            K.rotary_apply(*args)
    with pytest.raises(K.QF2Error):
        K.rotary_apply(x, None, pos, f, layout="other")
    with pytest.raises(K.QF2Error):
        K.rotary_apply_(x[:, :1].expand(2, 4, 3, 64), None, pos, f)


def test_agrees_with_rope_apply(cuda):
    """The interleaved layout on the positions of a rope_apply table gives its rotation."""
    from quantfun2_b200 import kernels as K

    x = torch.randn(2, 100, 4, 128, device=cuda).bfloat16()
    pos = torch.arange(100, device=cuda)
    f = K.rotary_inv_freq(128, device=cuda)
    theta = pos.double()[:, None] * f
    table = torch.polar(torch.ones_like(theta), theta).to(torch.complex64)
    a, _ = K.rope_apply(x, x, table)
    b, _ = K.rotary_apply(x, None, pos, f, layout="interleaved")
    # both round a value known to 2^-20 of the row's greatest
    tol = 2 * (2.0 ** -8 * a.double().abs() + 2.0 ** -20 * x.double().abs().amax())
    assert ((a.double() - b.double()).abs() <= tol).all()


def test_derivatives_are_refused(cuda):
    """Neither a gradient nor a forward tangent is dropped without a word."""
    from torch.autograd import forward_ad

    from quantfun2_b200 import attention as A
    from quantfun2_b200 import kernels as K

    x = torch.randn(1, 4, 2, 64, device=cuda)
    h = x.bfloat16()
    pos, f = torch.arange(4, device=cuda), K.rotary_inv_freq(64, device=cuda)
    calls = [lambda t: K.rotary_apply(t, None, pos, f), lambda t: K.rotary_apply(x, t, pos, f), lambda t: K.rotary_apply_(t, None, pos, f),
             lambda t: A.masked_attn(t.bfloat16(), h, h), lambda t: A.masked_attn(h, h, t.bfloat16()),
             lambda t: A.masked_attn(h, h, h, slopes=t[0, :, 0, 0].contiguous())]
    for call in calls:
        call(x.clone())
        with forward_ad.dual_level():
            with pytest.raises(K.QF2Error, match="tangent"):
                call(forward_ad.make_dual(x.clone(), torch.ones_like(x)))
            call(x.clone())                                              # no tangent of its own
        with pytest.raises(Exception):
            torch.func.jvp(lambda t: call(t), (x.clone(),), (torch.ones_like(x),))
        with pytest.raises(Exception):
            torch.func.grad(lambda t: call(t)[0].float().sum())(x.clone())
    with pytest.raises(K.QF2Error, match="gradient"):
        K.rotary_apply(x, None, pos, f.clone().requires_grad_())
    with pytest.raises(K.QF2Error, match="gradient"):
        A.masked_attn(h, h, h, out=h.clone().requires_grad_())
