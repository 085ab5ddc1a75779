"""Derivatives of the rotary positions in forward mode, alone and over the gradient; the cache's results have none."""
import pytest
import torch
from torch.autograd import forward_ad

import mxfp4_ref as R
from ffa_mi355x.rope_axes import AxisRope

pytestmark = pytest.mark.gpu


def _case(gpu, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = [torch.randn(2, 5, H, 128, generator=g).to(dtype).to(gpu) for H in (4, 2, 4, 2)]
    return AxisRope((20, 44), device=gpu), torch.randint(0, 9000, (2, 2, 5), generator=g).to(gpu), *x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inverse", [False, True])
def test_tangents_are_turned(gpu, dtype, inverse):
    rope, pos, q, k, tq, tk = _case(gpu, dtype)
    want = rope.rotate(pos, tq, tk, inverse=inverse)
    value = rope.rotate(pos, q, k, inverse=inverse)
    with forward_ad.dual_level():
        got = rope.rotate(pos, forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk), inverse=inverse)
        for x, v, t in zip(got, value, want):
            x = forward_ad.unpack_dual(x)
            assert torch.equal(x.primal, v) and torch.equal(x.tangent, t)
        (one, other) = (forward_ad.unpack_dual(x) for x in rope.rotate(pos, q, forward_ad.make_dual(k, tk), inverse=inverse))
        assert torch.equal(other.tangent, want[1]) and (one.tangent is None or (one.tangent == 0).all())
        alone = forward_ad.unpack_dual(rope.rotate(pos, forward_ad.make_dual(q, tq), inverse=inverse))
        assert torch.equal(alone.primal, value[0]) and torch.equal(alone.tangent, want[0])
        with torch.no_grad():  # which does not switch forward mode off
            assert torch.equal(forward_ad.unpack_dual(rope.rotate(pos, forward_ad.make_dual(q, tq), inverse=inverse)).tangent, want[0])
        with pytest.raises(ValueError):
            rope.rotate(pos, forward_ad.make_dual(q, tq), inplace=True)
        assert forward_ad.unpack_dual(rope.rotate(pos, q)).tangent is None


def test_tangents_of_gradients(gpu):
    """The gradient of sum((R q)^3) along a tangent, against differences of the gradient."""
    rope, pos, q, _, tq, _ = _case(gpu, seed=1)

    def gradient(x):
        x = x.detach().requires_grad_()
        return torch.autograd.grad((rope.rotate(pos, x) ** 3).sum(), x)[0]

    with forward_ad.dual_level():
        x = forward_ad.make_dual(q.clone().requires_grad_(), tq)
        (g,) = torch.autograd.grad((rope.rotate(pos, x) ** 3).sum(), x, create_graph=True)
        got = forward_ad.unpack_dual(g).tangent
    # 3 R^-1 (R q)^2 along t is 6 R^-1 (R q)(R t); its central difference is that exactly, but for rounding: of values of at most
    # 3 |R q|^2 < 3 (2^4)^2 at a step of 1/2, ten operations each
    want = gradient(q + tq / 2) - gradient(q - tq / 2)
    assert (got - want).abs().max() < 10 * 2.0 ** -24 * 3 * 2.0 ** 8
    again = rope.rotate(pos, 6 * rope.rotate(pos, q) * rope.rotate(pos, tq), inverse=True)  # of at most 6 x 2^6, the same bound
    assert (got - again).abs().max() < 10 * 2.0 ** -24 * 3 * 2.0 ** 8


def test_appended_rows_have_no_derivatives(gpu):
    rope, _, q, k, tq, tk = _case(gpu)
    cache = R.make_cache(2, 2, gpu)
    pos, table = torch.zeros(2, dtype=torch.int32, device=gpu), torch.arange(2, dtype=torch.int32, device=gpu)[:, None]
    got = cache.append_rotary(q.clone().requires_grad_(), k.clone().requires_grad_(), k, pos, table, rope, values=True)
    assert not any(x.requires_grad for x in got)
    with forward_ad.dual_level():
        got = cache.append_rotary(forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk), k, pos, table, rope, values=True)
        assert all(forward_ad.unpack_dual(x).tangent is None for x in got)
