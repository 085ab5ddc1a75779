"""The cache that holds keys and values in 4 bits, on the GPU against its definition in 64 bits: rotary positions with
several axes, append, read-back, exact attention, and a run of them together.

What a page holds is compared byte by byte (codes and powers of two are decided by exact comparisons, so every
implementation of the definition gives the same ones); where keys are turned first, in fp32, but for elements that lie
within the turn's error of a midpoint.
"""
import math

import numpy as np
import pytest
import torch

import mxfp4_ref as R
from attend_ref import U, assert_close, reference
from ffa_mi355x.attend import SharedPrefix
from ffa_mi355x.pages import PagePool
from ffa_mi355x.paged_mxfp4 import PagedMXFP4Cache
from ffa_mi355x.rope_axes import AxisRope

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALF_STEP = {**U, torch.float32: 2.0 ** -24}


def _rand(g, *shape):
    return torch.randn(shape, generator=g)


def _f64(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------------------------- rotary positions
def _check_turned(got, x, positions, rope, inverse=False):
    want = R.rotate(_f64(x), positions.cpu().numpy(), rope.axis, rope.inv_freq, rope.adjacent, inverse)
    limit = R.turn_bound(_f64(x), rope.adjacent) + HALF_STEP[got.dtype] * (1 + 2.0 ** -10) * np.abs(want) + 2.0 ** -25
    assert (np.abs(_f64(got) - want) <= limit).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("sections,order", [((64,), "blocks"), ((16, 24, 24), "blocks"), ((24, 20, 20), "cycled"),
                                            ((10, 30, 4, 20), "cycled")])
@pytest.mark.parametrize("B,T,HQ,HKV", [(1, 1, 1, 1), (3, 1, 7, 1), (1, 67, 32, 8), (2, 1030, 3, 2)])
def test_rotate(gpu, dtype, pairs, sections, order, B, T, HQ, HKV):
    g = torch.Generator().manual_seed(3)
    rope = AxisRope(sections, device=gpu, pairs=pairs, order=order)
    q, k = _rand(g, B, T, HQ, 128).to(TYPES[dtype]).to(gpu), _rand(g, B, T, HKV, 128).to(TYPES[dtype]).to(gpu)
    pos = torch.randint(-100, 200000, (len(sections), B, T), generator=g).to(gpu)
    rq, rk = rope.rotate(pos, q, k)
    _check_turned(rq, q, pos, rope)
    _check_turned(rk, k, pos, rope)
    back = rope.rotate(pos.int(), q, inverse=True)
    _check_turned(back, q, pos, rope, inverse=True)


def test_rotate_far_positions(gpu):
    """Angles of positions that fp32 does not hold, and frequencies of the caller's."""
    g = torch.Generator().manual_seed(5)
    freq = torch.rand(64, generator=g, dtype=torch.float64)
    rope = AxisRope((32, 32), device=gpu, inv_freq=freq)
    q = _rand(g, 1, 9, 2, 128).to(gpu)
    pos = torch.tensor([2 ** 24 + 1, 2 ** 31 + 7, -2 ** 31 - 1, 10 ** 7, 0, 1, -1, 123456789, 2 ** 25 + 3], device=gpu).expand(2, 9)
    got, want = rope.rotate(pos, q), R.rotate(_f64(q), pos[:, None].cpu().numpy(), rope.axis, rope.inv_freq, False)
    # the product in turns is off by 2^-53 of 2^31 / (2 pi) turns, on either side: 2 pi 2^-24 in the angle at most
    limit = R.turn_bound(_f64(q), False) + 2.0 ** -20 * np.abs(_f64(q)).max() + 2.0 ** -24 * np.abs(want)
    assert (np.abs(_f64(got) - want) <= limit).all()


def test_rotate_many_tokens(gpu):
    """Sixteen tokens a workgroup, the last one's fewer; two sequences in one workgroup."""
    g = torch.Generator().manual_seed(9)
    rope, q, k = AxisRope((64,), device=gpu), _rand(g, 2, 8205, 1, 128).bfloat16().to(gpu), _rand(g, 2, 8205, 1, 128).bfloat16().to(gpu)
    pos = torch.randint(0, 2 ** 20, (1, 2, 8205), generator=g).to(gpu)
    for x, y in zip((q, k), rope.rotate(pos, q, k)):
        _check_turned(y, x, pos, rope)


def test_rotate_strides_and_in_place(gpu):
    """Views of a joined projection, heads before tokens, one position row for all sequences, and in place."""
    g = torch.Generator().manual_seed(7)
    rope = AxisRope((16, 24, 24), device=gpu)
    B, T, HQ, HKV = 2, 33, 6, 2
    joined = _rand(g, B, T, (HQ + 2 * HKV) * 128).half().to(gpu)
    q, k = joined[..., :HQ * 128].view(B, T, HQ, 128), joined[..., HQ * 128:(HQ + HKV) * 128].view(B, T, HKV, 128)
    pos = torch.randint(0, 5000, (3, B, T), generator=g).to(gpu)
    want = rope.rotate(pos, q.contiguous(), k.contiguous())
    got = rope.rotate(pos, q, k)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    hq = q.transpose(1, 2).contiguous()  # [B, H, T, 128], as transformers keeps them
    assert torch.equal(rope.rotate(pos, hq.transpose(1, 2)), want[0])
    wide = torch.zeros(B, T, HQ, 132, dtype=q.dtype, device=gpu)  # rows that no 16-byte load reaches: copied
    wide[..., :128] = q
    assert torch.equal(rope.rotate(pos, wide[..., :128]), want[0])
    one = pos[:, 0]
    assert torch.equal(rope.rotate(one, q), rope.rotate(one[:, None].expand(3, B, T).contiguous(), q))
    assert torch.equal(rope.rotate(pos.transpose(1, 2).contiguous().transpose(1, 2), q), want[0])
    rest = joined[..., (HQ + HKV) * 128:].clone()
    a, b = rope.rotate(pos, q, k, inplace=True)
    assert a is q and b is k and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(joined[..., (HQ + HKV) * 128:], rest)
    with pytest.raises(ValueError):
        rope.rotate(pos, wide[..., :128], inplace=True)
    with pytest.raises(ValueError):
        rope.rotate(pos, q[:, :1].expand(B, T, HQ, 128), inplace=True)


def test_rotate_in_place_beside_a_graph(gpu):
    """What autograd saved before it was turned in place is refused in the backward pass; q and k at one address are."""
    rope, pos = AxisRope((64,), device=gpu), torch.arange(5, device=gpu)[None]
    w = torch.randn(1, 5, 2, 128, device=gpu, requires_grad=True)
    x = torch.randn(1, 5, 2, 128, device=gpu)
    loss = (w * x).sum()
    rope.rotate(pos, x, inplace=True)
    with pytest.raises(RuntimeError):
        loss.backward()
    with torch.inference_mode():
        y = x.clone()
        assert torch.equal(rope.rotate(pos, y, inplace=True), rope.rotate(pos, x))
    with pytest.raises(ValueError):
        rope.rotate(pos, x, x[:, :, :1], inplace=True)
    with pytest.raises(ValueError):
        rope.rotate(pos, w, inplace=True)


def test_rotate_empty_and_refusals(gpu):
    rope = AxisRope((64,), device=gpu)
    q = torch.zeros(2, 0, 4, 128, device=gpu)
    assert rope.rotate(torch.zeros(1, 2, 0, dtype=torch.int64, device=gpu), q).shape == q.shape
    x, pos = torch.randn(2, 3, 4, 128, device=gpu), torch.arange(6, device=gpu).view(1, 2, 3)
    a, b = rope.rotate(pos, x[:, :, :0], x)  # no query heads
    assert a.shape == (2, 3, 0, 128) and torch.equal(b, rope.rotate(pos, x))
    a, b = rope.rotate(pos, x, x[:, :, :0])
    assert b.shape == (2, 3, 0, 128) and torch.equal(a, rope.rotate(pos, x))
    for bad in ((pos.float(), x), (pos[:, :1].contiguous(), x), (pos.cpu(), x), (pos, x[..., :64]), (pos, x[0])):
        with pytest.raises(ValueError):
            rope.rotate(*bad)
    with pytest.raises(ValueError):
        rope.rotate(pos, x, x.half())
    with pytest.raises(NotImplementedError):
        rope.rotate(pos, x.double())


@pytest.mark.parametrize("pairs", ["half", "adjacent"])
def test_rotate_gradient(gpu, pairs):
    """The gradient of the formula, and differences of the function."""
    g = torch.Generator().manual_seed(11)
    rope = AxisRope((20, 44), device=gpu, pairs=pairs)
    q, k = _rand(g, 2, 5, 3, 128).to(gpu).requires_grad_(), _rand(g, 2, 5, 1, 128).to(gpu).requires_grad_()
    pos = torch.randint(0, 9000, (2, 2, 5), generator=g).to(gpu)
    gq, gk = _rand(g, 2, 5, 3, 128).to(gpu), _rand(g, 2, 5, 1, 128).to(gpu)
    rq, rk = rope.rotate(pos, q, k)
    dq, dk = torch.autograd.grad([rq, rk], [q, k], [gq, gk])
    _check_turned(dq, gq, pos, rope, inverse=True)
    _check_turned(dk, gk, pos, rope, inverse=True)
    d = _rand(g, 2, 5, 3, 128).to(gpu)  # linear: a difference of any size is the derivative but for rounding
    change = ((rope.rotate(pos, (q + d).detach()) - rope.rotate(pos, (q - d).detach())).double() / 2 * gq.double()).sum()
    assert abs(float(change - (dq.double() * d.double()).sum())) < 2.0 ** -20 * float((gq.abs() * d.abs()).sum() + gq.abs().sum())
    (only,) = torch.autograd.grad(rope.rotate(pos, q, k)[0], [q], [gq])  # k's result unused
    assert torch.equal(only, dq)
    (second,) = torch.autograd.grad((torch.autograd.grad(rope.rotate(pos, q).square().sum(), q, create_graph=True)[0] * gq).sum(), q)
    assert torch.allclose(second, 2 * gq, atol=1e-5)  # a rotation keeps lengths: the gradient of |R q|^2 is 2 q
    with pytest.raises(ValueError):
        rope.rotate(pos, q, inplace=True)
    with torch.no_grad():
        assert not rope.rotate(pos, q).requires_grad


# ---------------------------------------------------------------------------- append and read-back
def _edges(g, shape):
    """Values as the quantizer meets them: normal ones, whole blocks of zeros, ties, large, tiny, infinities, NaN."""
    x = _rand(g, *shape)
    flat = x.view(-1, 32)
    n = flat.shape[0]
    pick = torch.randperm(n, generator=g)
    part = max(1, n // 10)
    flat[pick[:part]] = 0
    flat[pick[part:2 * part]] = (torch.randint(-28, 29, (len(pick[part:2 * part]), 32), generator=g) / 4).float()  # quarters
    flat[pick[2 * part:3 * part]] *= 2.0 ** -30
    flat[pick[3 * part:4 * part]] *= 30000.0
    flat[pick[4 * part:4 * part + 1], 3] = float("inf")
    flat[pick[4 * part + 1:4 * part + 2], 7] = float("nan")
    flat[pick[4 * part + 2:4 * part + 3], 9] = -0.0
    return x


def _append_case(g, B, T, HKV, dtype, dev, pos, seed=0):
    npg = [-(-(p + T) // 64) for p in pos]
    P = sum(npg) + 3
    ids = torch.randperm(P, generator=g).to(torch.int32)
    cols = max(max(npg), 1) + 1
    table = torch.full((B, cols), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(npg):
        table[b, :n] = ids[at:at + n]
        at += n
    cache = R.make_cache(P, HKV, dev, seed)
    k, v = _edges(g, (B, T, HKV, 128)).to(dtype).to(dev), _edges(g, (B, T, HKV, 128)).to(dtype).to(dev)
    return cache, table, k, v


def _expect(before, table, pos, k, v):
    """The pools (numpy) after tokens k, v [B, T, HKV, 128] (64 bits; None: left as they are) at pos[b] + n."""
    pools = {n: x.copy() for n, x in before.items()}
    for name, x in (("k", k), ("v", v)):
        if x is None:
            continue
        code, byte = R.quantize(x)
        for b in range(x.shape[0]):
            for n in range(x.shape[1]):
                p = pos[b] + n
                if 0 <= p < 64 * table.shape[1] and 0 <= int(table[b, p // 64]) < before["k"].shape[0]:
                    R.write(pools, int(table[b, p // 64]), p % 64, name, code[b, n], byte[b, n])
    return pools


def _same_pools(cache, want):
    got = R.to_numpy(cache)
    for n in got:
        bad = np.argwhere(got[n] != want[n])
        assert bad.size == 0, f"{n}: {len(bad)} bytes differ, first at {bad[0]}"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("B,T,HKV,pos", [
    (1, 1, 1, [0]), (3, 1, 2, [63, 64, 5]),            # one token: the other half of its byte stays
    (2, 2, 1, [4, 7]), (2, 15, 3, [0, 50]),            # pairs that share bytes, and pairs that do not
    (2, 16, 2, [0, 61]), (1, 64, 2, [0]),              # a quarter of a page, a whole one
    (3, 65, 1, [63, 0, 31]), (2, 200, 2, [17, 64]),    # several pages, partly theirs
])
def test_append(gpu, dtype, B, T, HKV, pos):
    """Every byte of the pools: the new tokens' and those of all others, which stay; the values given back."""
    g = torch.Generator().manual_seed(13)
    cache, table, k, v = _append_case(g, B, T, HKV, TYPES[dtype], gpu, pos)
    before = R.to_numpy(cache)
    want = _expect(before, table, pos, _f64(k), _f64(v))
    p = torch.tensor(pos, dtype=torch.int32, device=gpu)
    kh, vh = cache.append(k, v, p, table.to(gpu), ragged=True, values=True)
    _same_pools(cache, want)
    assert kh.dtype == k.dtype and np.array_equal(_f64(kh), R.held(_f64(k)), equal_nan=True)
    assert np.array_equal(_f64(vh), R.held(_f64(v)), equal_nan=True)
    assert cache.append(k, v, p, table.to(gpu), ragged=True) is None  # again: the same
    _same_pools(cache, want)


def test_append_keys_alone_and_mixed_types(gpu):
    g = torch.Generator().manual_seed(17)
    cache, table, k, v = _append_case(g, 2, 21, 2, torch.float32, gpu, [3, 60])
    before, pos = R.to_numpy(cache), torch.tensor([3, 60], device=gpu)
    kh, vh = cache.append(k, None, pos, table.to(gpu), True, values=True)
    assert vh is None
    _same_pools(cache, _expect(before, table, [3, 60], _f64(k), None))
    kh, vh = cache.append(k.half(), v.bfloat16(), pos, table.to(gpu), True, values=True)
    _same_pools(cache, _expect(before, table, [3, 60], _f64(k.half()), _f64(v.bfloat16())))
    assert kh.dtype == vh.dtype == torch.float16
    assert np.array_equal(_f64(kh), R.held(_f64(k.half())), equal_nan=True)


@pytest.mark.parametrize("T", [3, 80])
def test_append_strides(gpu, T):
    """Views of a joined projection and heads before tokens store the same bytes."""
    g = torch.Generator().manual_seed(19)
    pos = torch.tensor([5, 62], dtype=torch.int32, device=gpu)
    cache, table, k, v = _append_case(g, 2, T, 2, torch.bfloat16, gpu, [5, 62])
    start = [t.clone() for t in cache.pools()]
    cache.append(k, v, pos, table.to(gpu), True)
    want = R.to_numpy(cache)
    joined = torch.zeros(2, T, 6, 128, dtype=k.dtype, device=gpu)
    joined[:, :, 2:4], joined[:, :, 4:] = k, v
    for kk, vv in ((joined[:, :, 2:4], joined[:, :, 4:]),
                   (k.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2))):
        for t, s in zip(cache.pools(), start):
            t.copy_(s)
        cache.append(kk, vv, pos.long(), table.long().to(gpu), True)
        _same_pools(cache, want)


@pytest.mark.parametrize("T", [1, 5, 70])
def test_append_outside_the_table(gpu, T):
    """check=False: tokens outside the table or on pages outside the pool are not written; the others are, and the values
    come back for all.  check=True refuses."""
    g = torch.Generator().manual_seed(23)
    pos = [62, 0, -3, 120]
    cache, table, k, v = _append_case(g, 4, T, 1, torch.float16, gpu, [62, 0, 0, 120])
    table = table[:, :2].clone()
    table[1, 0] = cache.P  # outside the pool
    before = R.to_numpy(cache)
    p = torch.tensor(pos, dtype=torch.int32, device=gpu)
    kh, vh = cache.append(k, v, p, table.to(gpu), values=True, check=False)
    _same_pools(cache, _expect(before, table, pos, _f64(k), _f64(v)))
    assert np.array_equal(_f64(kh), R.held(_f64(k)), equal_nan=True) and np.array_equal(_f64(vh), R.held(_f64(v)), equal_nan=True)
    with pytest.raises(ValueError):
        cache.append(k, v, p, table.to(gpu))
    with pytest.raises(ValueError):
        cache.append(k, v, p[:2], table.to(gpu))


def test_append_nothing(gpu):
    cache = R.make_cache(3, 2, gpu)
    before = R.to_numpy(cache)
    k = torch.zeros(2, 0, 2, 128, device=gpu)
    got = cache.append(k, k, torch.zeros(2, dtype=torch.int32, device=gpu), torch.zeros(2, 1, dtype=torch.int32, device=gpu), values=True)
    assert [x.shape for x in got] == [k.shape, k.shape]
    _same_pools(cache, before)


def _near_border(x, bound):
    """Blocks and elements of x [..., 128] (64 bits) that an error of `bound` could put on the other side of a border."""
    b, e = x.reshape(x.shape[:-1] + (4, 32)), bound.reshape(x.shape[:-1] + (4, 32))
    top, off = np.abs(b).max(-1), e.max(-1)
    _, byte = R.quantize(x)
    lo, up = (np.maximum(top - off, 0), top + off)
    edge = 7 * 2.0 ** (byte - 127.0)
    block = (up > edge) | (lo <= edge / 2) & (byte > R.LOW)
    s = 2.0 ** (byte[..., None] - 127.0)
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5])
    near = (np.abs(np.abs(b)[..., None] / s[..., None] - mids) <= (e / s)[..., None]).any(-1) | (np.abs(b) <= e)
    return block, (near | block[..., None]).reshape(x.shape)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("B,T,HQ,HKV,pos", [(3, 1, 8, 2, [0, 63, 100]), (2, 9, 3, 1, [60, 5]), (2, 150, 7, 1, [33, 64]), (1, 64, 0, 2, [0])])
def test_append_rotary(gpu, dtype, pairs, B, T, HQ, HKV, pos):
    g = torch.Generator().manual_seed(29)
    cache, table, k, v = _append_case(g, B, T, HKV, TYPES[dtype], gpu, pos)
    k = _rand(g, B, T, HKV, 128).to(k.dtype).to(gpu)
    q = _rand(g, B, T, HQ, 128).to(k.dtype).to(gpu) if HQ else None
    rope = AxisRope((16, 24, 24), device=gpu, pairs=pairs)
    where = torch.randint(0, 3000, (3, B, T), generator=g).to(gpu)
    p = torch.tensor(pos, dtype=torch.int32, device=gpu)
    qr, kh, vh = cache.append_rotary(q, k, v, p, table.to(gpu), rope, where, True, values=True)
    if HQ:
        _check_turned(qr, q, where, rope)
    turned = R.rotate(_f64(k), where.cpu().numpy(), rope.axis, rope.inv_freq, rope.adjacent)
    block, near = _near_border(turned, R.turn_bound(_f64(k), rope.adjacent))
    assert near.mean() < 0.01
    got = R.to_numpy(cache)
    code, byte = R.quantize(turned)
    for b in range(B):
        pages = [int(x) for x in table[b, :-(-(pos[b] + T) // 64)]]
        (kc, kb), (vc, vb) = R.codes_of(got, pages)
        kc, kb, vc, vb = (x[pos[b]:pos[b] + T] for x in (kc, kb, vc, vb))
        assert (kb == byte[b])[~block[b]].all() and (kc == code[b])[~near[b]].all()
        wc, wb = R.quantize(_f64(v[b]))
        assert (vc == wc).all() and (vb == wb).all()
        assert np.array_equal(_f64(kh[b]), R.values(kc, kb)) and np.array_equal(_f64(vh[b]), R.values(vc, vb), equal_nan=True)
    # positions by default: the token's own, on every axis
    default = cache.append_rotary(q, k, v, p, table.to(gpu), rope, None, True, values=True)
    own = (p[:, None] + torch.arange(T, device=gpu)).expand(3, B, T).contiguous()
    given = cache.append_rotary(q, k, v, p, table.to(gpu), rope, own, True, values=True)
    for a, b in zip(default, given):
        assert (a is None and b is None) or torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    assert cache.append_rotary(None, k, v, p, table.to(gpu), rope, own, True) is None


@pytest.mark.parametrize("dtype,pairs,B,T,HQ,HKV,pos", [
    ("bf16", "half", 2, 90, 900, 2, [33, 64]),     # a long prompt's kernel, at the size of its tiles' edges
    ("fp32", "adjacent", 1, 64, 2600, 1, [63]),    # a token in the first tile, 63 in the second
    ("fp16", "half", 1, 131, 1300, 3, [0]),
])
def test_append_rotary_of_many_heads(gpu, dtype, pairs, B, T, HQ, HKV, pos):
    test_append_rotary(gpu, dtype, pairs, B, T, HQ, HKV, pos)


def test_append_at_once_and_in_parts(gpu):
    """A prompt in one call, in pieces of several sizes, and the same without the turn: the same bytes and values."""
    g = torch.Generator().manual_seed(53)
    rope, T, pos = AxisRope((64,), device=gpu), 2300, [17, 128]
    cache, table, k, v = _append_case(g, 2, T, 8, torch.bfloat16, gpu, pos)
    q, table = _rand(g, 2, T, 24, 128).bfloat16().to(gpu), table.to(gpu)
    start = [t.clone() for t in cache.pools()]
    p = torch.tensor(pos, dtype=torch.int32, device=gpu)
    whole = cache.append_rotary(q, k, v, p, table, rope, None, True, values=True)
    want = R.to_numpy(cache)
    for cuts in ([1, 2, 66, 67, 130, 1000, 2300], [63, 64, 2299, 2300]):
        for t, s in zip(cache.pools(), start):
            t.copy_(s)
        got, at = [], 0
        for cut in cuts:
            got.append(cache.append_rotary(q[:, at:cut], k[:, at:cut], v[:, at:cut], p + at, table, rope, None, True, values=True))
            at = cut
        _same_pools(cache, want)
        for i in range(3):
            assert torch.equal(torch.cat([x[i] for x in got], 1).nan_to_num(7.0), whole[i].nan_to_num(7.0))
    for t, s in zip(cache.pools(), start):
        t.copy_(s)
    cache.append(k, v, p, table, True)
    want, at = R.to_numpy(cache), 0
    for t, s in zip(cache.pools(), start):
        t.copy_(s)
    for cut in (1, 2, 5, 70, 2300):
        cache.append(k[:, at:cut], v[:, at:cut], p + at, table, True)
        at = cut
    _same_pools(cache, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,T,HKV", [(70, 1, 4), (140, 3, 2), (300, 2, 1), (33, 31, 8)])
def test_append_of_many_sequences(gpu, dtype, B, T, HKV):
    g = torch.Generator().manual_seed(59)
    pos = [(37 * b) % 130 for b in range(B)]
    cache, table, k, v = _append_case(g, B, T, HKV, TYPES[dtype], gpu, pos)
    want = _expect(R.to_numpy(cache), table, pos, _f64(k), _f64(v))
    kh, vh = cache.append(k, v, torch.tensor(pos, dtype=torch.int32, device=gpu), table.to(gpu), ragged=True, values=True)
    _same_pools(cache, want)
    assert np.array_equal(_f64(kh), R.held(_f64(k)), equal_nan=True) and np.array_equal(_f64(vh), R.held(_f64(v)), equal_nan=True)


def test_append_rotary_refusals(gpu):
    cache, rope = R.make_cache(2, 1, gpu), AxisRope((64,), device=gpu)
    k, pos, table = torch.zeros(1, 2, 1, 128, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu), torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    for q in (k.half(), k[:, :1], k[..., :64], k[0]):
        with pytest.raises(ValueError):
            cache.append_rotary(q, k, k, pos, table, rope)
    with pytest.raises(ValueError):
        cache.append_rotary(k, k, k, pos, table, rope, torch.zeros(2, 1, 2, dtype=torch.int64, device=gpu))
    with pytest.raises(ValueError):
        cache.append_rotary(k, k, k, pos, table, AxisRope((64,), device="cpu"))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lens,HKV", [([1], 1), ([64, 0, 63], 3), ([200, 65], 2)])
def test_dequantize(gpu, dtype, lens, HKV):
    """All bytes that pages may hold, blocks of NaN among them; zeros past the lengths; bad pages read page 0."""
    g = torch.Generator().manual_seed(31)
    cols = max(-(-n // 64) for n in lens) + 1
    P = len(lens) * cols + 1
    cache = R.make_cache(P, HKV, gpu, seed=31)
    for s in (cache.k_scale, cache.v_scale):
        b = torch.randint(R.LOW, R.HIGH + 1, s.shape, generator=g)
        s.copy_(torch.where(torch.rand(s.shape, generator=g) < 0.02, 255, b))
    table = torch.randperm(P, generator=g)[:len(lens) * cols].view(len(lens), cols).to(torch.int32)
    sl = torch.tensor(lens, device=gpu)
    T = max(lens)
    k, v = cache.dequantize(table.to(gpu), T, sl, TYPES[dtype])
    assert k.shape == (len(lens), -(-T // 64) * 64, HKV, 128) and k.dtype == v.dtype == TYPES[dtype]
    for b, n in enumerate(lens):
        kk, vv = R.logical_kv(cache, table[b, :-(-T // 64)].tolist())
        for got, want in ((k, kk), (v, vv)):
            assert np.array_equal(_f64(got[b, :n]), want[:n], equal_nan=True) and (got[b, n:] == 0).all()
    k2, v2 = cache.dequantize(table.to(gpu), T, None, TYPES[dtype])
    assert all(torch.equal(k2[b, :n].nan_to_num(9.0), k[b, :n].nan_to_num(9.0)) for b, n in enumerate(lens))
    bad, good = table.clone(), table.clone()
    bad[0, 0], good[0, 0] = -1, 0
    for x, y in zip(cache.dequantize(bad.to(gpu), T, sl, TYPES[dtype]), cache.dequantize(good.to(gpu), T, sl, TYPES[dtype])):
        assert torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0))
    with pytest.raises(ValueError):
        cache.dequantize(table.to(gpu), 64 * cols + 1)
    assert cache.dequantize(table.to(gpu), 0)[0].shape == (len(lens), 0, HKV, 128)


# ---------------------------------------------------------------------------- attention
def _fill(cache, k, v, table_row, start=0):
    dev = cache.v.device
    cache.append(k[None].to(dev), v[None].to(dev), torch.tensor([start], dtype=torch.int32, device=dev), table_row[None].to(dev))


def _batch(lens, HQ, HKV, L, dtype, seed, dev):
    """A cache of sequences with pages in random order, and queries that look for some keys."""
    g = torch.Generator().manual_seed(seed)
    npg = [-(-n // 64) for n in lens]
    P = sum(npg) + 2
    ids = torch.randperm(P, generator=g)
    cache = R.make_cache(P, HKV, dev, seed=seed)
    table = torch.zeros((len(lens), max(npg) + 1), dtype=torch.int32)
    q = _rand(g, len(lens), L, HQ, 128).to(dtype)
    at = 0
    for b, n in enumerate(lens):
        table[b, :npg[b]] = ids[at:at + npg[b]]
        at += npg[b]
        if n == 0:
            continue
        k, v = _rand(g, n, HKV, 128), _rand(g, n, HKV, 128)
        for h in range(HKV):
            t = int(torch.randint(0, n, (1,), generator=g))
            x = q[b, -1, h * (HQ // HKV)].float()
            k[t, h] = 0.8 * x / x.norm() * math.sqrt(128) + 0.6 * k[t, h]
        _fill(cache, k, v, table[b])
    return cache, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), q.to(dev)


# attend_ref's bound counts a rounding of K to fp16, which mxfp4 keys do not need, and one of the weights (2^-11).  Where
# rows are few the weights times V's powers of two are the operand: the same 2^-11 but where they fall below fp16's normal
# numbers, and there steps of 2^-24 below weights of 2^8 and more: 2^-33 of the row's largest weight times V's largest
# power of two a token, which the bound's n 2^-25 2^-8 covers for V's of this size.
def _check(cache, table, lens, q, out, q_lens=None, scale=SCALE, tokens=None, slack=0.0):
    B, L = q.shape[:2]
    for b in range(B):
        n = int(lens[b])
        ql = L if q_lens is None else int(q_lens[b])
        if n == 0:
            assert (out[b] == 0).all()
            continue
        k, v = R.logical_kv(cache, table[b, :-(-n // 64)].tolist())
        o, bound = reference(q[b], k[:n], v[:n], n, ql, scale, tokens)
        rows = slice(None) if tokens is None else tokens
        assert_close(out[b][rows], o[rows], bound[rows] + slack, q.dtype, f"sequence {b}")


@pytest.mark.parametrize("lens,HQ,HKV,L", [
    ([1], 4, 4, 1),                      # one token
    ([1, 63, 64, 65, 0], 8, 2, 1),       # around a page, an empty sequence
    ([700, 255, 257], 32, 8, 1),         # several pages a wave
    ([130, 40], 14, 2, 3),               # groups of 7 rows, 21 rows: two tiles
    ([200, 5], 16, 1, 5),                # 80 rows: several row blocks; fewer keys than rows of a tile
    ([90, 64], 12, 4, 33),               # 99 rows of a chunk
    ([300], 48, 1, 1), ([65], 6, 6, 2),  # 48 rows of one head; one row a head
])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attend_lengths(gpu, lens, HQ, HKV, L, dtype):
    cache, table, sl, q = _batch(lens, HQ, HKV, L, TYPES[dtype], 3, gpu)
    _check(cache, table, lens, q, cache.attend(q, table, sl))


@pytest.mark.parametrize("B,HQ,HKV,L", [(65, 8, 2, 1), (70, 4, 1, 5), (130, 16, 4, 1), (700, 2, 1, 1)])
def test_attend_many_sequences(gpu, B, HQ, HKV, L):
    """More sequences than a wave has lanes, than half a round of workgroups and than a whole one; lengths from none to
    several page ranges, in no order."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 300, (B,), generator=g).tolist()
    lens[0], lens[B // 2], lens[63], lens[64] = 0, 3000, 64, 0
    lens[B - 1] = 1 if B % 2 else 2100
    cache, table, sl, q = _batch(lens, HQ, HKV, L, torch.bfloat16, 83, gpu)
    out = cache.attend(q, table, sl)
    some = sorted({0, B // 2, 62, 63, 64, B - 1} | set(range(1, B, 1 + B // 12)))
    _check(cache, table[some], [lens[b] for b in some], q[some], out[some])
    alone = torch.cat([cache.attend(q[b:b + 1], table[b:b + 1], sl[b:b + 1]) for b in range(B)])
    assert torch.allclose(alone.float(), out.float(), atol=2.0 ** -7, rtol=2.0 ** -7)
    assert torch.equal(cache.attend(q, table, torch.zeros_like(sl), T=100), torch.zeros_like(out))


def test_attend_long_and_scale(gpu):
    """Page ranges split over many workgroups; a scale of the caller's; T above every length."""
    lens = [9000, 4097]
    cache, table, sl, q = _batch(lens, 8, 2, 1, torch.float16, 7, gpu)
    table = torch.cat([table, torch.full((2, 300), -1, dtype=torch.int32, device=gpu)], 1)
    _check(cache, table, lens, q, cache.attend(q, table, sl, T=20000, scale=0.03), scale=0.03)


@pytest.mark.parametrize("L,HQ", [(1, 4), (6, 4), (40, 8)])
@pytest.mark.parametrize("scale", [-0.05, 0.0, 2.0])
def test_attend_other_scales(gpu, scale, L, HQ):
    cache, table, sl, q = _batch([150], HQ, 1, L, torch.float16, 73, gpu)
    _check(cache, table, [150], q, cache.attend(q, table, sl, scale=scale), scale=scale)


def test_attend_padded_batch(gpu):
    lens, ql = [130, 64, 2, 0], [5, 1, 5, 0]
    cache, table, sl, q = _batch(lens, 8, 2, 5, torch.bfloat16, 11, gpu)
    for b, n in enumerate(ql):
        q[b, n:] = float("nan")
    out = cache.attend(q, table, sl, q_lens=torch.tensor(ql, device=gpu))
    _check(cache, table, lens, q, out, q_lens=ql)
    assert (out[2, :3] == 0).all() and (out[2, 3:] != 0).any()
    assert (cache.attend(q, table, torch.zeros_like(sl), T=130) == 0).all()


def test_attend_large_queries(gpu):
    cache, table, sl, q = _batch([80], 8, 2, 1, torch.bfloat16, 17, gpu)
    for f in (2.0 ** 30, 2.0 ** -40):
        _check(cache, table, [80], q * f, cache.attend(q * f, table, sl, scale=SCALE / f), scale=SCALE / f)


@pytest.mark.parametrize("n,L,HQ,HKV", [
    (3300, 150, 8, 2),    # 600 rows over 52 pages: 256-row workgroups, split ranges
    (1500, 300, 32, 4),   # few pages, many rows: smaller workgroups, ranges not split
    (700, 100, 4, 4),     # 100 rows of each head: a workgroup's waves with two tiles, one and none
])
def test_attend_chunks(gpu, n, L, HQ, HKV):
    cache, table, sl, q = _batch([n], HQ, HKV, L, torch.float16, 67, gpu)
    out = cache.attend(q, table, sl)
    _check(cache, table, [n], q, out, tokens=sorted({0, 1, 63, L // 2, L - 64, L - 2, L - 1} & set(range(L))))
    for i in range(0, L, 7):  # every part of the chunk against the same rows as short chunks of their own
        part = cache.attend(q[:, i:i + 7].contiguous(), table, torch.tensor([n - L + min(i + 7, L)], device=gpu))
        assert torch.allclose(part.float(), out[:, i:i + 7].float(), atol=2.0 ** -8, rtol=2.0 ** -8)


@pytest.mark.parametrize("n,L,HQ", [(200, 70, 4), (200, 9, 16), (200, 5, 2), (200, 1, 4), (9000, 3, 4), (3300, 150, 4)])
@pytest.mark.parametrize("where", ["first", "last"])
def test_attend_nan_blocks(gpu, n, L, HQ, where):
    """A block of NaN in V counts in its 32 columns for the rows that see it and in no other; a key's for the whole row.
    Slots that hold no token yet are random bytes throughout."""
    cache, table, sl, q = _batch([n], HQ, 1, L, torch.float16, 13, gpu)
    at = n - 3 if where == "last" else 5  # the last 3 query tokens see it, or all
    sees = max(L - 3, 0) if where == "last" else 0
    k, v = torch.randn(1, 1, 128), torch.randn(1, 1, 128)
    v[0, 0, 40] = float("inf")
    _fill(cache, k, v, table[0], at)
    out = cache.attend(q, table, sl)[0].float()
    assert torch.isnan(out[sees:, :, 32:64]).all() and torch.isfinite(out[:sees]).all()
    assert torch.isfinite(out[..., :32]).all() and torch.isfinite(out[..., 64:]).all()
    some = sorted({0, L // 2, L - 1})
    _check(cache, table, [n], q, out.to(q.dtype)[None], tokens=some)
    k[0, 0, 3] = float("nan")
    v[0, 0, 40] = 1.0
    _fill(cache, k, v, table[0], at)
    out = cache.attend(q, table, sl)[0].float()
    assert torch.isnan(out[sees:]).all() and torch.isfinite(out[:sees]).all()


@pytest.mark.parametrize("n,L,HQ", [(300, 1, 4), (300, 5, 4), (300, 40, 4), (9000, 1, 4)])
@pytest.mark.parametrize("power", [13, 0, -10, -20])
def test_attend_sizes_of_values(gpu, n, L, HQ, power):
    """V's from the largest to the smallest that the format holds, and blocks far apart in one page."""
    g = torch.Generator().manual_seed(37)
    cache, table, sl, q = _batch([n], HQ, 1, L, torch.bfloat16, 37, gpu)
    v = _rand(g, n, 1, 128).clamp(-3, 3) * 2.0 ** power
    v[::3, :, 32:64] *= 2.0 ** -12
    v[1::5, :, 64:96] = 0
    v[2::7, :, 96:] *= 2.0 ** -3
    _fill(cache, _rand(g, n, 1, 128), v, table[0])
    out = cache.attend(q, table, sl)
    # steps below fp16's normal numbers: 2^-25 of weights 2^8 and more times V's largest power of two, a token; the level
    # is at most six and the weights' sum at least the largest
    steps = n * 2.0 ** -33 * 6 * 2.0 ** (power + 1)
    _check(cache, table, [n], q, out, tokens=sorted({0, L // 2, L - 1}), slack=steps)
    # one token whose values are 2^20 times the others', with a weight of next to nothing
    k, big = _rand(g, 1, 1, 128), _rand(g, 1, 1, 128).clamp(-2, 2) * 2.0 ** 13
    _fill(cache, -40 * torch.sign(q[0, 0, 0].float().cpu()).view(1, 1, 128), big, table[0], 3)
    out = cache.attend(q, table, sl)
    k, vv = R.logical_kv(cache, table[0, :-(-n // 64)].tolist())
    o, bound = reference(q[0], k[:n], vv[:n], n, L, SCALE, [0])
    # the fp16 operand's steps are now 2^-33 of 2^13
    assert_close(out[0][[0]], o[[0]], bound[[0]] + n * 2.0 ** -33 * 6 * 2.0 ** 13, q.dtype)


@pytest.mark.parametrize("n,L,HQ", [(2000, 1, 4), (2000, 4, 8), (2000, 40, 1), (2000, 30, 4), (9000, 1, 8), (3300, 150, 4)])
def test_attend_constant_values(gpu, n, L, HQ):
    """V of ones gives ones, whatever the weights round to: the sum below the fraction bar is that of the weights that are
    multiplied.  (Both sums are chains of at most 52 pages x 32 fp32 additions, off by 52 x 32 x 2^-24 < 2^-13 each; half a
    step of fp16 below 1 is 2^-12.)"""
    g = torch.Generator().manual_seed(101)
    cache, table, sl, _ = _batch([n], HQ, 1, 1, torch.float16, 101, gpu)
    u = torch.sign(_rand(g, 128))
    k = (-u).repeat(n, 1, 1)
    k[3::64] = u
    _fill(cache, k, torch.ones(n, 1, 128), table[0])
    q = u.expand(1, L, HQ, 128).half().contiguous().to(gpu)
    for step in range(24):
        out = cache.attend(q, table, sl, scale=(2 + step / 12) * math.log(2) / 256)
        assert (out == 1).all(), (step, out.float().min(), out.float().max())


@pytest.mark.parametrize("depth", [20, 25, 27, 30])
@pytest.mark.parametrize("n,L,HQ", [(2000, 1, 4), (2000, 4, 8), (2000, 30, 4), (9000, 1, 8), (3300, 150, 4)])
def test_attend_many_small_weights(gpu, depth, n, L, HQ):
    """Keys far below the largest score, which together weigh something: their weights are not lost below fp16's steps."""
    g = torch.Generator().manual_seed(103)
    cache, table, sl, _ = _batch([n], HQ, 1, 1, torch.float16, 103, gpu)
    u = torch.sign(_rand(g, 128))
    k, vv = (-u).repeat(n, 1, 1), torch.ones(n, 1, 128)
    k[3], vv[3] = u, 0
    _fill(cache, k, vv, table[0])
    q = u.expand(1, L, HQ, 128).half().contiguous().to(gpu)
    scale = depth * math.log(2) / 256
    out = cache.attend(q, table, sl, scale=scale)
    _check(cache, table, [n], q, out, scale=scale, tokens=sorted({0, L // 2, L - 1}))


# Where sequences and KV heads leave CUs idle their rows go by sixteens to as many workgroups.  The same cases beside so many
# copies of their sequences that the kernels for 17 to 256 rows take them.
@pytest.mark.parametrize("copies,case", [
    (300, (test_attend_lengths, [130, 40], 14, 2, 3, "fp16")),       # 21 rows, ranges not split
    (200, (test_attend_lengths, [2600, 1700, 0], 20, 4, 5, "bf16")),  # 25 rows, even ranges of a ragged batch
    (300, (test_attend_lengths, [200, 5], 16, 1, 5, "bf16")),        # 80 rows
    (300, (test_attend_lengths, [300], 48, 1, 1, "fp16")),           # 48 rows
    (40, (test_attend_lengths, [2600, 1700, 0, 3100], 16, 2, 6, "bf16")),   # 48 rows, even ranges
    (30, (test_attend_lengths, [3100, 0, 1700, 2600], 16, 2, 14, "fp16")),  # 112 rows
    (12, (test_attend_lengths, [64, 1700, 3100, 2600], 16, 2, 30, "bf16")),  # 240 rows
    (25, (test_attend_nan_blocks, 9000, 10, 4, "first")), (25, (test_attend_nan_blocks, 9000, 10, 4, "last")),
    (300, (test_attend_padded_batch,)), (300, (test_attend_large_queries,)),
    (300, (test_attend_other_scales, -0.05, 6, 4)), (300, (test_attend_other_scales, 0.0, 40, 8)),
    (300, (test_attend_other_scales, -0.05, 40, 8)), (300, (test_attend_other_scales, 2.0, 40, 8)),
    (100, (test_attend_chunks, 3300, 150, 8, 2)), (20, (test_attend_chunks, 1500, 300, 32, 4)),
    (300, (test_attend_chunks, 700, 100, 4, 4)), (150, (test_attend_chunks, 3300, 71, 2, 2)),
    *[(n, (test_attend_nan_blocks, *x, where)) for where in ("first", "last")
      for n, x in ((200, (200, 70, 4)), (300, (200, 9, 16)), (300, (200, 5, 4)), (150, (9000, 5, 4)), (300, (200, 10, 4)),
                   (150, (4000, 15, 4)), (100, (3300, 150, 4)))],
    *[(300, (test_attend_sizes_of_values, n, L, 4, power)) for power in (13, 0, -20) for n, L in ((300, 5), (300, 40), (4000, 6))],
    *[(300, (test_attend_constant_values, *x)) for x in ((2000, 4, 8), (2000, 40, 1), (2000, 30, 4))],
    (100, (test_attend_constant_values, 3300, 150, 4)),
    *[(n, (test_attend_many_small_weights, depth, *x)) for depth in (20, 30)
      for n, x in ((300, (2000, 4, 8)), (300, (2000, 30, 4)), (100, (3300, 150, 4)))],
])
def test_attend_among_copies(gpu, monkeypatch, copies, case):
    attend = PagedMXFP4Cache.attend

    def crowded(self, q, table, lens=None, *, q_lens=None, **kw):
        got = attend(self, *(t.repeat(copies, *[1] * (t.ndim - 1)) for t in (q, table, lens)),
                     q_lens=None if q_lens is None else q_lens.repeat(copies), **kw)
        got = got.view(copies, *q.shape)
        # copies differ by where their ranges end: by each's bound, far below a step and a half of the type
        assert torch.allclose(got[0].float(), got[-1].float(), rtol=2.0 ** -6, atol=2.0 ** -6 * float(got[0].float().nan_to_num(0).abs().max()),
                              equal_nan=True)
        return got[copies // 2]

    monkeypatch.setattr(PagedMXFP4Cache, "attend", crowded)
    case[0](gpu, *case[1:])


@pytest.mark.parametrize("lens,L,HQ,HKV", [([1000, 990], 990, 16, 4), ([1500], 1500, 16, 4), ([400, 700, 650, 64], 600, 8, 2)])
def test_attend_prompts(gpu, lens, L, HQ, HKV):
    """Prompts of many workgroups, two a CU: every row of every block is written, with the right keys (padded ones zeros)."""
    cache, table, sl, q = _batch(lens, HQ, HKV, L, torch.bfloat16, 89, gpu)
    ql = [min(n, L) for n in lens]
    out = cache.attend(q, table, sl, q_lens=torch.tensor(ql, device=gpu))
    for b, n in enumerate(ql):
        assert (out[b, n:] == 0).all() and (out[b, :n] != 0).any(-1).all()
        rows = sorted({0, 1, 63, 64, 127, n // 2, n - 65, n - 1} & set(range(n)))
        k, v = R.logical_kv(cache, table[b, :-(-lens[b] // 64)].tolist())
        o, bound = reference(q[b], k[:lens[b]], v[:lens[b]], lens[b], n, SCALE, rows)
        assert_close(out[b][rows], o[rows], bound[rows], q.dtype, f"sequence {b}")
        for i in range(0, n, 97):  # against short chunks of their own
            m = min(i + 6, n)
            part = cache.attend(q[b:b + 1, i:m].contiguous(), table[b:b + 1], torch.tensor([lens[b] - n + m], device=gpu))
            assert torch.allclose(part[0].float(), out[b, i:m].float(), atol=2.0 ** -6, rtol=2.0 ** -7)


@pytest.mark.parametrize("L,HQ", [(1, 4), (3, 16), (6, 16), (14, 16), (31, 16)])
def test_attend_padded_ragged_batches(gpu, L, HQ):
    """Sequences of none to 52 pages with none to all of L query tokens, in kernels for 2 to 248 rows."""
    g = torch.Generator().manual_seed(L)
    B = 60 if L < 14 else 24
    lens = torch.randint(0, 3300, (B,), generator=g).tolist()
    lens[3], lens[-1], lens[7] = 3300, 0, 2
    ql = [min(int(x), n) for x, n in zip(torch.randint(0, L + 1, (B,), generator=g), lens)]
    cache, table, sl, q = _batch(lens, HQ, 2, L, torch.bfloat16, 97, gpu)
    for b, n in enumerate(ql):
        q[b, n:] = float("nan")
    out = cache.attend(q, table, sl, q_lens=torch.tensor(ql, device=gpu))
    for b in range(B):
        assert (out[b, ql[b]:] == 0).all()
        assert torch.isfinite(out[b]).all()
    some = [b for b in range(0, B, 5) if ql[b]]
    for b in some:
        rows = sorted({0, ql[b] // 2, ql[b] - 1})
        k, v = R.logical_kv(cache, table[b, :-(-lens[b] // 64)].tolist())
        o, bound = reference(q[b], k[:lens[b]], v[:lens[b]], lens[b], ql[b], SCALE, rows)
        assert_close(out[b][rows], o[rows], bound[rows], q.dtype, f"sequence {b}")


def _forked(sizes, prefix, own, HQ, HKV, L, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    lens, b = [], 0
    for n, p in zip(sizes, prefix):
        lens += [p + x for x in own[b:b + n]]
        b += n
    P = sum(-(-x // 64) + 1 for x in lens) + sum(-(-p // 64) for p in prefix)
    ids = torch.randperm(P, generator=g).tolist()
    cache = R.make_cache(P, HKV, dev, seed=seed)
    table = torch.full((len(lens), max(-(-x // 64) for x in lens) + 2), -1, dtype=torch.int32)
    b = 0
    for n, p in zip(sizes, prefix):
        sp = p // 64
        shared = [ids.pop() for _ in range(sp)]
        kp, vp = _rand(g, p, HKV, 128), _rand(g, p, HKV, 128)
        for i in range(b, b + n):
            table[i, :sp] = torch.tensor(shared, dtype=torch.int32)
            for j in range(sp, -(-lens[i] // 64)):
                table[i, j] = ids.pop()
            if lens[i]:
                k, v = torch.cat([kp, _rand(g, own[i], HKV, 128)]), torch.cat([vp, _rand(g, own[i], HKV, 128)])
                dev_row = table[i][None].to(dev)
                cache.append(k[None].to(dev), v[None].to(dev), torch.zeros(1, dtype=torch.int32, device=dev), dev_row, True)
        b += n
    q = _rand(g, len(lens), L, HQ, 128).to(dtype)
    return cache, table.to(dev), lens, torch.tensor(lens, dtype=torch.int32, device=dev), q.to(dev)


@pytest.mark.parametrize("sizes,prefix,HQ,HKV,L,step", [
    ([4], [200], 8, 2, 1, 37),                     # a partial page at the prefix's end, 16 rows
    ([3, 1, 5], [640, 100, 64], 8, 2, 1, 37),      # a group of one, a prefix of one page
    ([2, 9], [63, 130], 16, 2, 1, 37),             # a prefix below a page, 72 rows
    ([6], [3000], 14, 2, 3, 37),                   # groups of 7 rows, 126 rows, three drafted tokens
    ([40], [700], 8, 1, 1, 211),                   # 320 rows, and own parts of several pages: both kinds in one launch
    ([17, 3, 30], [900, 64, 320], 16, 2, 3, 211),  # the same with uneven groups and 24 own rows
])
def test_attend_shared_prefix(gpu, sizes, prefix, HQ, HKV, L, step):
    B = sum(sizes)
    own = [(step * b) % (4 * step) + L for b in range(B)]
    cache, table, lens, sl, q = _forked(sizes, prefix, own, HQ, HKV, L, torch.bfloat16, 23, gpu)
    plan = SharedPrefix(table, sl, group_sizes=sizes)
    assert plan.pages == [p // 64 if n > 1 else 0 for n, p in zip(sizes, prefix)]
    out = cache.attend(q, table, sl, shared=plan)
    some = list(range(0, B, 1 if B < 12 else 5))
    _check(cache, table[some], [lens[b] for b in some], q[some], out[some])
    for other in (cache.attend(q, table, sl), cache.attend(q, table, sl, T=64 * table.shape[1], shared=plan)):
        assert torch.allclose(out.float(), other.float(), atol=2.0 ** -6, rtol=2.0 ** -7)


def test_attend_shapes_streams_and_repeats(gpu):
    lens = [1000, 300]
    cache, table, sl, q = _batch(lens, 8, 2, 1, torch.bfloat16, 41, gpu)
    want = cache.attend(q, table, sl, T=1000)
    for _ in range(3):
        assert torch.equal(want, cache.attend(q, table, sl, T=1000))
    wide = torch.zeros((2, 8, 256), dtype=q.dtype, device=gpu)
    wide[..., :128] = q[:, 0]
    got = cache.attend(wide[..., :128], table.long(), sl.long())
    assert got.shape == (2, 8, 128) and torch.equal(got, want[:, 0])
    buf = torch.empty_like(got)
    assert cache.attend(q[:, 0], table, sl, out=buf) is buf and torch.equal(buf, got)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = cache.attend(q, table, sl, T=1000)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want, got)
    for bad in (dict(T=10 ** 6), dict(out=buf), dict(shared=SharedPrefix(table.repeat(2, 1), sl.repeat(2)))):
        with pytest.raises(ValueError):
            cache.attend(q, table, sl, **bad)
    with pytest.raises(NotImplementedError):
        cache.attend(q.float(), table, sl)


def test_attend_two_streams_and_two_graphs(gpu):
    """Calls that overlap on two streams, and two captured calls replayed in turn, do not share partials."""
    sets = [_batch([4000, 900], 8, 2, 1, torch.bfloat16, 83 + i, gpu) for i in range(2)]
    want = [c.attend(q, t, sl, T=4000) for c, t, sl, q in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (c, t, sl, q) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                outs[i].append(c.attend(q, t, sl, T=4000))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])
    graphs, caught = [], []
    for c, t, sl, q in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            caught.append(c.attend(q, t, sl, T=4000))
        graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for o in caught:
            o.zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(caught[0], want[0]) and torch.equal(caught[1], want[1])


# ---------------------------------------------------------------------------- together
def test_a_layer_from_prompt_to_samples(gpu):
    """A prompt in two chunks, forked into samples, decoded, compacted: every step's attention against the held values that
    the appends gave back, in 64 bits."""
    g = torch.Generator().manual_seed(43)
    HQ, HKV, dt = 8, 2, torch.bfloat16
    cache = R.make_cache(40, HKV, gpu, seed=43)
    pool = PagePool([cache])
    rope = AxisRope((16, 24, 24), device=gpu)
    table = torch.full((2, 8), -1, dtype=torch.int32, device=gpu)
    lens = torch.zeros(2, dtype=torch.int32, device=gpu)
    held = [[torch.zeros(0, HKV, 128)] * 2 for _ in range(2)]  # k, v of each sequence

    def step(n):
        nonlocal lens
        B = table.shape[0]
        q, k, v = (_rand(g, B, n, H, 128).to(dt).to(gpu) for H in (HQ, HKV, HKV))
        where = torch.stack([lens[:, None] + torch.arange(n, device=gpu)] * 3) + torch.tensor([0, 5, 9], device=gpu)[:, None, None]
        pool.extend(table, lens, n)
        qr, kh, vh = cache.append_rotary(q, k, v, lens, table, rope, where, True, values=True)
        _check_turned(qr, q, where, rope)
        lens = lens + n
        out = cache.attend(qr, table, lens)
        for b in range(B):
            held[b] = [torch.cat([x, y[b].float().cpu()]) for x, y in zip(held[b], (kh, vh))]
            kk, vv = (x.double().numpy() for x in held[b])
            o, bound = reference(qr[b], kk, vv, len(kk), n, SCALE)
            assert_close(out[b], o, bound, dt, f"sequence {b}")
        return out

    step(130)
    step(37)
    parents = torch.tensor([0, 1, 1, 0, 1], device=gpu)
    child = pool.fork(table, lens, parents)
    pool.free(table, lens)
    table, lens = child, lens[parents]
    held = [list(held[p]) for p in parents.tolist()]
    for _ in range(3):
        step(1)
    assert pool.compact(table) == int((pool.refs > 0).sum())
    step(1)
    step(30)
    k, v = cache.dequantize(table, int(lens.max()), lens, dt)
    for b in range(5):
        n = int(lens[b])
        assert torch.equal(k[b, :n].float().cpu(), held[b][0]) and torch.equal(v[b, :n].float().cpu(), held[b][1])


def test_a_captured_decode_step(gpu):
    """Turn, store and attend in one graph, replayed with new inputs and grown lengths, eager work between: every replay
    equals the eager step."""
    g = torch.Generator().manual_seed(47)
    cache, table, sl, _ = _batch([100, 63, 129], 8, 2, 1, torch.bfloat16, 47, gpu)
    table = torch.cat([table, torch.zeros_like(table)], 1)
    other = R.make_cache(cache.P, 2, gpu)
    for a, b in zip(other.pools(), cache.pools()):
        a.copy_(b)
    rope = AxisRope((24, 20, 20), device=gpu, order="cycled")
    q, k, v = (torch.empty(3, 1, H, 128, dtype=torch.bfloat16, device=gpu) for H in (8, 2, 2))

    def step(c):
        qr = c.append_rotary(q, k, v, sl, table, rope, check=False)
        return qr, c.attend(qr, table, sl + 1, T=192)

    def inputs():
        for x in (q, k, v):
            x.copy_(_rand(g, *x.shape))

    inputs()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(cache)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, out = step(cache)
    for i in range(4):
        inputs()
        graph.replay()
        torch.cuda.synchronize()
        want_q, want = step(other)
        assert torch.equal(qr, want_q) and torch.equal(out, want)
        for a, b in zip(cache.pools(), other.pools()):
            assert torch.equal(a, b)
        sl += 1


@pytest.mark.parametrize("L", [1, 5, 12])
def test_a_captured_step_of_growing_ranges(gpu, L):
    """Attention captured at a capacity, replayed with lengths that move the page ranges, between none and all of it."""
    full = [2600, 700, 6000] * 25
    cache, table, sl, q = _batch(full[:3], 16, 2, L, torch.float16, 101, gpu)
    table, q, sl = table.repeat(25, 1), q.repeat(25, 1, 1, 1), torch.zeros(75, dtype=torch.int32, device=gpu)
    run = lambda: cache.attend(q, table, sl, T=6000)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    g = torch.Generator().manual_seed(103)
    for share in (0.0, 0.01, 0.4, 1.0, 0.7):
        lens = [int(n * share) if share in (0.0, 1.0) else int(torch.randint(0, int(n * share) + 1, (1,), generator=g)) for n in full]
        sl.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run())
        some = [b for b in (0, 1, 2, 36, 74) if lens[b] >= L]
        for b in some:
            _check(cache, table[b:b + 1], [lens[b]], q[b:b + 1], out[b:b + 1], tokens=sorted({0, L - 1}))


def test_long_offsets(gpu):
    """A pool whose offsets pass 32 bits: its last pages are written and read like its first."""
    HKV = 64
    P = 2 ** 32 // (HKV * 4096) + 40  # K codes of more than 4 GiB
    cache = PagedMXFP4Cache(P, HKV, gpu)
    g = torch.Generator().manual_seed(53)
    low, high = torch.tensor([[1, 2, 3]], dtype=torch.int32, device=gpu), torch.tensor([[P - 1, P - 5, P - 2]], dtype=torch.int32, device=gpu)
    k, v = _rand(g, 1, 150, HKV, 128).half().to(gpu), _rand(g, 1, 150, HKV, 128).half().to(gpu)
    z = torch.zeros(1, dtype=torch.int32, device=gpu)
    for t in (low, high):
        cache.append(k, v, z, t)
        cache.append(k[:, :1], v[:, 1:2], z + 150, t)
    a, b = cache.dequantize(low, 151, z + 151), cache.dequantize(high, 151, z + 151)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and (a[0] != 0).any()
    for L in (1, 40):
        q = _rand(g, 1, L, HKV, 128).half().to(gpu)
        assert torch.equal(cache.attend(q, low, z + 151), cache.attend(q, high, z + 151))
