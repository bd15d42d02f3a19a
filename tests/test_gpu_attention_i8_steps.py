"""Decode attention over 8-bit values whose steps differ by many powers of two, large steps at positions of next to no weight among them."""
import math

import pytest
import torch

from test_gpu_cache_i8 import DEV, HALF

pytestmark = pytest.mark.gpu


def attention(q, cache, n, scale):
    """One sequence's n positions in float64, and what the kernel's arithmetic may be off by.  q [nq, d].  Half a step of a position's values is what 8 bits cannot tell
    apart; what is asked for here is 2^-27 of that of the position that counts most, for each position, and rounding."""
    nq, d = q.shape
    kc, vc, ks, vs = (c[0, :, :n].double() for c in cache)
    rep = nq // kc.shape[0]
    kc, vc, ks, vs = (c.repeat_interleave(rep, 0) for c in (kc, vc, ks, vs))
    q = q.double()
    s = torch.einsum("hd,htd->ht", q, kc) * ks * scale
    p = torch.softmax(s, -1)
    # a score: q in steps of 2^-23 of its largest, three roundings; exp2 2^-22
    off = abs(scale) * ks * 2.0 ** -24 * q.abs().amax(-1, keepdim=True) * kc.abs().sum(-1) + 2.0 ** -22 * s.abs() + 2.0 ** -22
    w = p * vs
    out, size = torch.einsum("ht,htd->hd", w, vc), torch.einsum("ht,htd->hd", w, vc.abs())
    tol = torch.einsum("ht,htd->hd", w * off, vc.abs()) + out.abs() * (p * off).sum(-1, keepdim=True)
    # p * step as two f16 numbers: 2^-21; what is below them: the largest p * step is at least 2^3 of the range, f16 ends
    # at 2^-24, so half of that is 2^-28 of the largest for each position; fp32 sums in any order
    tol += size * (2.0 ** -21 + 2.0 ** -23 * (n / 64 + 200)) + n * 2.0 ** -28 * 127 * w.amax(-1, keepdim=True)
    # fp32 powers of two end at 2^-126, taken relative to at most 2^9 times the largest: a weight below 2^-117 of that, give or take a score's error, may be 0
    tol += (w * (p < 2.0 ** -116 * p.amax(-1, keepdim=True))).sum(-1, keepdim=True) * 127
    return out, tol


def compare(wf, q, cache, scale=None):
    b, nkv, t, d = cache.k.shape
    nq = q.shape[1] // d
    scale = d ** -0.5 if scale is None else scale
    got = wf.ops.attn_decode_i8(q, cache, scale=scale).view(nq, d).double()
    want, tol = attention(q.view(nq, d), cache, t, scale)
    tol = tol + HALF[q.dtype] * want.abs() + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


def ordinary(wf, g, nkv, t, d):
    codes = [torch.randint(-127, 128, (1, nkv, t, d), generator=g, device=DEV, dtype=torch.int8) for _ in range(2)]
    return wf.KVCacheI8(*codes, *(torch.rand(1, nkv, t, generator=g, device=DEV) * 0.02 + 0.01 for _ in range(2)))


@pytest.mark.parametrize("d,nq,nkv,dt", [(64, 4, 2, torch.bfloat16), (128, 8, 1, torch.float16), (128, 16, 1, torch.bfloat16), (64, 12, 1, torch.float16)])
@pytest.mark.parametrize("t,where", [(200, 0), (200, 199), (200, 77), (64, 63), (17, 3), (3000, 1500), (3000, 2999)])
def test_a_large_step_without_weight(wf, d, nq, nkv, dt, t, where):
    """The others' values stay what they are, whatever power of two the one position's step is ahead of theirs."""
    g = torch.Generator(device=DEV).manual_seed(t + where)
    cache = ordinary(wf, g, nkv, t, d)
    q = torch.randn(1, nq * d, generator=g, device=DEV)
    q.view(nq, d)[:, 0] = 8.0
    q = q.to(dt)
    cache.k[:, :, where] = 0
    cache.k[:, :, where, 0] = -127
    for power in (12, 20, 24, 28, 40, 80, 120):
        # its weight: 2^-(power + 8) of an ordinary one's, so that it counts for nothing although its values are large
        cache.k_scale[:, :, where] = (power + 8) * math.log(2) / (8.0 * 127 * d ** -0.5)
        cache.v_scale[:, :, where] = 2.0 ** power * 0.01
        compare(wf, q, cache)


@pytest.mark.parametrize("order", ["rising", "falling", "any"])
@pytest.mark.parametrize("d,nq,nkv,t", [(64, 8, 1, 256), (128, 4, 1, 1000), (128, 16, 1, 500), (64, 40, 2, 130), (128, 32, 8, 4000)])
def test_steps_as_far_apart_as_the_weights(wf, d, nq, nkv, t, order):
    """Every position counts for about as much, with weights that span 2^100; other heads of the group see the same steps with other weights."""
    g = torch.Generator(device=DEV).manual_seed(t)
    cache = ordinary(wf, g, nkv, t, d)
    first = torch.linspace(-127, 127, t).round()
    if order == "falling":
        first = first.flip(0)
    elif order == "any":
        first = first[torch.randperm(t, generator=torch.Generator().manual_seed(t))]
    cache.k[..., 0] = first.to(torch.int8).to(DEV)
    cache.k_scale.fill_(0.01)
    far = 50 * math.log(2) / (127 * 0.01 * d ** -0.5)  # a query's first element that makes the scores span 2^100
    steps = torch.exp2(-first * (50 / 127)).to(DEV)
    cache.v_scale.mul_(steps)
    q = torch.randn(1, nq * d, generator=g, device=DEV)
    q.view(nq, d)[:, 0] = far
    q.view(nq, d)[1::3, 0] = 0.0
    q.view(nq, d)[2::3, 0] = -far / 2
    compare(wf, q.bfloat16(), cache)


@pytest.mark.parametrize("least", [2.0 ** -107, 2.0 ** -119, 1e-30, 1e30, 2.0 ** 120])
def test_steps_next_to_nothing_and_next_to_everything(wf, least):
    g = torch.Generator(device=DEV).manual_seed(5)
    cache = ordinary(wf, g, 2, 300, 64)
    q = torch.randn(1, 8 * 64, generator=g, device=DEV).bfloat16()
    cache.v_scale.mul_(least)
    cache.v_scale.mul_(100 if least < 1 else 1)
    compare(wf, q, cache)
    cache.v_scale[:, :, ::2] = 0
    compare(wf, q, cache)
    cache.v_scale.zero_()
    assert not wf.ops.attn_decode_i8(q, cache).any()
