"""What the operators on an 8-bit cache take for rows, heads and tables, and what they refuse."""
import pytest
import torch

from test_gpu_cache_i8 import DEV, a_cache, tables

pytestmark = pytest.mark.gpu
B, S, NQ, NKV, D, T = 2, 3, 8, 2, 64, 16


def setup(wf, s, b=B):
    g = torch.Generator(device=DEV).manual_seed(s)
    q, k, v = (torch.randn(b * s, n * D, generator=g, device=DEV).bfloat16() for n in (NQ, NKV, NKV))
    return q, k, v, *tables(T, D), torch.full((b,), 4, device=DEV), a_cache(wf, g, b, NKV, T, D)


def copies(cache):
    return cache._make(c.clone() for c in cache)


@pytest.mark.parametrize("s", [1, S])
def test_rows_in_any_number_of_dimensions(wf, s):
    q, k, v, cos, sin, pos, cache = setup(wf, s)
    one, two = copies(cache), copies(cache)
    want = wf.ops.rope_kv_i8_(q.clone(), k, v, cos, sin, pos, one, s)
    for shape in ((B, s, -1, D), (B * s, -1, D), (B, s, -1)):
        got = wf.ops.rope_kv_i8_(q.clone().view(shape), k.view(shape), v.view(shape), cos, sin, pos, two, s)
        assert torch.equal(got.view_as(want), want) and all(torch.equal(a, b) for a, b in zip(one, two))
    long = tables(T + 5, D)  # longer tables
    got = wf.ops.rope_kv_i8_(q.clone(), k, v, *long, pos, two, s)
    assert torch.equal(got, want)
    if s == 1:
        want = wf.ops.attn_decode_i8(want, one, pos)
        for shape in ((B, NQ, D), (B, 1, NQ, D), (B, 1, NQ * D), (B, NKV, NQ // NKV, D)):
            assert torch.equal(wf.ops.attn_decode_i8(got.view(shape), one, pos), want)
        alone = wf.KVCacheI8(*(c[:1] for c in one))
        assert torch.allclose(wf.ops.attn_decode_i8(got[0], alone, pos[0]).float(), want[:1].float(), rtol=2.0 ** -7, atol=1e-6)  # divided among the CTAs differently: both roundings


def test_other_numbers_of_rows_are_not_taken_for_heads(wf):
    q, k, v, cos, sin, pos, cache = setup(wf, S)
    before = copies(cache)
    q1, k1, v1 = q[:B], k[:B], v[:B]

    def rope(q=q1, k=k1, v=v1, cos=cos, sin=sin, pos=pos, cache=cache, s=1, **kw):
        return lambda: wf.ops.rope_kv_i8_(q, k, v, cos, sin, pos, cache, s, **kw)

    def attend(q=q1, cache=cache, pos=pos):
        return lambda: wf.ops.attn_decode_i8(q, cache, pos)

    first = wf.KVCacheI8(*(c[:1] for c in cache))
    wide = torch.zeros(B, 2 * NKV * D, dtype=torch.bfloat16, device=DEV)
    for bad in (rope(q, k, v), rope(q[:S], k[:S], v[:S], pos=pos[:1], cache=first), rope(q=q[:3]), rope(k=k[:3]), rope(v=v[:3]), rope(k=wide, v=wide), rope(q=q1[:, :-2].contiguous()),
                rope(q.view(B, S, NQ, D), k.view(B, S, NKV, D), v.view(B, S, NKV, D)), rope(q, k, v, s=S - 1), rope(out=q[:3].clone()),
                rope(cos=cos.repeat(1, 2)), rope(sin=sin.repeat(1, 2)), rope(cos=cos.flatten()), rope(cos=cos[:-1]), rope(s=1 << 62),
                attend(q), attend(q[:3]), attend(q[:2], first, pos[:1]), attend(q[:2].view(2, NQ, D), first, pos[:1]), attend(q1[:, :-2].contiguous()), attend(q.view(B, S, NQ * D)),
                attend(torch.zeros((), dtype=torch.bfloat16, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    assert all(torch.equal(a, b) for a, b in zip(cache, before))


def test_outputs_beside_the_inputs(wf):
    """Rotated queries between the columns of one tensor with q, k and v; an output that shares rows with them in any other way is refused."""
    q, k, v, cos, sin, pos, cache = setup(wf, S)
    two = copies(cache)
    want = wf.ops.rope_kv_i8_(q, k, v, cos, sin, pos, cache, S, out=torch.empty_like(q))
    n, m = NQ * D, NKV * D
    room = torch.zeros(B * S + 1, 2 * (n + m) + 8, dtype=torch.bfloat16, device=DEV)
    cols = [room[:B * S, a:a + w] for a, w in ((0, n), (n, m), (n + m, m), (n + 2 * m, n))]
    for c, x in zip(cols, (q, k, v)):
        c.copy_(x)
    assert torch.equal(wf.ops.rope_kv_i8_(*cols[:3], cos, sin, pos, two, S, out=cols[3]), want) and torch.equal(cols[0], q)
    assert all(torch.equal(a, b) for a, b in zip(cache, two))
    flat = torch.zeros(4 * B * S * n, dtype=torch.bfloat16, device=DEV)
    for q2, out in ((cols[0], room[1:, :n]), (cols[0], room[:B * S, 8:8 + n]), (cols[3], room[:B * S, n:2 * n]), (flat[:q.numel()].view_as(q), flat[D:D + q.numel()].view_as(q))):
        with pytest.raises(RuntimeError, match="share"):
            wf.ops.rope_kv_i8_(q2, *cols[1:3], cos, sin, pos, two, S, out=out)
    got = wf.ops.rope_kv_i8_(flat[:q.numel()].view_as(q).copy_(q), k, v, cos, sin, pos, two, S, out=flat[q.numel():2 * q.numel()].view_as(q))  # one behind the other
    assert torch.equal(got, want)


def test_workspaces_of_streams_that_are_not_torchs_own(wf):
    """Nothing is kept for them beyond the call: their handles do not say which stream it is."""
    q, k, v, cos, sin, pos, cache = setup(wf, 1)
    want, own = wf.ops.attn_decode_i8(q, cache, pos), torch.cuda.Stream()
    foreign = torch.cuda.ExternalStream(torch.cuda.Stream().cuda_stream)
    torch.cuda.synchronize()

    def kept(stream):
        before = torch.cuda.memory_allocated()
        with torch.cuda.stream(stream):
            for _ in range(3):
                got = wf.ops.attn_decode_i8(q, cache, pos)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del got
        return torch.cuda.memory_allocated() - before

    kept(own)
    assert kept(own) == 0  # the one that is kept
    assert kept(foreign) == 0
    with torch.cuda.stream(torch.cuda.ExternalStream(2)):  # the per-thread default stream
        with pytest.raises(ValueError, match="workspace"):
            wf.ops.attn_decode_i8(q, cache, pos)
