"""Log probabilities of rows whose logits are large: masked throughout by a constant, a token forced or forbidden by one, values close together far from zero."""
import pytest
import torch

from test_gpu_token_logprobs import DEV, HALF, TINY, agree, formula, oracle

pytestmark = pytest.mark.gpu
EDGE = 2.0 ** 20
LARGE = {torch.float16: [3e4, 3.3e4, 6e4], torch.bfloat16: [1e6, 1.1e6, 1e9, 5e9, 1e10, 1e12, 1e20, 2.0 ** 95], torch.float32: [1e6, EDGE, 1.1e6, 2e7, 1e9, 5e9, 1e10, 1e12, 1e20, 2.0 ** 95, 2.0 ** 97]}


def rows(dt, v, g):
    """For each constant, of both signs: nothing but it; one of it among ordinary logits; ordinary ones among it; values next to it.  For float32 also values on both sides
    of +-2^20, in rising, falling and any order."""
    out = []
    for c in LARGE[dt]:
        for c in (c, -c):
            out.append(torch.full((v,), c))
            x = torch.randn(v, generator=g) * 3
            x[v // 3] = c
            out.append(x)
            x = torch.full((v,), c)
            x[v // 2:v // 2 + 9] = torch.randn(9, generator=g) * 3
            out.append(x)
            near = c * (1 + torch.randint(-6, 7, (v,), generator=g) * 2 * HALF[dt] * 0.999)
            out.append(near.clamp(-torch.finfo(dt).max, torch.finfo(dt).max))
    if dt == torch.float32:
        for c in (EDGE, -EDGE):
            steps = c + torch.linspace(-12, 12, v)
            out += [steps, steps.flip(0), steps[torch.randperm(v, generator=g)], c + torch.randint(-9, 10, (v,), generator=g) * 0.125]
    return torch.stack(out).to(dt)


@pytest.mark.parametrize("v,least", [(1001, 1), (9001, 500), (60000, 1), (400003, 1)])  # a warp, a block, a cluster (of few and of many batches) for a row
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_large_logits(wf, dt, v, least):
    g = torch.Generator().manual_seed(v)
    x = rows(dt, v, g)
    n = x.shape[0]
    tok = torch.randint(v, (n,), generator=g)
    tok[1::4] = v // 3  # the one that is forced or forbidden
    tok[2::4] = v // 2 + 3
    times = -(-least // n)
    dx, dtok = x.to(DEV).repeat(times, 1), tok.to(DEV).repeat(times)
    for some in range(0, n, 24):  # launches of few rows where a cluster is to take one
        pick = slice(some, min(n, some + 24)) if least == 1 else slice(0, n * times)
        for top in (0, 5):
            got = wf.token_logprobs(dx[pick], dtok[pick], top=top)
            for first in range(0, got.logprob.shape[0], n if least > 1 else 24):
                at = slice(some, min(n, some + 24)) if least == 1 else slice(0, n)
                here = slice(first, first + (at.stop - at.start))
                want, tol = oracle(x[at], tok[at], top)
                for a, w, t in zip(got, want[:3], tol):
                    agree(a[here], w, t)
                assert torch.equal(got.top_id[here].cpu(), want[3])
        if least > 1:
            break


@pytest.mark.parametrize("v", [1001, 30001])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_gradient_of_large_logits(wf, dt, v):
    g = torch.Generator().manual_seed(v + 1)
    x = rows(dt, v, g)
    n = x.shape[0]
    tok = torch.randint(v, (n,), generator=g).to(DEV)
    x = x.to(DEV).requires_grad_()
    got = wf.token_logprobs(x, tok, top=5)
    ws = [torch.randn(n, generator=g).to(DEV), torch.randn(n, generator=g).to(DEV), torch.randn(n, 5, generator=g).to(DEV)]
    (dx,) = torch.autograd.grad([got.logprob, got.entropy, got.top_logprob], x, ws)
    want, size = formula(x, tok, got.top_id, *ws)
    # as in the test of ordinary logits; a probability with a logarithm below -200 is 0 on both sides
    logp = torch.log_softmax(x.detach().double().cpu(), -1).clamp(min=-200)
    off = 2.0 ** -21 * (4 + logp.abs()) + 2.0 ** -23 * (v / 256 + 64)
    assert ((dx.double().cpu() - want).abs() <= HALF[dt] * want.abs() + off * size + TINY[dt] + 1e-37).all()


@pytest.mark.parametrize("n,v", [(3000, 1), (3000, 5), (2000, 1000), (600, 9000), (20, 60000)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_a_row_that_one_token_has_all_of(wf, dt, n, v):
    """No probability above 1 and no entropy below 0, not even by a rounding: what is taken of them (the logarithm of the rest, a root) would be NaN."""
    g = torch.Generator(device=DEV).manual_seed(v)
    x = torch.randn(n, v, generator=g, device=DEV)
    x[:, v // 2] = torch.exp(torch.rand(n, generator=g, device=DEV) * 7 + 3) + 20
    x[::2] -= 500
    x = x.to(dt)
    tok = torch.full((n,), v // 2, device=DEV)
    got = wf.token_logprobs(x, tok, top=1)
    assert (got.logprob <= 0).all() and (got.top_logprob <= 0).all() and (got.entropy >= 0).all() and torch.log1p(-got.logprob.exp()).isnan().sum() == 0
    for a, w, t in zip(got, *oracle(x, tok, 1)):
        agree(a, w, t)
