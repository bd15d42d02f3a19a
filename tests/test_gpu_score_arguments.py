"""Scores of tokens wherever and however they are kept, and what is refused before the cache is touched."""
import pytest
import torch

from test_gpu_decoder_i8 import make, prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(), dict(cache_dtype=torch.int8, head_dtype=torch.int8)])
def test_tokens_of_other_types_and_places(wf, kw):
    m, ids = make(wf, **kw), prompt(3, 9)
    want = m.score(ids, top=2)
    for other in (ids.cpu(), ids.int(), ids.int().cpu()):
        assert all(torch.equal(a, b) for a, b in zip(m.score(other, top=2), want))


def test_too_many_alternatives(wf):
    m, ids = make(wf), prompt(3, 9)
    m.prefill(ids)
    before = [L["kc"].clone() for L in m.layers], m.tok.clone(), int(m.pos)
    for top in (-1, 33):
        with pytest.raises(ValueError):
            m.score(prompt(3, 20).flip(0), top=top)
    assert all(torch.equal(a, L["kc"]) for a, L in zip(before[0], m.layers)) and torch.equal(m.tok, before[1]) and int(m.pos) == before[2]
