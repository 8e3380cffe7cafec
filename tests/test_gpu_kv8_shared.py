"""A sequence on another's document, from its start to its end, with nothing looked at on the host."""
import pytest
import torch

from cleffa_amd import Kv8Cache, Kv8Plan, TextAttention
from tests.test_gpu_kv8 import HD, _int, _qkv, _say

pytestmark = pytest.mark.gpu


def borrow(cache, r, owner, pages):
    """Sequence r (without pages) starts on the first pages of another."""
    cache.tables[r, :pages] = cache.tables[owner, :pages]
    cache.state[2 + 2 * r], cache.state[3 + 2 * r] = 64 * pages, pages


def give_back(cache, r, pages):
    """Sequence r lets go of the pages that it borrowed; those of its own stay with it, for the plan that ends it."""
    cache.tables[r, :-pages] = cache.tables[r, pages:].clone()
    cache.state[2 + 2 * r] = 0
    cache.state[3 + 2 * r] -= pages


@pytest.mark.parametrize("doc,own", [(1, 70), (3, 1), (3, 64), (2, 200)])
def test_a_borrower_ends_and_the_document_stays(doc, own):
    """Requests come and go on one document: after each its own pages are free again, no page is there twice, and
    the next one's outputs are the first's bit for bit."""
    _say("document of", doc, "pages, own tokens", own)
    nh, nkv, pages = 8, 2, 12
    cache, att = Kv8Cache(1, nkv, pages, 3, 8), TextAttention(nh, nkv)
    plan = Kv8Plan(cache, 64 * doc, nh)
    plan.update(_int([64 * doc, 0, 0]))
    rows = _qkv(64 * doc, nh, nkv, 1)
    att.forward_kv8(*rows, plan.pos3, plan, cache, 0)
    plan, q = Kv8Plan(cache, own, nh), _qkv(own, nh, nkv, 2)[0]
    codes, outs = cache.k[0][cache.tables[0, :doc].long()].clone(), []
    for i in range(6):
        r = 1 + i % 2
        borrow(cache, r, 0, doc)
        new = torch.zeros(3, dtype=torch.int32, device="cuda")
        new[r] = own
        plan.update(new)
        outs.append(att.forward_kv8(q, rows[1], rows[2], plan.pos3, plan, cache, 0))
        give_back(cache, r, doc)
        new[r] = -1
        plan.update(new)
        plan.check()
        assert plan.failed() == 0
        held = torch.cat([cache.tables[0, :doc], cache.free[:int(cache.state[0])]])
        assert cache.state.tolist() == [pages - doc, 0, 64 * doc, doc, 0, 0, 0, 0]
        assert torch.equal(held.sort().values, torch.arange(pages, dtype=torch.int32, device="cuda"))
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    assert torch.equal(codes, cache.k[0][cache.tables[0, :doc].long()])
    # the document's own sequence goes on, and ends with all its pages
    plan.update(_int([own, 0, 0]))
    plan.check()
    plan.update(_int([-1, 0, 0]))
    plan.check()
    assert cache.state.tolist() == [pages, 0, 0, 0, 0, 0, 0, 0]
