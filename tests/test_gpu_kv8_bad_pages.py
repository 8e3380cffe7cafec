"""Page numbers that cannot be, seen by one thread of many while the others are done with their own."""
import numpy as np
import pytest
import torch

from cleffa_amd import Kv8Cache, Kv8Plan
from tests.test_gpu_kv8 import _int, _say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_seq", [3, 200, 1500])
@pytest.mark.parametrize("where", ["free", "released"])
def test_one_bad_page_refuses_the_pass(n_seq, where):
    """One page outside the pool, on the stack or among those that come back, in each part of a pass of many
    sequences: nothing changes, and the same pass with the page put right is planned."""
    _say("bad page", n_seq, where)
    for at in sorted({0, n_seq // 2, n_seq - 1}):
        cache = Kv8Cache(1, 1, 3 * n_seq, n_seq, 3)
        plan = Kv8Plan(cache, 65 * n_seq, 1)
        plan.update(_int([65] * n_seq))
        plan.check()
        new = np.full(n_seq, 64)
        spot = cache.free[at:at + 1] if where == "free" else cache.tables[at, 1:2]
        if where == "released":
            new[at] = -1
        good = spot.clone()
        spot.fill_(3 * n_seq)
        kept = [t.clone() for t in (cache.tables, cache.free, cache.state)]
        plan.update(_int(new))
        assert plan.status() == 8 and (plan.slots == -1).all() and (plan.cu_q == 0).all()
        cache.state[1] = 0
        assert all(torch.equal(a, b) for a, b in zip(kept, (cache.tables, cache.free, cache.state)))
        spot.copy_(good)
        plan.update(_int(new))
        plan.check()
        pages = torch.cat([cache.tables[r, :int(h)] for r, h in enumerate(cache.state[3::2].tolist())] + [cache.free[:int(cache.state[0])]])
        assert torch.equal(pages.sort().values, torch.arange(3 * n_seq, dtype=torch.int32, device="cuda"))
