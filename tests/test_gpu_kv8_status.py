"""What a program of several plans, or of a replayed one, learns about passes that could not be planned."""
import pytest
import torch

from cleffa_amd import Kv8Cache, Kv8Plan, TextAttention, _lib
from tests.test_gpu_kv8 import HD, _int, _qkv, _say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("elsewhere", [False, True])
def test_status_is_of_the_plan(elsewhere):
    """Two plans over one cache: a refused one stays refused when the other's next update is good."""
    cache = Kv8Cache(1, 1, 6, 2, 6)
    prompts, tokens = Kv8Plan(cache, 400, 2), Kv8Plan(cache, 2, 2, 1)
    after = torch.empty_like(cache.state) if elsewhere else None
    assert prompts.status() == tokens.status() == prompts.failed() == 0     # none made yet
    tokens.update(_int([1, 1]))
    tokens.check()
    prompts.update(_int([380, 10]), state_out=after)       # 6 + 1 pages of 6
    tokens.update(_int([1, 1]))
    assert prompts.status() & 1 and tokens.status() == 0 and int(cache.state[1]) == 0
    with pytest.raises(RuntimeError, match="too few free pages"):
        prompts.check()
    tokens.check()
    assert prompts.failed() & 1 and prompts.failed() == 0 and prompts.status() & 1 and tokens.failed() == 0
    prompts.update(_int([20, 0]))
    prompts.check()
    assert prompts.status() == prompts.failed() == 0


def test_failures_of_a_loop_are_kept():
    """Passes of a loop that are refused between good ones, the loop run step by step and from a graph."""
    nh, nkv = 4, 2
    for mode in ("eager", "graph"):
        _say("loop", mode)
        cache, att = Kv8Cache(1, nkv, 8, 2, 3), TextAttention(nh, nkv)
        plan, new = Kv8Plan(cache, 60, nh, 60), _int([0, 0])
        qkv, qn, kn = _qkv(60, nh, nkv, 1)
        out = torch.zeros(60, nh * HD, dtype=torch.bfloat16, device="cuda")

        def step():
            plan.update(new)
            att.forward_kv8(qkv, qn, kn, plan.pos3, plan, cache, 0, out=out)

        step()
        torch.cuda.synchronize()
        if mode == "graph":
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        lens = [0, 0]
        for a, b in [(30, 30), (61, 0), (1, 1), (40, 30), (60, 0), (60, 0), (0, 3)]:
            new.copy_(_int([a, b]))
            graph.replay() if mode == "graph" else step()
            good = a + b <= 60 and lens[0] + a <= 192
            assert (plan.status() == 0) == good
            lens = [lens[0] + a, lens[1] + b] if good else lens
            assert cache.state[2::2].tolist() == lens
        assert plan.status() == 0 and plan.failed() == 2 and plan.failed() == 0
        plan.update(_int([60, 0]))
        plan.update(_int([11, 0]))
        plan.update(_int([2, 0]))
        plan.update(_int([1, 0]))
        assert plan.status() == 0 and plan.failed() == 4


def test_a_buffer_that_was_not_cleared():
    """A plan buffer's first plan reports its own status alone, whatever the memory held."""
    cache = Kv8Cache(1, 1, 6, 2, 6)
    plan = Kv8Plan(cache, 10, 2)
    plan.work.fill_(-1)
    plan.update(_int([1, 1]))
    assert plan.status() == plan.failed() == 0
    plan.work[0] = 5                                       # no plan's header
    plan.work[_lib.KV8_PLAN_FAILED] = 77
    plan.update(_int([11, 0]))
    assert plan.status() == plan.failed() == 2
