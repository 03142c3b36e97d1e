"""A plan's workspace on other streams than the one that made the plan."""

import pytest
import torch

from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200.runner import check_device_status
from test_attention_ops_gpu import attend, cache, plan_for

pytestmark = pytest.mark.gpu

HEADS = (32, 8, 128, 16)  # query heads, kv heads, head_dim, page


def problem(seed=60):
    """Long single-token sequences: every unit is cut and joined through the
    counters in the workspace."""
    return cache([4000, 3001], [1, 1], *HEADS, torch.bfloat16, seed=seed)


def dirty(stream):
    """Leave freed blocks of all ones to `stream`'s next allocations."""
    with torch.cuda.stream(stream):
        for n in range(16, 26):
            torch.full((1 << n,), 255, dtype=torch.uint8, device="cuda")


def test_first_call_on_another_stream_finds_a_zeroed_workspace():
    c = problem()
    want = attend(plan_for(c, *HEADS, torch.bfloat16), c)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        dirty(a)
        with torch.cuda.stream(a):
            torch.cuda._sleep(20_000_000)  # what is queued here runs much later
            plan = plan_for(c, *HEADS, torch.bfloat16)
        with torch.cuda.stream(b):
            got = attend(plan, c)
        b.synchronize()
        assert torch.equal(got, want)
        torch.cuda.synchronize()
    check_device_status()


def test_making_a_plan_does_not_wait_for_queued_work():
    c = problem()
    a = torch.cuda.Stream()
    with torch.cuda.stream(a):
        plan_for(c, *HEADS, torch.bfloat16)
        torch.cuda._sleep(2_000_000_000)  # a second
        plan = plan_for(c, *HEADS, torch.bfloat16)
        assert not a.query()
        out = attend(plan, c)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()


def test_a_dropped_plan_keeps_its_workspace_until_its_calls_are_done():
    c = problem()
    want = attend(plan_for(c, *HEADS, torch.bfloat16), c)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(a):
            plan = plan_for(c, *HEADS, torch.bfloat16)
        with torch.cuda.stream(b):
            torch.cuda._sleep(20_000_000)
            got = attend(plan, c)
        del plan
        with torch.cuda.stream(a):  # takes and fills what the plan gave back
            held = [torch.full((1 << n,), 255, dtype=torch.uint8, device="cuda")
                    for n in range(16, 26)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del held
    check_device_status()


def test_plan_made_in_a_capture():
    c = problem()
    want = attend(plan_for(c, *HEADS, torch.bfloat16), c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan = plan_for(c, *HEADS, torch.bfloat16)
        held = attend(plan, c)
    for _ in range(2):
        held.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
    check_device_status()


def test_plans_take_up_the_memory_of_those_before():
    c = problem()
    for _ in range(2):
        attend(plan_for(c, *HEADS, torch.bfloat16), c)
        torch.cuda.synchronize()
    held = torch.cuda.memory_reserved()
    for _ in range(40):
        attend(plan_for(c, *HEADS, torch.bfloat16), c)
        torch.cuda.synchronize()
    assert torch.cuda.memory_reserved() == held
