"""Calls from a thread that has not used the GPU yet (autograd's, a server's):
nothing in it may have made the device's context current before."""

import threading

import pytest
import torch

from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200.runner import build_callable, check_device_status
from test_attention_ops_gpu import attend, cache, heads, normal, plan_for

pytestmark = pytest.mark.gpu


def in_a_thread(fn):
    got = []

    def run():
        try:
            got.append(fn())
        except Exception as e:  # handed to the caller
            got.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    torch.cuda.synchronize()
    check_device_status()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


def test_window_attention():
    q, k, v = heads(1, 200, 200, 4, 2, 64, torch.bfloat16)
    dout = normal(1, 200, 4, 64, seed=1, dtype=torch.bfloat16)
    out, lse = ops.window_attention_forward(q, k, v, window=50, sinks=2)
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    in_a_thread(lambda: ops.window_attention_forward(q, k, v, window=50, sinks=2, out=again,
                                                     lse=lse2))
    assert torch.equal(again, out) and torch.equal(lse2, lse)
    want = ops.window_attention_backward(dout, q, k, v, out, lse, window=50, sinks=2)
    grads = tuple(torch.empty_like(t) for t in want)
    in_a_thread(lambda: ops.window_attention_backward(dout, q, k, v, out, lse, window=50, sinks=2,
                                                      grads=grads))
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_window_attention_through_autograd():
    """The gradient runs in a thread of autograd's, in memory that the
    allocator holds already."""
    x = heads(1, 333, 333, 6, 2, 64, torch.float16)
    dout = normal(1, 333, 6, 64, seed=2, dtype=torch.float16)
    out, lse = ops.window_attention_forward(*x, window=100)
    want = ops.window_attention_backward(dout, *x, out, lse, window=100)
    for t in x:
        t.requires_grad_()
    ops.window_attention(*x, window=100).backward(dout)
    check_device_status()
    assert all(torch.equal(t.grad, g) for t, g in zip(x, want))


def test_paged_attention_and_append():
    c = cache([300, 77], [3, 1], 4, 2, 64, 16, torch.bfloat16)
    plan = plan_for(c, 4, 2, 64, 16, torch.bfloat16)
    want = attend(plan, c)
    out = torch.empty_like(want)
    in_a_thread(lambda: attend(plan, c, out=out))
    assert torch.equal(out, want)
    new = normal(4, 2, 64, seed=3, dtype=torch.bfloat16)
    in_a_thread(lambda: plan.append(new, new, c["k"], c["v"], c["table"], c["start"], c["len"]))
    assert torch.equal(c["k"][int(c["table"][1, 4]), 76 % 16], new[3])


@pytest.mark.parametrize("task,shape,cfg", [
    ("matmul", (512, 512, 512), {"BLOCK_M": 128, "BLOCK_N": 128, "BLOCK_K": 64, "GROUP_M": 8,
                                 "num_warps": 8, "num_stages": 3, "dtype": "bfloat16"}),
    ("attention", (4, 512, 64), {"BLOCK_M": 128, "BLOCK_N": 64, "num_warps": 4, "num_stages": 2,
                                 "dtype": "bfloat16"}),
])
def test_tasks(task, shape, cfg):
    if task == "matmul":
        m, n, k = shape
        ins = (normal(m, k, seed=4, dtype=torch.bfloat16), normal(k, n, seed=5,
                                                                  dtype=torch.bfloat16))
    else:
        ins = tuple(normal(*shape, seed=s, dtype=torch.bfloat16) for s in (4, 5, 6))
    kc = build_callable(task, shape, cfg, ins)
    want = kc.fn().clone()
    kc.fn().zero_()
    got = in_a_thread(kc.fn)
    assert torch.equal(got, want) and want.any()
