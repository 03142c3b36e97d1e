"""Calls without a gradient of their own do not lose one silently: their
results need the gradient that their inputs need, and refuse to pass it on."""

import pytest
import torch

from gpu_optimizer_b200 import attention_ops as ops
from test_attention_ops_gpu import attend, cache, heads, normal, plan_for

pytestmark = pytest.mark.gpu


def refuses(name, results):
    for r in results if isinstance(results, tuple) else (results,):
        assert r.requires_grad
        with pytest.raises(RuntimeError, match=f"{name} has no gradient.*window_attention"):
            r.float().sum().backward()


@pytest.mark.parametrize("which", [0, 1, 2])
def test_window_halves(which):
    x = heads(1, 20, 20, 4, 2, 64, torch.bfloat16)
    dout = normal(1, 20, 4, 64, seed=1, dtype=torch.bfloat16)
    want = ops.window_attention_forward(*x)
    grads = ops.window_attention_backward(dout, *x, *want)
    assert not any(t.requires_grad for t in (*want, *grads))
    x[which].requires_grad_()
    got = ops.window_attention_forward(*x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    refuses("window_attention_forward", got)
    back = ops.window_attention_backward(dout, *x, *want)
    assert all(torch.equal(a, b) for a, b in zip(back, grads))
    refuses("window_attention_backward", back)
    with torch.no_grad():
        assert not any(t.requires_grad for t in ops.window_attention_forward(*x))
        assert not any(t.requires_grad for t in ops.window_attention_backward(dout, *x, *want))
    out = ops.window_attention(*x)  # has one
    out.backward(dout)
    assert torch.equal(x[which].grad, grads[which])


def test_window_backward_of_a_needed_output_gradient():
    x = heads(1, 20, 20, 4, 2, 64, torch.bfloat16)
    want = ops.window_attention_forward(*x)
    dout = normal(1, 20, 4, 64, seed=1, dtype=torch.bfloat16).requires_grad_()
    refuses("window_attention_backward", ops.window_attention_backward(dout, *x, *want))


@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_attend(which):
    c = cache([40, 33], [3, 1], 4, 2, 64, 16, torch.bfloat16)
    plan = plan_for(c, 4, 2, 64, 16, torch.bfloat16)
    want = attend(plan, c)
    assert not want.requires_grad
    c[which].requires_grad_()
    buf = torch.empty_like(want)
    for got in (attend(plan, c), attend(plan, c, out=buf)):
        assert torch.equal(got, want)
        refuses("PagedAttention.attend", got)
    assert torch.equal(buf, want) and not buf.requires_grad  # the caller's tensor stays as it is
    with torch.no_grad():
        got = attend(plan, c, out=buf)
    assert not got.requires_grad and got.data_ptr() == buf.data_ptr()
