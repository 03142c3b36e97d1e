"""Arguments at the edge of their types: refused with a reason, not rounded
or cut to another value."""

import ctypes
import math

import pytest
import torch

from gpu_optimizer_b200 import _lib
from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200.runner import KernelBuildError
from test_attention_ops import call, heads, paged, window

PLAN = dict(heads_q=4, heads_kv=2, head_dim=64, page_size=16, max_seqs=2, max_q=4,
            dtype=torch.bfloat16, device="cuda:0")


@pytest.mark.parametrize("scale", [1e-60, 5e-324, 1e-39, 1e39])
def test_scales_that_no_float_holds_are_refused(scale):
    """1e-60 is 0 in 32 bits, which would ask for the default scale."""
    with pytest.raises(KernelBuildError, match="scale must be"):
        ops.PagedAttention(**PLAN, scale=scale)


@pytest.mark.parametrize("scale", [1e-39, 1.4e-45])
def test_scales_below_the_normal_numbers_are_refused(scale):
    """Times log2(e) and a masked score they may come out as 0 * -inf."""
    rc, log = call("gpo_window_workspace", window(scale=scale), ctypes.c_uint64(0))
    assert rc == _lib.BAD_ARGS and "scale" in log
    rc, log = call("gpo_cache_append", paged(scale=scale), None)
    assert rc == _lib.BAD_ARGS and "scale" in log
    tiny = 2.0 ** -126
    assert call("gpo_window_workspace", window(scale=tiny), ctypes.c_uint64(0))[0] == _lib.OK
    assert math.isclose(tiny, 1.1754944e-38, rel_tol=1e-6)


@pytest.mark.parametrize("bad", [{"heads_q": 2 ** 32 + 4}, {"heads_kv": 2 ** 32 + 2},
                                 {"head_dim": 2 ** 32 + 64}, {"heads_q": -2 ** 32 + 4}])
def test_sizes_that_32_bits_do_not_hold_are_refused(bad):
    with pytest.raises(KernelBuildError, match=next(iter(bad))):
        ops.PagedAttention(**{**PLAN, **bad})


def test_plans_may_allow_more_tokens_than_a_call_has():
    """4096 sequences or chunks of 2^20 tokens, if not both in one call: the
    plan is only refused for what a call could not hold alone."""
    try:
        ops.PagedAttention(**{**PLAN, "max_seqs": 4096, "max_q": 1 << 20})
    except KernelBuildError as e:
        pytest.fail(f"refused: {e}")
    except (RuntimeError, AssertionError):
        assert not torch.cuda.is_available()  # no device to allocate the workspace on
    for bad in ({"max_seqs": 65536}, {"max_q": (1 << 30) + 1}, {"max_q": 1 << 62, "max_seqs": 4}):
        with pytest.raises(KernelBuildError, match="num_seqs"):
            ops.PagedAttention(**{**PLAN, **bad})


def test_pointers_off_their_types_grid_are_refused():
    """A misaligned address is a fault on the device."""
    q = heads(4096, 2048, 256, 64)
    kv = heads(4096, 1024, 128, 64)
    dense = dict(q=q, k=kv, v=kv, out=q, lse=4098)
    rc, log = call("gpo_window_attention", window(**dense), None)
    assert rc == _lib.BAD_ARGS and "lse is not 4-byte aligned" in log
    grads = dict(dense, dout=q, dq=q, dk=kv, dv=kv)
    rc, log = call("gpo_window_attention_grad", window(**grads), None)
    assert rc == _lib.BAD_ARGS and "lse is not 4-byte aligned" in log
    pages = dict(k_pages=heads(4096, 2048, 128, 64), v_pages=heads(4096, 2048, 128, 64),
                 q=heads(4096, 0, 256, 64), out=heads(4096, 0, 256, 64), page_table=64, q_start=64,
                 kv_len=64, lse=64, k_new=heads(4096, 0, 128, 64), v_new=heads(4096, 0, 128, 64))
    for name in ("page_table", "q_start", "kv_len", "lse"):
        rc, log = call("gpo_paged_attention", paged(**{**pages, name: 66}), None)
        assert rc == _lib.BAD_ARGS and f"{name} is not 4-byte aligned" in log, log
    rc, log = call("gpo_cache_append", paged(**{**pages, "kv_len": 65}), None)
    assert rc == _lib.BAD_ARGS and "kv_len is not 4-byte aligned" in log
