"""Arguments at the edge of their types: refused with a reason, not rounded
or cut to another value."""

import ctypes
import math

import pytest
import torch

from gpu_optimizer_b200 import _lib
from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200.runner import KernelBuildError
from test_attention_ops import call, paged, window

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
