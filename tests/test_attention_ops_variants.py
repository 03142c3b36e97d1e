"""Which kernel instance a call launches (the rules behind the launch records
and behind the cases of test_attention_ops_variants_gpu.py)."""

import pytest

from gpu_optimizer_b200.attention_ops import kernel_name
from gpu_optimizer_b200.runner import KernelBuildError


@pytest.mark.parametrize("shape,cfg,want", [
    # two tiles of 128 rows per unit where every SM gets more than two tiles
    ((1, 1024, 1024, 32, 8, 128), {}, "bf16,D=128,dense,tiles=1"),
    ((1, 8192, 8192, 32, 8, 128), {"window": 1024, "sinks": 4}, "bf16,D=128,dense,tiles=2"),
    ((2, 257, 257, 8, 2, 64), {"dtype": "float16"}, "f16,D=64,dense,tiles=1"),
    # keys that no token sees: kv_len - q_len - window + 1 > sinks
    ((1, 60, 300, 4, 2, 64), {"window": 100}, "bf16,D=64,dense,tiles=1,unseen"),
    ((1, 60, 300, 4, 2, 64), {"window": 100, "sinks": 140}, "bf16,D=64,dense,tiles=1,unseen"),
    ((1, 60, 300, 4, 2, 64), {"window": 100, "sinks": 141}, "bf16,D=64,dense,tiles=1"),
    ((1, 60, 300, 4, 2, 64), {"window": 241}, "bf16,D=64,dense,tiles=1"),
    ((1, 60, 300, 4, 2, 64), {}, "bf16,D=64,dense,tiles=1"),
])
def test_dense(shape, cfg, want):
    assert kernel_name("attention_window", shape, cfg) == f"attn_fwd_kernel<{want}>"


@pytest.mark.parametrize("shape,tokens,want", [
    ((64, 1, 64, 32, 8, 128), 64, "tiles=1,cut"),
    ((4, 512, 16, 32, 8, 128), 2048, "tiles=2,cut"),
    # a plan that takes chunks, serving single tokens
    ((64, 512, 16, 32, 8, 128), 64, "tiles=2,cut"),
    ((256, 512, 16, 32, 8, 128), 256, "tiles=2"),
    ((1300, 1, 8, 2, 1, 128), 1300, "tiles=1"),
])
def test_paged(shape, tokens, want):
    assert kernel_name("attention_paged", shape, {}, tokens) == \
        f"attn_fwd_kernel<bf16,D=128,paged,{want}>"


def test_others_and_refusals():
    assert kernel_name("cache_append", (), {}) == "cache_append_kernel"
    assert kernel_name("attention_window_grad", (), {}) == "attn_grad_kernel"
    with pytest.raises(KernelBuildError, match="page_size"):
        kernel_name("attention_paged", (4, 1, 13, 32, 8, 128), {}, 4)
    with pytest.raises(KernelBuildError, match="head_dim"):
        kernel_name("attention_window", (1, 8, 8, 4, 2, 96), {})
