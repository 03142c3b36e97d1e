"""Every instance of the forward kernel against the 64-bit forms, at sizes
that the dispatch gives to it (asserted, so that a later rule cannot take an
instance out of the tests): two tiles per unit, dense and paged, cut and whole."""

import math

import pytest
import torch

from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200.attention_ops import kernel_name
from gpu_optimizer_b200.runner import build_callable, check_device_status
from test_attention_ops_gpu import (DTYPES, attend, cache, check_paged, check_window, heads,
                                    normal, plan_for)

pytestmark = pytest.mark.gpu


def config(dtype, window=None, sinks=0):
    return {"dtype": str(dtype).split(".")[1], "window": window or 0, "sinks": sinks}


def instance(dtype, d, form):
    return f"attn_fwd_kernel<{'bf16' if dtype == torch.bfloat16 else 'f16'},D={d},{form}>"


# ---------------------------------------------------------------------- dense
DENSE_TWO = [
    # batch, q_len, kv_len, heads_q, heads_kv, dim, window, sinks
    (1, 2700, 2700, 16, 16, 128, None, 0),    # causal: up to 22 blocks a unit
    (1, 2700, 2700, 16, 16, 64, None, 0),
    (2, 1400, 1400, 24, 8, 128, 300, 4),      # groups of three: rows 126, 127 unused
    (1, 2100, 2100, 32, 8, 64, 1000, 130),    # sinks in two blocks
    (1, 2055, 2055, 40, 8, 128, None, 0),     # groups of five; one token in the last tile
    (1, 2600, 3100, 16, 16, 128, 600, 5),     # a prefix in front
    (1, 2600, 3100, 16, 16, 64, 300, 4),      # of which keys 4..200 are not seen
    (3, 1800, 900, 8, 8, 128, 200, 3),        # tokens without a key
]


@pytest.mark.parametrize("case", DENSE_TWO, ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
def test_dense_two_tiles(case, dtype):
    b, q_len, kv_len, hq, hk, d, window, sinks = case
    unseen = window is not None and kv_len - q_len - window + 1 > sinks
    assert kernel_name("attention_window", case[:6], config(dtype, window, sinks)) == \
        instance(dtype, d, "dense,tiles=2" + (",unseen" if unseen else ""))
    q, k, v = heads(b, q_len, kv_len, hq, hk, d, dtype, seed=q_len)
    check_window(q, k, v, window, sinks, normal(b, q_len, hq, d, seed=9, dtype=dtype))


@pytest.mark.parametrize("d", [64, 128])
def test_dense_two_tiles_with_growing_scores(d):
    """Scores that grow along the keys (from -32 to 32) move the running
    maximum, and with it O in TMEM, every other block of both tiles."""
    n, h = 2700, 16
    assert kernel_name("attention_window", (1, n, n, h, h, d), config(torch.bfloat16)) == \
        instance(torch.bfloat16, d, "dense,tiles=2")
    q, k, v = heads(1, n, n, h, h, d, torch.bfloat16, seed=61)
    up = torch.linspace(-8, 8, n, device="cuda")[None, :, None, None]
    q = (q * 0.1 + 1).to(q.dtype)
    k = (k * 0.05 + up * 4 / math.sqrt(d)).to(k.dtype)
    check_window(q, k, v, None, 0)


def test_dense_two_tiles_of_strided_tensors():
    """Slices of a fused projection, an output in (batch, head, token, dim) order."""
    b, s, hq, hk, d = 2, 1500, 32, 8, 128
    assert kernel_name("attention_window", (b, s, s, hq, hk, d),
                       config(torch.bfloat16, 300, 4)) == \
        instance(torch.bfloat16, d, "dense,tiles=2")
    fused = normal(b, s, hq + 2 * hk, d, seed=62, dtype=torch.bfloat16)
    q, k, v = fused[:, :, :hq], fused[:, :, hq:hq + hk], fused[:, :, hq + hk:]
    check_window(q, k, v, 300, 4)
    want = ops.window_attention_forward(q.contiguous(), k.contiguous(), v.contiguous(),
                                        window=300, sinks=4)
    out = torch.empty(b, hq, s, d, dtype=q.dtype, device="cuda").transpose(1, 2)
    got = ops.window_attention_forward(q, k, v, window=300, sinks=4, out=out)
    assert torch.equal(out, want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------------------------- paged
PAGED_TWO = [
    # lengths, new tokens, heads_q, heads_kv, dim, page, window, sinks, the plan's max_q, cut
    ([3000, 2500, 1111, 2049], [700, 513, 300, 650], 32, 8, 128, 16, None, 0, 700, True),
    ([800, 640, 900, 911, 1300, 64, 77], [800, 640, 399, 250, 130, 1, 77], 24, 8, 64, 24, 200, 4,
     800, True),                                                   # groups of three, window, sinks
    ([900, 300, 1], [600, 300, 1], 40, 8, 128, 64, None, 0, 1024, True),     # groups of five
    ([6000, 5001], [700, 650], 32, 8, 64, 128, None, 0, 700, True),  # units over several CTAs
    ([300] * 4, [500] * 4, 32, 8, 128, 16, None, 0, 512, True),      # tokens without a key
    ([512, 300, 650] + [100 + 7 * i for i in range(37)], [512, 300, 65] + [1] * 37, 32, 8, 128, 16,
     None, 0, 512, False),
    ([777, 1000, 650, 0] + [40 + 3 * i for i in range(40)], [510, 301, 65, 0] + [2] * 40, 24, 8, 64,
     32, 150, 130, 512, False),
    # single tokens from a plan that takes chunks: the second tile is empty
    ([5000, 3333, 1] + [129 * i for i in range(1, 62)], [1] * 64, 32, 8, 128, 16, None, 0, 512,
     True),
    ([3000] + [5 * i for i in range(1, 64)], [1] * 64, 32, 8, 64, 64, 200, 4, 512, True),
    ([2000] + [2 * i for i in range(1, 256)], [1] * 256, 32, 8, 128, 16, None, 0, 512, False),
]


@pytest.mark.parametrize("case", PAGED_TWO, ids=lambda c: f"{len(c[0])}-{c[0][:3]}-{c[1][:3]}-{c[2:]}")
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
def test_paged_two_tiles(case, dtype):
    lengths, q_lens, hq, hk, d, page, window, sinks, max_q, cut = case
    assert kernel_name("attention_paged", (len(lengths), max_q, page, hq, hk, d),
                       config(dtype, window, sinks), sum(q_lens)) == \
        instance(dtype, d, "paged,tiles=2" + (",cut" if cut else ""))
    c = cache(lengths, q_lens, hq, hk, d, page, dtype, seed=len(lengths) + page)
    plan = plan_for(c, hq, hk, d, page, dtype, window, sinks, max_q=max_q)
    lse = torch.empty(c["q"].shape[:2], dtype=torch.float32, device="cuda")
    out = attend(plan, c, lse=lse)
    check_device_status()
    check_paged(c, out, lse, hq, hk, window, sinks, dtype)
    for _ in range(3):  # equal bits, and the plan's counters are back at zero each time
        again = attend(plan, c)
        assert torch.equal(again, out)
    check_device_status()


@pytest.mark.parametrize("cut", [True, False])
def test_paged_two_tiles_with_growing_scores(cut):
    """The running maximum moves all along; parts of cut units have maxima far
    apart."""
    hq, hk, d, page = 32, 8, 128, 16
    lengths, q_lens = ([2500, 1800], [700, 700]) if cut else ([900, 700] + [300] * 38,
                                                               [300, 200] + [40] * 38)
    max_q = 700 if cut else 512
    assert kernel_name("attention_paged", (len(lengths), max_q, page, hq, hk, d),
                       config(torch.bfloat16), sum(q_lens)) == \
        instance(torch.bfloat16, d, "paged,tiles=2" + (",cut" if cut else ""))
    c = cache(lengths, q_lens, hq, hk, d, page, torch.bfloat16, seed=63)
    c["q"] = (c["q"] * 0.1 + 1).to(torch.bfloat16)
    for b, n in enumerate(lengths):
        up = torch.linspace(-8, 8, n)[:, None, None] * 4 / math.sqrt(d)
        c["ks"][b] = (c["ks"][b] * 0.05 + up).to(torch.bfloat16)
        slots = torch.arange(n)
        ids = c["table"][b].cpu()[slots // page].long()
        c["k"][ids.cuda(), (slots % page).cuda()] = c["ks"][b].cuda()
    plan = plan_for(c, hq, hk, d, page, torch.bfloat16, max_q=max_q)
    lse = torch.empty(c["q"].shape[:2], dtype=torch.float32, device="cuda")
    out = attend(plan, c, lse=lse)
    check_device_status()
    check_paged(c, out, lse, hq, hk, None, 0, torch.bfloat16)


@pytest.mark.parametrize("lengths,q_len,max_q,d,form", [
    ([700, 90, 333], 1, 1, 64, "tiles=1,cut"),
    ([40 + 5 * i for i in range(200)], 1, 1, 128, "tiles=1"),  # whole: eight rounds of units
    ([60 + i % 50 for i in range(300)], 3, 3, 64, "tiles=1"),
])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
def test_paged_one_tile(lengths, q_len, max_q, d, form, dtype):
    hq, hk, page = 16, 8, 32
    n = len(lengths)
    assert kernel_name("attention_paged", (n, max_q, page, hq, hk, d), config(dtype),
                       n * q_len) == instance(dtype, d, "paged," + form)
    c = cache(lengths, [q_len] * n, hq, hk, d, page, dtype, seed=64)
    plan = plan_for(c, hq, hk, d, page, dtype, max_q=max_q)
    lse = torch.empty(c["q"].shape[:2], dtype=torch.float32, device="cuda")
    out = attend(plan, c, lse=lse)
    check_device_status()
    check_paged(c, out, lse, hq, hk, None, 0, dtype)


def test_launch_records_name_the_instance():
    q, k, v = heads(1, 2700, 2700, 16, 16, 128, torch.bfloat16)
    kc = build_callable("attention_window", (1, 2700, 2700, 16, 16, 128),
                        config(torch.bfloat16, 300, 4), (q, k, v))
    assert kc.launch["kernel"] == "attn_fwd_kernel<bf16,D=128,dense,tiles=2>"
    c = cache([64, 30], [3, 1], 4, 2, 64, 16, torch.bfloat16)
    kc = build_callable("attention_paged", (2, 3, 16, 4, 2, 64), config(torch.bfloat16),
                        (c["q"], c["k"], c["v"], c["table"], c["start"], c["len"]))
    assert kc.launch["kernel"] == "attn_fwd_kernel<bf16,D=64,paged,tiles=1,cut>"
