"""Keys that no row of a sequence sees (in front of the window, behind the
sinks) may hold anything: their pages may have gone to other sequences, their
slots may never have been written.  The results have the bits that they have
with finite values there."""

import math

import pytest
import torch

import attention_ops_ref as ref
from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200.runner import check_device_status
from test_attention_ops_gpu import DTYPES, attend, cache, check_paged, heads, normal, plan_for

pytestmark = pytest.mark.gpu


def hidden(q_len, kv_len, window, sinks):
    """Keys that no row sees, by the mask's definition."""
    return (~ref.visible(q_len, kv_len, window, sinks).any(0)).nonzero().flatten()


def poison_cache(c, page, window, sinks, other):
    """Entries of wholly hidden pages name page `other`; hidden slots of pages
    that are seen in part hold NaN (K, V) and infinities."""
    for b, (n, m) in enumerate(zip(c["lengths"], c["q_lens"])):
        keys = hidden(m, n, window, sinks) if m else torch.arange(0)
        for p in range(-(-n // page)):
            mine = keys[(keys >= p * page) & (keys < (p + 1) * page)]
            if len(mine) == page:
                c["table"][b, p] = other
            elif len(mine):
                at = int(c["table"][b, p])
                slots = (mine % page).cuda()
                c["k"][at, slots] = math.nan
                c["v"][at, slots] = math.nan
                c["k"][at, slots[::3]] = math.inf
                c["v"][at, slots[::3]] = -math.inf


HIDDEN_PAGED = [
    # lengths, new tokens, heads_q, heads_kv, dim, page, window, sinks
    ([1000], [1], 4, 1, 128, 16, 300, 0),
    ([1000, 77, 130, 513], [1, 1, 1, 1], 8, 2, 64, 16, 70, 4),
    ([700, 391], [1, 1], 4, 2, 64, 8, 1, 0),            # a window of one key
    ([900, 450], [40, 7], 6, 2, 128, 24, 100, 4),       # chunks
    ([900, 450], [40, 7], 4, 2, 64, 32, 100, 130),      # sinks end in the second block
    ([640, 300], [130, 1], 2, 1, 64, 256, 37, 1),       # pages larger than a block
    ([2000], [1], 16, 2, 128, 128, 200, 16),
    ([260], [1], 2, 2, 64, 64, 100, 150),               # sinks reach nearly to the window
    ([900] * 40, [65, 300] + [1] * 38, 16, 8, 64, 16, 90, 4),    # two tiles per unit, whole
    ([1500] * 4, [600] * 4, 16, 8, 128, 16, 200, 4),             # two tiles per unit, cut
]


@pytest.mark.parametrize("case", HIDDEN_PAGED, ids=lambda c: f"{c[0][:4]}-{c[1][:4]}-{c[2:]}")
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
@pytest.mark.parametrize("entry", ["page of NaN", "no page"])
def test_paged_hidden_pages_are_not_read(case, dtype, entry):
    lengths, q_lens, hq, hk, d, page, window, sinks = case
    c = cache(lengths, q_lens, hq, hk, d, page, dtype, seed=page)
    plan = plan_for(c, hq, hk, d, page, dtype, window, sinks)
    lse = torch.empty(c["q"].shape[:2], dtype=torch.float32, device="cuda")
    clean = attend(plan, c, lse=lse)
    clean_lse = lse.clone()
    used = set(c["table"][c["table"] >= 0].tolist())
    spare = next(p for p in range(c["k"].shape[0]) if p not in used)  # holds NaN alone
    poison_cache(c, page, window, sinks, spare if entry == "page of NaN" else -3)
    out = attend(plan, c, lse=lse)
    check_device_status()
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
    check_paged(c, out, lse, hq, hk, window, sinks, dtype)


HIDDEN_DENSE = [
    # batch, q_len, kv_len, heads_q, heads_kv, dim, window, sinks
    (1, 60, 300, 4, 2, 64, 100, 0),      # hidden keys end inside the first block that is seen
    (1, 60, 300, 4, 2, 128, 100, 5),
    (2, 1, 200, 4, 1, 64, 50, 0),
    (1, 33, 600, 3, 1, 128, 70, 130),    # sinks end in the second block
    (1, 40, 210, 2, 2, 64, 90, 60),      # hidden keys and visible ones at both ends of a block
    (1, 6000, 6500, 8, 8, 64, 300, 4),   # two tiles per unit
    (1, 2600, 3100, 16, 16, 128, 400, 0),
]


@pytest.mark.parametrize("case", HIDDEN_DENSE, ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
def test_window_hidden_keys_may_hold_anything(case, dtype):
    b, q_len, kv_len, hq, hk, d, window, sinks = case
    q, k, v = heads(b, q_len, kv_len, hq, hk, d, dtype, seed=kv_len)
    want = ops.window_attention_forward(q, k, v, window=window, sinks=sinks)
    keys = hidden(q_len, kv_len, window, sinks).cuda()
    assert len(keys) and len(keys) % 128
    for t in (k, v):
        t[:, keys] = math.nan
        t[:, keys[::3]] = math.inf
        t[:, keys[1::3]] = -math.inf
    got = ops.window_attention_forward(q, k, v, window=window, sinks=sinks)
    check_device_status()
    assert torch.isfinite(want[0]).all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("case", HIDDEN_DENSE, ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
@pytest.mark.parametrize("which", ["k", "v"])
def test_window_gradient_hidden_keys_may_hold_anything(case, dtype, which):
    b, q_len, kv_len, hq, hk, d, window, sinks = case
    mask = {"window": window, "sinks": sinks}
    q, k, v = heads(b, q_len, kv_len, hq, hk, d, dtype, seed=kv_len)
    dout = normal(b, q_len, hq, d, seed=41, dtype=dtype)
    out, lse = ops.window_attention_forward(q, k, v, **mask)
    want = ops.window_attention_backward(dout, q, k, v, out, lse, **mask)
    keys = hidden(q_len, kv_len, window, sinks).cuda()
    t = k if which == "k" else v
    t[:, keys] = math.nan
    t[:, keys[::3]] = math.inf
    got = ops.window_attention_backward(dout, q, k, v, out, lse, **mask)
    check_device_status()
    for a, w in zip(got, want):
        assert torch.isfinite(w).all() and torch.equal(a, w)
    assert not got[1][:, keys].any() and not got[2][:, keys].any()


@pytest.mark.parametrize("case", [
    (1, 300, 100, 4, 2, 64, None, 0),
    (2, 513, 130, 3, 1, 128, 40, 4),     # tokens without a key end inside a tile
    (1, 1500, 700, 8, 8, 128, 200, 0),
    (1, 260, 4, 16, 2, 64, 2, 1),
], ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
@pytest.mark.parametrize("which", ["q", "dout"])
def test_window_tokens_without_a_key_may_hold_anything(case, dtype, which):
    """More queries than keys: the first ones see nothing, give nothing to dK
    and dV, and their own gradient is 0."""
    b, q_len, kv_len, hq, hk, d, window, sinks = case
    mask = {"window": window, "sinks": sinks}
    q, k, v = heads(b, q_len, kv_len, hq, hk, d, dtype, seed=kv_len)
    dout = normal(b, q_len, hq, d, seed=42, dtype=dtype)
    out, lse = ops.window_attention_forward(q, k, v, **mask)
    want = ops.window_attention_backward(dout, q, k, v, out, lse, **mask)
    blind = q_len - kv_len
    t = q if which == "q" else dout
    t[:, :blind] = math.nan
    t[:, :blind:3] = -math.inf
    again, lse2 = ops.window_attention_forward(q, k, v, **mask)
    assert torch.equal(again, out) and torch.equal(lse2, lse)
    got = ops.window_attention_backward(dout, q, k, v, out, lse, **mask)
    check_device_status()
    for a, w in zip(got, want):
        assert torch.isfinite(w).all() and torch.equal(a, w)
    assert not got[0][:, :blind].any()
