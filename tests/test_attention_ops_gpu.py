"""Window attention (forward, gradient), paged attention and cache append
against plain 64-bit forms, at the sizes, masks and layouts where such kernels
go wrong.  The bounds are derived in attention_ops_ref.py."""

import math
import random

import pytest
import torch

import attention_ops_ref as ref
from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200.runner import (KernelBuildError, build_callable, check_device_status,
                                       warm_compile)

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def normal(*shape, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def heads(b, q_len, kv_len, hq, hk, d, dtype, seed=0):
    return (normal(b, q_len, hq, d, seed=seed, dtype=dtype),
            normal(b, kv_len, hk, d, seed=seed + 1, dtype=dtype),
            normal(b, kv_len, hk, d, seed=seed + 2, dtype=dtype))


def check_window(q, k, v, window, sinks, dout=None, scale=None):
    """Forward (and gradient, given dout) against the 64-bit form."""
    mask = {"window": window, "sinks": sinks, "scale": scale}
    out, lse = ops.window_attention_forward(q, k, v, **mask)
    got = {"out": out}
    if dout is not None:
        got.update(zip(("dq", "dk", "dv"),
                       ops.window_attention_backward(dout, q, k, v, out, lse, **mask)))
    check_device_status()
    g = q.shape[2] // k.shape[2]
    see = ref.visible(q.shape[1], k.shape[1], window, sinks, "cuda")
    s = scale or q.shape[3] ** -0.5
    u = ref.unit(q.dtype)
    for b in range(q.shape[0]):
        for hk in range(k.shape[2]):
            want = {n: 0.0 for n in ("dk", "dv")}
            bound = {n: 0.0 for n in ("dk", "dv")}
            for h in range(hk * g, (hk + 1) * g):
                r = ref.head(q[b, :, h], k[b, :, hk], v[b, :, hk], see, s,
                             None if dout is None else dout[b, :, h])
                e = ref.bounds(r, q.dtype, s)
                ref.within("out", out[b, :, h], r["out"], e["out"])
                fin = torch.isfinite(r["lse"])
                assert torch.equal(torch.isfinite(lse[b, :, h]), fin)
                assert (lse[b, :, h][~fin] == -math.inf).all()
                assert (lse[b, :, h][fin] - r["lse"][fin]).abs().max().item() < ref.R \
                    if fin.any() else True
                if dout is not None:
                    ref.within("dq", got["dq"][b, :, h], r["dq"], e["dq"])
                    for n in ("dk", "dv"):
                        want[n] = want[n] + r[n]
                        bound[n] = bound[n] + e[n]
            if dout is not None:
                for n in ("dk", "dv"):
                    ref.within(n, got[n][b, :, hk], want[n], bound[n] + u * want[n].abs())
    return got, lse


# ------------------------------------------------------- window: sizes, masks
WINDOW_CASES = [
    # batch, q_len, kv_len, heads_q, heads_kv, dim, window, sinks
    (1, 1, 1, 1, 1, 64, None, 0),
    (2, 2, 2, 4, 2, 128, 1, 0),
    (1, 127, 127, 2, 2, 64, None, 0),
    (1, 128, 128, 1, 1, 128, 64, 4),
    (1, 129, 129, 3, 1, 64, 100, 2),
    (2, 257, 257, 8, 2, 64, 128, 4),      # window of one block
    (1, 300, 300, 5, 1, 128, 129, 0),     # five heads: rows 125..127 of a tile unused
    (1, 511, 511, 7, 1, 64, 37, 1),
    (1, 640, 640, 6, 2, 128, 200, 130),   # sinks in two blocks
    (1, 1000, 1000, 16, 1, 64, 1, 3),     # a window of one key
    (1, 200, 200, 24, 1, 128, 50, 200),   # every key a sink
    (1, 700, 700, 2, 1, 128, 699, 5),
    (1, 64, 1000, 4, 4, 64, None, 0),     # a prefix in front
    (2, 33, 500, 4, 2, 128, 70, 4),
    (1, 300, 100, 4, 2, 64, None, 0),     # fewer keys than queries: rows without a key
    (1, 300, 100, 2, 1, 128, 40, 4),
    (1, 513, 130, 1, 1, 64, 8, 0),
    (1, 40, 40, 128, 1, 64, 16, 2),       # 128 heads: one token per tile
    (1, 37, 37, 100, 1, 64, None, 0),
    (3, 2050, 2050, 4, 1, 64, 256, 4),    # far pieces of the sinks' gradient
    (2, 250, 250, 6, 2, 64, 100, 2),      # sinks whose window reaches the last token
    (1, 300, 300, 4, 4, 128, 290, 140),   # the same, sinks in two key tiles
    (4, 1724, 1551, 8, 1, 64, 11, 4),     # whole tiles without a key between others
    (2, 6000, 500, 4, 1, 64, 100, 4),     # most tiles without a key
]


@pytest.mark.parametrize("case", WINDOW_CASES, ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
def test_window_forward_and_gradient(case, dtype):
    b, q_len, kv_len, hq, hk, d, window, sinks = case
    q, k, v = heads(b, q_len, kv_len, hq, hk, d, dtype, seed=q_len)
    dout = normal(b, q_len, hq, d, seed=9, dtype=dtype)
    check_window(q, k, v, window, sinks, dout)


def test_window_random_shapes():
    r = random.Random(5)
    for i in range(25):
        hk = r.choice((1, 2, 3))
        hq = hk * r.randint(1, 9)
        d, q_len = r.choice((64, 128)), r.randint(1, 700)
        kv_len = r.choice((q_len, r.randint(1, 700)))
        window = r.choice((None, r.randint(1, 300)))
        sinks = r.choice((0, r.randint(1, 150)))
        q, k, v = heads(1, q_len, kv_len, hq, hk, d, r.choice(DTYPES), seed=i)
        check_window(q, k, v, window, sinks, normal(1, q_len, hq, d, seed=99, dtype=q.dtype))


@pytest.mark.parametrize("q_len,kv_len", [(0, 5), (5, 0), (0, 0)])
def test_window_lengths_of_zero(q_len, kv_len):
    q, k, v = heads(2, q_len, kv_len, 4, 2, 64, torch.bfloat16)
    out, lse = ops.window_attention_forward(q, k, v)
    dq, dk, dv = ops.window_attention_backward(out, q, k, v, out, lse)
    check_device_status()
    assert out.shape == q.shape and not out.any() and not dq.any()
    assert (lse == -math.inf).all() and not dk.any() and not dv.any()


def test_window_batch_of_zero():
    q, k, v = heads(0, 4, 4, 4, 2, 64, torch.bfloat16)
    out, lse = ops.window_attention_forward(q, k, v)
    grads = ops.window_attention_backward(out, q, k, v, out, lse)
    assert out.numel() == 0 and all(g.numel() == 0 for g in grads)


# ------------------------------------------------------------ window: layouts
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
def test_window_reads_strided_tensors(dtype):
    """Slices of a fused projection, (batch, head, token, dim) storage, a
    broadcast key head, rows off the 16-byte grid."""
    b, s, hq, hk, d = 2, 150, 6, 2, 64
    mask = {"window": 60, "sinks": 3}
    fused = normal(b, s, hq + 2 * hk, d, seed=1, dtype=dtype)
    q, k, v = fused[:, :, :hq], fused[:, :, hq:hq + hk], fused[:, :, hq + hk:]
    dout = normal(b, hq, s, d, seed=2, dtype=dtype).transpose(1, 2)
    check_window(q, k, v, 60, 3, dout)
    want = ops.window_attention_forward(q.contiguous(), k.contiguous(), v.contiguous(), **mask)
    views = [
        tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)),
        (q.flip(1).flip(1), k[:, :, :], v.clone()),
    ]
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    views.append((odd, k, v))
    wide = torch.empty(*q.shape[:3], d + 4, dtype=dtype, device="cuda")[..., :d]
    wide.copy_(q)
    views.append((wide, k, v))
    for vw in views:
        got = ops.window_attention_forward(*vw, **mask)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = k[:, :, :1].expand(b, s, hk, d)  # stride 0: one key head for all
    got = ops.window_attention_forward(q, one, v, **mask)
    want = ops.window_attention_forward(q, one.contiguous(), v, **mask)
    assert torch.equal(got[0], want[0])


def test_window_gradient_of_broadcast_inputs():
    """Autograd sums the gradients of an expanded K/V and of a strided dout."""
    q, k, v = (t.requires_grad_() for t in heads(1, 70, 70, 4, 1, 64, torch.float16, seed=3))
    k2, v2 = k.detach().clone().requires_grad_(), v.detach().clone().requires_grad_()
    out = ops.window_attention(q, k.expand(1, 70, 2, 64), v.expand(1, 70, 2, 64), window=30)
    out.sum().backward()  # the gradient is an expanded scalar
    q2 = q.detach().clone().requires_grad_()
    ops.window_attention(q2, k2, v2, window=30).backward(torch.ones_like(out))
    check_device_status()
    assert torch.allclose(q.grad, q2.grad, rtol=2 ** -9, atol=2 ** -12)
    # two heads' gradients, each rounded once, against one rounded sum
    for a, b in ((k.grad, k2.grad), (v.grad, v2.grad)):
        assert torch.allclose(a, b, rtol=2 ** -8, atol=2 ** -8)


# ------------------------------------------------------------- window: values
def test_window_masked_places_may_hold_anything():
    """NaN and infinities in keys that a row does not see do not reach it:
    here no row sees keys [0, 40) any more."""
    q, k, v = heads(1, 60, 300, 4, 2, 64, torch.bfloat16, seed=4)
    want = ops.window_attention_forward(q, k, v, window=100)
    k[:, :40], v[:, :40] = math.nan, 0.0
    k[:, 5], k[:, 6] = math.inf, -math.inf
    got = ops.window_attention_forward(q, k, v, window=100)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    dout = normal(1, 60, 4, 64, seed=5, dtype=q.dtype)
    clean = k.clone()
    clean[:, :40] = 0
    a = ops.window_attention_backward(dout, q, clean, v, *want, window=100)
    k[:, :40] = 0
    v[:, :40] = torch.inf
    v[:, 3] = math.nan
    b = ops.window_attention_backward(dout, q, k, v, *want, window=100)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_window_infinities_and_nan_that_are_seen():
    q, k, v = heads(1, 140, 140, 2, 1, 64, torch.bfloat16, seed=6)
    q[0, 50, 0, 3] = math.nan
    out, lse = ops.window_attention_forward(q, k, v)
    bad = torch.isnan(out).any(-1)
    assert bad[0, 50, 0] and bad.sum() == 1 and torch.isnan(lse).sum() == 1
    k[0, 100] = math.nan  # seen by tokens 100 and later
    out, _ = ops.window_attention_forward(q, k, v)
    bad = torch.isnan(out).any(-1)
    assert bad[0, 100:].all() and not bad[0, :50].any()


def test_window_large_scores():
    """Scores that grow along the keys move the running maximum in every
    block; scores far apart leave one key."""
    q, k, v = heads(1, 600, 600, 2, 1, 64, torch.bfloat16, seed=7)
    k = (k * torch.linspace(0.1, 12, 600, device="cuda")[None, :, None, None]).to(k.dtype)
    u = torch.ones(64, device="cuda", dtype=q.dtype)
    q = q * 0.1 + u
    k = k * 0.05 + (torch.linspace(-8, 8, 600, device="cuda")[None, :, None, None] * u).to(k.dtype)
    check_window(q.contiguous(), k.contiguous(), v, None, 0,
                 normal(1, 600, 2, 64, seed=8, dtype=q.dtype) * 0.1)


def test_window_scale():
    q, k, v = heads(1, 200, 200, 2, 2, 128, torch.float16, seed=9)
    check_window(q, k, v, 90, 1, normal(1, 200, 2, 128, seed=10, dtype=q.dtype), scale=0.02)


# ----------------------------------------------------------- window: gradient
@pytest.mark.parametrize("window,sinks", [(None, 0), (17, 3)])
def test_window_gradient_against_differences(window, sinks):
    """Directional derivatives of the 64-bit forward by central differences
    against the kernel's gradients."""
    dtype = torch.float16
    q, k, v = heads(1, 75, 75, 3, 1, 64, dtype, seed=11)
    dout = normal(1, 75, 3, 64, seed=12, dtype=dtype)
    got, _ = check_window(q, k, v, window, sinks, dout)
    see = ref.visible(75, 75, window, sinks, "cuda")

    def f(q, k, v):
        return sum((ref.head(q[0, :, h], k[0, :, 0], v[0, :, 0], see, 0.125)["out"] *
                    dout[0, :, h].double()).sum() for h in range(3))

    x = [t.double() for t in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.sign(torch.randn(x[i].shape, generator=torch.Generator().manual_seed(i),
                                   dtype=torch.float64)).cuda()
        eps = 1e-5
        lo, hi = list(x), list(x)
        hi[i], lo[i] = x[i] + eps * d, x[i] - eps * d
        diff = ((f(*hi) - f(*lo)) / (2 * eps)).item()
        # error of each of n gradient elements at most 2 u of its size, of
        # either sign along d: sqrt(n) of them add up, 6 deviations allowed
        g = got[name].double()
        tol = 6 * 4 * ref.unit(dtype) * g.norm().item() + 1e-6 * abs(diff)
        assert abs((g * d).sum().item() - diff) <= tol


def test_window_gradient_is_reproducible():
    q, k, v = heads(2, 1500, 1500, 8, 2, 64, torch.bfloat16, seed=13)
    dout = normal(2, 1500, 8, 64, seed=14, dtype=q.dtype)
    out, lse = ops.window_attention_forward(q, k, v, window=128, sinks=4)
    first = ops.window_attention_backward(dout, q, k, v, out, lse, window=128, sinks=4)
    for _ in range(5):
        again = ops.window_attention_backward(dout, q, k, v, out, lse, window=128, sinks=4)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_window_autograd_and_streams():
    """Through autograd, on a stream that is not the tensors' own."""
    q, k, v = (t.requires_grad_() for t in heads(1, 320, 320, 4, 2, 128, torch.bfloat16, seed=15))
    dout = normal(1, 320, 4, 128, seed=16, dtype=torch.bfloat16)
    want, lse = ops.window_attention_forward(q, k, v, window=50, sinks=2)
    grads = ops.window_attention_backward(dout, q, k, v, want, lse, window=50, sinks=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.window_attention(q, k, v, window=50, sinks=2)
        out.backward(dout)
    torch.cuda.current_stream().wait_stream(side)
    check_device_status()
    assert torch.equal(out, want)
    for t, g in zip((q, k, v), grads):
        assert torch.equal(t.grad, g)


def test_window_in_a_graph():
    q, k, v = heads(1, 300, 300, 4, 2, 64, torch.bfloat16, seed=17)
    dout = normal(1, 300, 4, 64, seed=18, dtype=q.dtype)

    def step():
        out, lse = ops.window_attention_forward(q, k, v, window=64, sinks=2)
        return out, *ops.window_attention_backward(dout, q, k, v, out, lse, window=64, sinks=2)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step()
    q.copy_(normal(*q.shape, seed=19, dtype=q.dtype))
    want = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))


# ---------------------------------------------------------------------- paged
def cache(lengths, q_lens, hq, hk, d, page, dtype, seed=0, width=None, spare=3, fill=math.nan):
    """A paged problem: pages in random order, slots without a token hold
    ``fill``, table entries behind a sequence's pages are out of range."""
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // page) for n in lengths]
    pages = sum(per) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    width = width or max(1, max(per))
    table = torch.full((len(lengths), width), 1 << 30, dtype=torch.int32)
    table[:, ::2] = -7
    kp = torch.full((pages, page, hk, d), fill, dtype=dtype)
    vp = torch.full((pages, page, hk, d), fill, dtype=dtype)
    ks, vs, at = [], [], 0
    for b, n in enumerate(lengths):
        table[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
        k = torch.randn(n, hk, d, generator=g).to(dtype)
        v = torch.randn(n, hk, d, generator=g).to(dtype)
        ks.append(k)
        vs.append(v)
        slots = torch.arange(n)
        ids = table[b, slots // page].long()
        kp[ids, slots % page], vp[ids, slots % page] = k, v
    start = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    q = torch.randn(int(start[-1]), hq, d, generator=g).to(dtype)
    return {"q": q.cuda(), "k": kp.cuda(), "v": vp.cuda(), "table": table.cuda(),
            "start": start.cuda(), "len": torch.tensor(lengths, dtype=torch.int32).cuda(),
            "ks": ks, "vs": vs, "lengths": lengths, "q_lens": q_lens}


def plan_for(c, hq, hk, d, page, dtype, window=None, sinks=0, max_q=None, max_seqs=None):
    return ops.PagedAttention(heads_q=hq, heads_kv=hk, head_dim=d, page_size=page,
                              max_seqs=max_seqs or len(c["lengths"]),
                              max_q=max_q or max(1, max(c["q_lens"])), dtype=dtype,
                              window=window, sinks=sinks)


def attend(plan, c, **kw):
    return plan.attend(c["q"], c["k"], c["v"], c["table"], c["start"], c["len"], **kw)


def check_paged(c, out, lse, hq, hk, window, sinks, dtype):
    g, at = hq // hk, 0
    for b, (n, m) in enumerate(zip(c["lengths"], c["q_lens"])):
        see = ref.visible(m, n, window, sinks, "cuda")
        for h in range(hq):
            r = ref.head(c["q"][at:at + m, h], c["ks"][b][:, h // g].cuda(),
                         c["vs"][b][:, h // g].cuda(), see, out.shape[-1] ** -0.5)
            ref.within("out", out[at:at + m, h], r["out"], ref.bounds(r, dtype)["out"])
            fin = torch.isfinite(r["lse"])
            assert torch.equal(torch.isfinite(lse[at:at + m, h]), fin)
            if fin.any():
                assert (lse[at:at + m, h] - r["lse"])[fin].abs().max().item() < ref.R
        at += m


PAGED_CASES = [
    # lengths, new tokens, heads_q, heads_kv, dim, page, window, sinks
    ([1], [1], 1, 1, 64, 8, None, 0),
    ([777], [1], 8, 2, 128, 16, None, 0),
    ([128, 127, 129, 1], [1, 1, 1, 1], 4, 4, 64, 16, None, 0),
    ([300, 0, 17, 64], [1, 0, 1, 1], 6, 2, 128, 24, None, 0),       # an idle slot
    ([2000, 90], [1, 1], 16, 1, 64, 48, 200, 4),
    ([5000], [1], 4, 1, 128, 64, None, 0),                          # one unit over many SMs
    ([100, 40], [100, 40], 4, 2, 64, 32, None, 0),                  # prompts
    ([700, 333, 5], [130, 33, 5], 4, 2, 128, 16, None, 0),          # chunks
    ([900, 450, 12, 64], [200, 1, 12, 3], 14, 2, 64, 256, 100, 4),  # mixed, window
    ([600], [600], 1, 1, 64, 8, 50, 130),
    ([513, 1025], [70, 1], 3, 1, 128, 128, 64, 1),
    ([40], [60], 4, 2, 64, 16, None, 0),                            # tokens without a key
    ([1000] * 9, [64] * 9, 32, 8, 64, 16, None, 0),                 # whole units
    ([4096], [256], 8, 1, 128, 512, None, 0),                       # a page of four blocks
]


@pytest.mark.parametrize("case", PAGED_CASES, ids=lambda c: f"{c[0][:4]}-{c[1][:4]}-{c[2:]}")
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
def test_paged_attention(case, dtype):
    lengths, q_lens, hq, hk, d, page, window, sinks = case
    c = cache(lengths, q_lens, hq, hk, d, page, dtype, seed=len(lengths) + page)
    plan = plan_for(c, hq, hk, d, page, dtype, window, sinks)
    lse = torch.empty(c["q"].shape[:2], dtype=torch.float32, device="cuda")
    for _ in range(3):  # the plan's counters are back at zero each time
        out = attend(plan, c, lse=lse)
        check_device_status()
        check_paged(c, out, lse, hq, hk, window, sinks, dtype)


def test_paged_random_batches_of_one_plan():
    """Calls of one plan with other batches, lengths and widths."""
    r = random.Random(3)
    hq, hk, d, page = 8, 2, 64, 16
    plan = ops.PagedAttention(heads_q=hq, heads_kv=hk, head_dim=d, page_size=page, max_seqs=20,
                              max_q=90, dtype=torch.bfloat16, window=150, sinks=5)
    for i in range(15):
        n = r.randint(1, 20)
        lengths = [r.choice((0, 1, r.randint(1, 900))) for _ in range(n)]
        q_lens = [min(m, r.choice((1, 1, r.randint(1, 90)))) for m in lengths]
        if sum(q_lens) == 0:
            continue
        c = cache(lengths, q_lens, hq, hk, d, page, torch.bfloat16, seed=i,
                  width=max(-(-max(lengths) // page), 1) + r.randint(0, 5))
        lse = torch.empty(c["q"].shape[:2], dtype=torch.float32, device="cuda")
        out = attend(plan, c, lse=lse)
        check_device_status()
        check_paged(c, out, lse, hq, hk, 150, 5, torch.bfloat16)


def test_paged_many_short_sequences():
    """More sequences than a launch cuts into stretches."""
    n = 1300
    lengths = [1 + (i * 7) % 40 for i in range(n)]
    c = cache(lengths, [1] * n, 2, 1, 64, 8, torch.bfloat16, seed=21)
    plan = plan_for(c, 2, 1, 64, 8, torch.bfloat16)
    lse = torch.empty(c["q"].shape[:2], dtype=torch.float32, device="cuda")
    out = attend(plan, c, lse=lse)
    check_device_status()
    check_paged(c, out, lse, 2, 1, None, 0, torch.bfloat16)


def test_paged_equals_dense():
    """A chunk over a cache sees what the dense form's last rows see."""
    b, s, hq, hk, d, page = 2, 400, 8, 2, 128, 16
    q, k, v = heads(b, s, s, hq, hk, d, torch.bfloat16, seed=22)
    want, _ = ops.window_attention_forward(q, k, v, window=90, sinks=4)
    per = s // page
    kp, vp = (t.reshape(b * per, page, hk, d) for t in (k, v))
    table = torch.arange(b * per, dtype=torch.int32, device="cuda").view(b, per)
    plan = ops.PagedAttention(heads_q=hq, heads_kv=hk, head_dim=d, page_size=page, max_seqs=b,
                              max_q=s, dtype=torch.bfloat16, window=90, sinks=4)
    for chunk in (1, 37, 256):
        start = torch.tensor([0, chunk, 2 * chunk], dtype=torch.int32, device="cuda")
        out = plan.attend(q[:, -chunk:].reshape(-1, hq, d), kp, vp, table, start,
                          torch.full((b,), s, dtype=torch.int32, device="cuda"))
        check_device_status()
        r = want[:, -chunk:].reshape(-1, hq, d).float()
        # two roundings of P and of the result, over at most 1 in weight
        assert ((out.float() - r).abs() <= 4 * 2.0 ** -8 * v.abs().max().float()).all()


def test_paged_offsets_past_32_bits():
    """The last pages of a cache of more than 2^32 elements."""
    hk, d, page = 8, 128, 64
    pages = (1 << 32) // (hk * d * page) + 40
    kp = torch.empty(pages, page, hk, d, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    n = 200
    ids = torch.tensor([pages - 1, 0, pages - 3, pages // 2], dtype=torch.int32)
    k, v = normal(n, hk, d, seed=23, dtype=kp.dtype), normal(n, hk, d, seed=24, dtype=kp.dtype)
    plan = ops.PagedAttention(heads_q=8, heads_kv=hk, head_dim=d, page_size=page, max_seqs=1,
                              max_q=n, dtype=torch.bfloat16)
    table = ids[None].cuda()
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    whole = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    plan.append(k, v, kp, vp, table, whole, length)
    slots = torch.arange(n)
    at = ids[slots // page].long().cuda(), (slots % page).cuda()
    assert torch.equal(kp[at], k) and torch.equal(vp[at], v)
    q = normal(3, 8, d, seed=25, dtype=kp.dtype)
    last = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    lse = torch.empty(3, 8, dtype=torch.float32, device="cuda")
    out = plan.attend(q, kp, vp, table, last, length, lse=lse)
    check_device_status()
    c = {"q": q, "ks": [k], "vs": [v], "lengths": [n], "q_lens": [3]}
    check_paged(c, out, lse, 8, hk, None, 0, torch.bfloat16)


def test_paged_strided_cache_and_output():
    """K and V interleaved in one tensor, (page, head, slot, dim) storage, an
    output inside a wider tensor."""
    hq, hk, d, page = 4, 2, 64, 16
    c = cache([300, 50], [20, 1], hq, hk, d, page, torch.float16, seed=26)
    plan = plan_for(c, hq, hk, d, page, torch.float16)
    want = attend(plan, c)
    both = torch.stack((c["k"], c["v"]), 1)
    got = plan.attend(c["q"], both[:, 0], both[:, 1], c["table"], c["start"], c["len"])
    assert torch.equal(got, want)
    kt, vt = (c[n].transpose(1, 2).contiguous().transpose(1, 2) for n in "kv")
    wide = torch.zeros(21, hq + 3, d + 8, dtype=torch.float16, device="cuda")
    got = plan.attend(c["q"], kt, vt, c["table"], c["start"], c["len"], out=wide[:, 1:hq + 1, :d])
    assert torch.equal(got, want)
    assert not wide[:, :, d:].any() and not wide[:, 0].any() and not wide[:, hq + 1:].any()


def test_paged_lengths_that_do_not_fit_are_reported():
    """Device lengths the host has not seen: the sequence is skipped and the
    device status says so; the others are computed."""
    hq, hk, d, page = 2, 1, 64, 16
    c = cache([64, 64], [2, 2], hq, hk, d, page, torch.bfloat16, seed=27)
    plan = plan_for(c, hq, hk, d, page, torch.bfloat16)
    want = attend(plan, c)
    c["len"][0] = 65  # one more than the table has room for
    out = attend(plan, c, out=torch.full_like(want, 7.0))
    with pytest.raises(RuntimeError, match="0x20"):
        check_device_status()
    assert torch.equal(out[2:], want[2:]) and (out[:2] == 7.0).all()
    c["len"][0] = 64
    assert torch.equal(attend(plan, c), want)
    check_device_status()


def test_paged_plans_on_two_streams():
    hq, hk, d, page = 8, 2, 128, 16
    cs = [cache([3000, 77], [1, 1], hq, hk, d, page, torch.bfloat16, seed=s) for s in (28, 29)]
    plans = [plan_for(c, hq, hk, d, page, torch.bfloat16) for c in cs]
    want = [attend(p, c) for p, c in zip(plans, cs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = []
    for _ in range(20):
        got = []
        for s, p, c in zip(streams, plans, cs):
            with torch.cuda.stream(s):
                got.append(attend(p, c))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_paged_in_a_graph():
    """A captured decode step follows the lengths on the device."""
    hq, hk, d, page = 4, 2, 64, 16
    c = cache([500, 200], [1, 1], hq, hk, d, page, torch.bfloat16, seed=30)
    plan = plan_for(c, hq, hk, d, page, torch.bfloat16)
    attend(plan, c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = attend(plan, c)
    for lengths in ([499, 64], [1, 200], [500, 200]):
        c["len"].copy_(torch.tensor(lengths, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, attend(plan, c))


# --------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16"])
@pytest.mark.parametrize("lengths,q_lens,hk,d,page", [
    ([1], [1], 1, 64, 8),
    ([100, 0, 7, 33], [1, 0, 7, 20], 2, 128, 16),
    ([300, 300], [300, 129], 8, 64, 24),
    ([65] * 40, [1] * 40, 4, 128, 64),
])
def test_append_writes_the_new_rows_alone(lengths, q_lens, hk, d, page, dtype):
    c = cache(lengths, q_lens, hk, hk, d, page, dtype, seed=31, fill=5.0)
    plan = plan_for(c, hk, hk, d, page, dtype)
    t = sum(q_lens)
    fused = normal(t, 2 * hk, d, seed=32, dtype=dtype)
    k, v = fused[:, :hk], fused[:, hk:]
    want_k, want_v, at = c["k"].clone(), c["v"].clone(), 0
    table = c["table"].cpu()
    for b, (n, m) in enumerate(zip(lengths, q_lens)):
        slots = torch.arange(n - m, n)
        ids = table[b, slots // page].long().cuda(), (slots % page).cuda()
        want_k[ids], want_v[ids] = k[at:at + m], v[at:at + m]
        at += m
    plan.append(k, v, c["k"], c["v"], c["table"], c["start"], c["len"])
    torch.cuda.synchronize()
    assert torch.equal(c["k"], want_k) and torch.equal(c["v"], want_v)


def test_append_skips_slots_and_pages_outside():
    c = cache([40, 40], [8, 8], 1, 1, 64, 16, torch.bfloat16, seed=33, fill=5.0)
    plan = plan_for(c, 1, 1, 64, 16, torch.bfloat16)
    before = c["k"].clone()
    k = normal(16, 1, 64, seed=34, dtype=torch.bfloat16)
    c["table"][0, 2] = 1 << 20     # a page that does not exist
    c["len"][1] = 4                # more new tokens than keys: slots below 0
    plan.append(k, k, c["k"], c["v"], c["table"], c["start"], c["len"])
    torch.cuda.synchronize()
    changed = (c["k"] != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [int(c["table"][1, 0])]
    assert torch.equal(c["k"][changed[0], :4], k[12:])


def test_append_then_attend_serves_the_dense_result():
    """A prompt in chunks, then single tokens, against the dense form."""
    hq, hk, d, page, s = 6, 2, 64, 16, 150
    q, k, v = heads(1, s, s, hq, hk, d, torch.bfloat16, seed=35)
    want, _ = ops.window_attention_forward(q, k, v, window=40, sinks=2)
    pages = -(-s // page)
    kp = torch.full((pages, page, hk, d), math.nan, dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    table = torch.randperm(pages).to(torch.int32)[None].cuda()
    plan = ops.PagedAttention(heads_q=hq, heads_kv=hk, head_dim=d, page_size=page, max_seqs=1,
                              max_q=64, dtype=torch.bfloat16, window=40, sinks=2)
    at = 0
    for m in [64, 50, 30] + [1] * 6:
        start = torch.tensor([0, m], dtype=torch.int32, device="cuda")
        length = torch.tensor([at + m], dtype=torch.int32, device="cuda")
        plan.append(k[0, at:at + m], v[0, at:at + m], kp, vp, table, start, length)
        out = plan.attend(q[0, at:at + m], kp, vp, table, start, length)
        check_device_status()
        err = (out.float() - want[0, at:at + m].float()).abs().max().item()
        assert err <= 4 * 2.0 ** -8 * v.abs().max().item()
        at += m


# ------------------------------------------------------------------- refusals
def refused(match, f, *a, **kw):
    with pytest.raises(KernelBuildError, match=match):
        f(*a, **kw)


def test_window_refusals():
    q, k, v = heads(1, 8, 8, 4, 2, 64, torch.bfloat16)
    f = ops.window_attention_forward
    refused("CUDA tensor", f, q.cpu(), k, v)
    refused("float16 or bfloat16", f, q.float(), k, v)
    refused("must be torch.bfloat16", f, q, k.half(), v)
    refused("4 dimensions", f, q[0], k, v)
    refused("belong together", f, q, k, v[:, :7])
    refused("belong together", f, q, k[..., :32], v[..., :32])
    refused("multiple of heads_kv", f, q[:, :, :3], k, v)
    refused("head_dim must be 64 or 128", f, *(t[..., :32].contiguous() for t in (q, k, v)))
    refused("window must be at least 1", f, q, k, v, window=0)
    refused("sinks must not be negative", f, q, k, v, sinks=-1)
    for scale in (0.0, -1.0, math.nan):
        refused("scale must be positive", f, q, k, v, scale=scale)
    refused("finite", f, q, k, v, scale=math.inf)
    refused("out must have shape", f, q, k, v, out=q[:, :4])
    many = normal(1, 2, 129, 64, seed=1, dtype=torch.bfloat16)
    refused("128 query heads", f, many, k[:, :2, :1], v[:, :2, :1])
    out, lse = f(q, k, v)
    g = ops.window_attention_backward
    refused("lse has shape", g, q, q, k, v, out, lse[:, :4])
    refused("lse must be torch.float32", g, q, q, k, v, out, lse.half())
    refused("dout has shape", g, q[:, :4], q, k, v, out, lse)
    overlap = torch.empty(1, 8, 1, 64, dtype=q.dtype, device="cuda").expand(1, 8, 4, 64)
    refused("rows overlap", f, q, k, v, out=overlap)


def test_paged_refusals():
    c = cache([40], [4], 4, 2, 64, 16, torch.bfloat16, seed=36)
    make = dict(heads_q=4, heads_kv=2, head_dim=64, page_size=16, max_seqs=1, max_q=4,
                dtype=torch.bfloat16)
    refused("page_size must be a multiple of 8", ops.PagedAttention, **{**make, "page_size": 12})
    refused("head_dim", ops.PagedAttention, **{**make, "head_dim": 80})
    refused("float16 or bfloat16", ops.PagedAttention, **{**make, "dtype": torch.float32})
    refused("multiple of heads_kv", ops.PagedAttention, **{**make, "heads_q": 5})
    refused("at least 1", ops.PagedAttention, **{**make, "max_q": 0})
    plan = ops.PagedAttention(**make)
    args = [c["q"], c["k"], c["v"], c["table"], c["start"], c["len"]]

    def bad(i, t, match):
        refused(match, plan.attend, *args[:i], t, *args[i + 1:])

    bad(0, c["q"][:, :3], "q has shape")
    bad(0, c["q"].half(), "q must be")
    bad(1, c["k"][:, :8], "k_pages has shape")
    bad(1, c["k"][:2], "different numbers of pages")
    bad(3, c["table"].long(), "page_table must be torch.int32")
    bad(3, c["table"].repeat(2, 1), "2 sequences")
    bad(4, c["start"][:1], "0 in q_start")
    bad(5, c["len"].cpu(), "CUDA tensor")
    refused("out must have shape", plan.attend, *args, out=c["q"][:2])
    refused("k has shape", plan.append, c["q"], c["q"], *args[1:])


# ----------------------------------------------------- through build_callable
def test_build_callable_runs_the_operators():
    q, k, v = heads(2, 100, 100, 4, 2, 64, torch.bfloat16, seed=37)
    dout = normal(2, 100, 4, 64, seed=38, dtype=q.dtype)
    cfg = {"dtype": "bfloat16", "window": 30, "sinks": 2}
    shape = (2, 100, 100, 4, 2, 64)
    kc = build_callable("attention_window", shape, cfg, (q, k, v))
    warm_compile(kc)
    want, lse = ops.window_attention_forward(q, k, v, window=30, sinks=2)
    assert torch.equal(kc.fn(), want) and kc.fn().data_ptr() == kc.fn().data_ptr()
    kg = build_callable("attention_window_grad", shape, cfg, (dout, q, k, v, want, lse))
    for a, b in zip(kg.fn(), ops.window_attention_backward(dout, q, k, v, want, lse, window=30,
                                                           sinks=2)):
        assert torch.equal(a, b)
    c = cache([64, 30], [3, 1], 4, 2, 64, 16, torch.bfloat16, seed=39)
    shape = (2, 3, 16, 4, 2, 64)
    paged = build_callable("attention_paged", shape, cfg,
                           (c["q"], c["k"], c["v"], c["table"], c["start"], c["len"]))
    warm_compile(paged)
    assert torch.equal(paged.fn(), attend(plan_for(c, 4, 2, 64, 16, torch.bfloat16, 30, 2), c))
    new = normal(4, 2, 64, seed=40, dtype=torch.bfloat16)
    app = build_callable("cache_append", shape, cfg,
                         (new, new, c["k"], c["v"], c["table"], c["start"], c["len"]))
    kp, vp = app.fn()
    last = int(c["table"][1, 1])
    assert torch.equal(kp[last, 13], new[3]) and torch.equal(vp[last, 13], new[3])
    for bad_cfg, bad_shape, ins, match in (
            ({**cfg, "dtype": "float32"}, shape, (q, k, v), "dtype must be"),
            (cfg, (2, 100), (q, k, v), "shape needs 6"),
            (cfg, (2, 99, 100, 4, 2, 64), (q, k, v), "q has shape"),
            (cfg, (2, 100, 100, 4, 2, 64), (q, k), "takes 3 inputs"),
            (cfg, (2, 100, 100, 4, 2, 64), (q.half(), k, v), "does not match")):
        refused(match, build_callable, "attention_window", bad_shape, bad_cfg, ins)
