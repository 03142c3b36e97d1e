"""Device data of paged calls that does not fit the buffers: what is computed
or written all the same, and what the device status says."""

import pytest
import torch

from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200 import _lib
from gpu_optimizer_b200.runner import KernelBuildError
from test_attention_ops_gpu import normal

pytestmark = pytest.mark.gpu


def flags():
    """Flags of the device's error word since the last look at it."""
    return _lib.device_status(torch.cuda.current_stream().cuda_stream)[1]


def plan(hq, hk, d, page, seqs, max_q, **mask):
    return ops.PagedAttention(heads_q=hq, heads_kv=hk, head_dim=d, page_size=page, max_seqs=seqs,
                              max_q=max_q, dtype=torch.bfloat16, **mask)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("entry", [0, -1, 5])
def test_attend_of_a_cache_without_pages_reads_zeros(entry):
    p = plan(4, 2, 64, 16, 1, 3)
    q = normal(3, 4, 64, seed=50, dtype=torch.bfloat16)
    none = torch.empty(0, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(3, 4, dtype=torch.float32, device="cuda")
    out = p.attend(q, none, none, ints(entry, entry)[None], ints(0, 3), ints(20), lse=lse)
    flags()
    # scores of 0 over 18, 19 and 20 keys
    want = torch.tensor([18.0, 19.0, 20.0], device="cuda").log()[:, None].expand(3, 4)
    assert not out.any() and torch.allclose(lse, want, rtol=1e-5)


def written(pages, before):
    """Pages that have changed."""
    return (pages != before).flatten(1).any(1).nonzero().flatten().tolist()


@pytest.mark.parametrize("start,length,kept", [
    ([0, 4, 8], [40, 49], [0]),      # one key more than the table has room for
    ([0, 4, 8], [40, -1], [0]),
    ([0, 4, 9], [40, 40], [0]),      # ends behind the rows
    ([-1, 4, 8], [40, 40], [1]),
    ([0, 6, 4], [40, 40], [0]),      # descending
])
def test_append_reports_and_skips_sequences_that_do_not_fit(start, length, kept):
    """As the attention does: the same sequences, the same status."""
    p = plan(1, 1, 64, 16, 2, 8)
    table = ints(0, 1, 2, 3, 4, 5).view(2, 3)
    kp = torch.zeros(6, 16, 1, 64, dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    new = normal(8, 1, 64, seed=51, dtype=torch.bfloat16)
    flags()
    p.append(new, new, kp, vp, table, ints(*start), ints(*length))
    assert flags() == 0x20
    assert written(kp, torch.zeros_like(kp)) == [3 * b + 2 for b in kept]
    assert torch.equal(kp, vp)
    p.attend(new, kp, vp, table, ints(*start), ints(*length))
    assert flags() == 0x20


def test_append_takes_chunks_longer_than_the_attention():
    """max_q bounds the attention's tiles alone."""
    p = plan(1, 1, 64, 16, 1, 2)
    kp = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    new = normal(20, 1, 64, seed=52, dtype=torch.bfloat16)
    flags()
    p.append(new, new, kp, vp, ints(0, 1)[None], ints(0, 20), ints(20))
    assert flags() == 0 and torch.equal(kp.flatten(0, 1)[:20], new)


def test_append_of_tokens_in_front_of_the_first_key():
    """kv_len < q_len: tokens without a position have no slot, which is no error."""
    p = plan(1, 1, 64, 16, 1, 8)
    kp = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    new = normal(8, 1, 64, seed=53, dtype=torch.bfloat16)
    flags()
    p.append(new, new, kp, vp, ints(0)[None], ints(0, 8), ints(3))
    assert flags() == 0 and torch.equal(kp[0, :3], new[5:]) and not kp[0, 3:].any()


@pytest.mark.parametrize("max_q", [1, 40])
@pytest.mark.parametrize("window,slot,reported", [
    (None, 0, True), (None, 9, True), (None, 10, False),  # entry 10: behind the last key
    (30, 0, True), (30, 1, False), (30, 6, False), (30, 9, True),
])
def test_attend_reports_seen_pages_outside_the_cache(max_q, window, slot, reported):
    """Entries of pages without a visible key may be anything."""
    p = plan(4, 2, 64, 16, 1, max_q, window=window, sinks=4 if window else 0)
    n, m = 155, min(max_q, 5)
    kp = normal(12, 16, 2, 64, seed=54, dtype=torch.bfloat16)
    vp = normal(12, 16, 2, 64, seed=55, dtype=torch.bfloat16)
    q = normal(m, 4, 64, seed=56, dtype=torch.bfloat16)
    table = torch.arange(12, dtype=torch.int32, device="cuda")[None].clone()
    flags()
    want = p.attend(q, kp, vp, table, ints(0, m), ints(n))
    assert flags() == 0
    for entry in (-1, 12, 1 << 30):
        table[0, slot] = entry
        out = p.attend(q, kp, vp, table, ints(0, m), ints(n))
        assert flags() == (0x20 if reported else 0)
        assert torch.isfinite(out).all() and torch.equal(out, want) != reported


def test_attend_reads_a_cache_whose_heads_are_one():
    """A cache with one kv head, expanded: read in place by attend, refused by
    append, which would write its rows over each other."""
    p = plan(4, 4, 64, 16, 1, 2)
    k = normal(5, 16, 1, 64, seed=57, dtype=torch.bfloat16)
    v = normal(5, 16, 1, 64, seed=58, dtype=torch.bfloat16)
    q = normal(2, 4, 64, seed=59, dtype=torch.bfloat16)
    where = ints(4, 2, 0, 1, 3)[None], ints(0, 2), ints(70)
    flags()
    got = p.attend(q, k.expand(-1, -1, 4, -1), v.expand(-1, -1, 4, -1), *where)
    want = p.attend(q, k.repeat(1, 1, 4, 1), v.repeat(1, 1, 4, 1), *where)
    assert flags() == 0 and torch.equal(got, want)
    with pytest.raises(KernelBuildError, match="rows overlap"):
        p.append(normal(2, 4, 64, seed=60, dtype=torch.bfloat16), q, k.expand(-1, -1, 4, -1),
                 v.expand(-1, -1, 4, -1), *where)
