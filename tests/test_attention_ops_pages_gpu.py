"""Device data of paged calls that does not fit the buffers: what is computed
or written all the same, and what the device status says."""

import pytest
import torch

from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200 import _lib
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
