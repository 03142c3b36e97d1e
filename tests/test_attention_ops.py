"""Window / paged attention operators on the host: record layouts, argument
checks of the C entry points (which come before any CUDA call), the plain
forms' own consistency."""

import ctypes
import math

import pytest
import torch

import attention_ops_ref as ref
from gpu_optimizer_b200 import _lib
from gpu_optimizer_b200 import attention_ops as ops
from gpu_optimizer_b200.runner import KernelBuildError, build_callable


def window(**kw):
    a = dict(dtype=3, head_dim=64, heads_q=4, heads_kv=2, batch=1, q_len=8, kv_len=8, window=0,
             sinks=0, scale=0.0, reserved=0)
    return _lib.GpoWindowArgs(**{**a, **kw})


def paged(**kw):
    a = dict(dtype=3, head_dim=64, heads_q=4, heads_kv=2, num_seqs=2, tokens=8, max_q=4,
             num_pages=5, page_size=16, table_width=4, table_stride=4, window=0, sinks=0,
             scale=0.0, reserved=0)
    return _lib.GpoPagedArgs(**{**a, **kw})


def call(name, *args):
    log = ctypes.create_string_buffer(256)
    rc = getattr(_lib.load(), name)(*args, log, 256)
    return rc, log.value.decode()


def test_record_layouts():
    assert ctypes.sizeof(_lib.GpoHeads) == 32
    assert ctypes.sizeof(_lib.GpoWindowArgs) == 4 * 4 + 5 * 8 + 8 + 4 * 32 + 8 + 4 * 32 + 16
    assert ctypes.sizeof(_lib.GpoPagedArgs) == 4 * 4 + 9 * 8 + 8 + 6 * 32 + 6 * 8


@pytest.mark.parametrize("bad,why", [
    ({"dtype": 0}, "float16 or bfloat16"), ({"head_dim": 80}, "head_dim"),
    ({"heads_q": 5}, "multiple of heads_kv"), ({"heads_kv": 0}, "multiple of heads_kv"),
    ({"heads_q": 258, "heads_kv": 2}, "128 query heads"), ({"window": -1}, "negative"),
    ({"sinks": -1}, "negative"), ({"scale": -1.0}, "scale"), ({"scale": math.nan}, "scale"),
    ({"scale": math.inf}, "scale"), ({"q_len": -1}, "lengths"), ({"kv_len": 1 << 31}, "lengths"),
    ({"batch": 70000}, "batch"), ({"reserved": 1}, "reserved"),
])
def test_window_arguments_are_refused(bad, why):
    rc, log = call("gpo_window_workspace", window(**bad), ctypes.c_uint64(0))
    assert rc in (_lib.BAD_ARGS, _lib.BAD_CONFIG) and why in log
    rc, log = call("gpo_window_attention", window(**bad), None)
    assert rc in (_lib.BAD_ARGS, _lib.BAD_CONFIG) and why in log


@pytest.mark.parametrize("bad,why", [
    ({"page_size": 4}, "page_size"), ({"page_size": 20}, "page_size"),
    ({"num_seqs": -1}, "num_seqs"), ({"tokens": 1 << 31}, "tokens"),
    ({"table_stride": 3}, "table_stride"), ({"table_width": 1 << 28}, "table_width"),
    ({"num_pages": -1}, "num_pages"), ({"head_dim": 96}, "head_dim"),
])
def test_paged_arguments_are_refused(bad, why):
    for name in ("gpo_paged_attention", "gpo_cache_append"):
        rc, log = call(name, paged(**bad), None)
        assert rc in (_lib.BAD_ARGS, _lib.BAD_CONFIG) and why in log


def heads(ptr, *strides):
    return _lib.GpoHeads(ptr, *strides)


def test_pointers_and_strides_are_refused():
    ok = heads(4096, 2048, 256, 64)
    kv = heads(4096, 1024, 128, 64)
    good = dict(q=ok, k=kv, v=kv, out=ok)
    for bad, why in ((dict(q=heads(0, 2048, 256, 64)), "q is null"),
                     (dict(k=heads(4100, 1024, 128, 64)), "k is not 16-byte aligned"),
                     (dict(v=heads(4096, 1024, 100, 64)), "v: strides"),
                     (dict(q=heads(4096, 2048, -256, 64)), "q: strides"),
                     (dict(q=heads(4096, 2048, 1 << 40, 64)), "q: strides"),
                     (dict(out=heads(4096, 2048, 256, 0)), "out: written rows overlap")):
        rc, log = call("gpo_window_attention", window(**{**good, **bad}), None)
        assert rc == _lib.BAD_ARGS and why in log, log
    grads = dict(good, dout=ok, dq=ok, dk=kv, dv=kv)
    rc, log = call("gpo_window_attention_grad", window(**grads), None)
    assert rc == _lib.BAD_ARGS and "lse is null" in log
    rc, log = call("gpo_window_attention_grad", window(**grads, lse=4096, workspace=256,
                                                       workspace_bytes=10), None)
    assert rc == _lib.BAD_ARGS and "workspace" in log
    pages = dict(k_pages=heads(4096, 2048, 128, 64), v_pages=heads(4096, 2048, 128, 64),
                 q=heads(4096, 0, 256, 64), out=heads(4096, 0, 256, 64))
    rc, log = call("gpo_paged_attention", paged(**pages), None)
    assert rc == _lib.BAD_ARGS and "page_table" in log
    rc, log = call("gpo_paged_attention", paged(**pages, page_table=64, q_start=64, kv_len=64),
                   None)
    assert rc == _lib.BAD_ARGS and "workspace" in log
    rc, log = call("gpo_cache_append", paged(**pages, page_table=64, q_start=64, kv_len=64), None)
    assert rc == _lib.BAD_ARGS and "k_new is null" in log


def test_empty_problems_need_no_device():
    assert call("gpo_window_attention", window(batch=0), None) == (_lib.OK, "")
    assert call("gpo_window_attention", window(q_len=0), None) == (_lib.OK, "")
    assert call("gpo_window_attention_grad", window(q_len=0, kv_len=0), None) == (_lib.OK, "")
    assert call("gpo_paged_attention", paged(tokens=0), None) == (_lib.OK, "")
    assert call("gpo_cache_append", paged(num_seqs=0), None) == (_lib.OK, "")


def test_workspaces():
    size = ctypes.c_uint64(0)
    assert call("gpo_window_workspace", window(), size)[0] == _lib.OK
    assert size.value == 256 + 2 * 1024  # counter, statistics of one tile per kv head
    assert call("gpo_window_workspace", window(q_len=1000, kv_len=1000, window=100, sinks=4),
                size)[0] == _lib.OK
    # 64 tokens a tile: 16 tiles; tokens behind the window of the first key
    # tile: tiles 4 .. 15 in pieces of 4; sums of 4 keys, 1 + 3 pieces, dk and dv
    assert size.value == 256 + 2 * 16 * 1024 + 2 * 4 * 4 * 2 * 64 * 4
    small = ctypes.c_uint64(0)
    assert call("gpo_paged_workspace", paged(), size)[0] == _lib.OK
    assert call("gpo_paged_workspace", paged(num_seqs=1, tokens=1), small)[0] == _lib.OK
    assert 0 < small.value <= size.value  # a call never needs more than its plan


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(KernelBuildError, match="CUDA tensor"):
        ops.window_attention_forward(q, q, q)
    with pytest.raises(KernelBuildError, match="CUDA tensors"):
        build_callable("attention_window", (1, 4, 4, 2, 2, 64), {"dtype": "bfloat16"}, (q, q, q))
    with pytest.raises(KernelBuildError, match="no B200 kernel family"):
        build_callable("attention_unknown", (1,), {}, (q,))


def test_plain_form_of_the_tests():
    """The 64-bit form against torch's own softmax and autograd."""
    torch.manual_seed(0)
    q, k, v = (torch.randn(n, 64, dtype=torch.float64, requires_grad=True) for n in (30, 40, 40))
    do = torch.randn(30, 64, dtype=torch.float64)
    see = ref.visible(30, 40, 12, 3)
    out = torch.softmax((q @ k.T / 8).masked_fill(~see, -math.inf), -1) @ v
    out.backward(do)
    r = ref.head(q.detach(), k.detach(), v.detach(), see, 1 / 8, do)
    for a, b in ((r["out"], out), (r["dq"], q.grad), (r["dk"], k.grad), (r["dv"], v.grad)):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-12)
    # p = 15 (row 5 of 30 over 40): window 4..15, sinks 0..2
    assert see[5].nonzero().flatten().tolist() == [0, 1, 2, *range(4, 16)]
