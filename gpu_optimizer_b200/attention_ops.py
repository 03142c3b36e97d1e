"""Window attention with sinks (forward and gradient) and paged attention.

Operators for models whose attention the search tasks of this package do not
cover: grouped heads, strided tensors, a sliding window with sink tokens, a
gradient, and a paged K/V cache.  They run on ``libgpo.so`` (include/gpo.h)
like the tasks do; ``runner.build_callable`` builds them too, under the names
``attention_window``, ``attention_window_grad``, ``attention_paged`` and
``cache_append``.

* ``window_attention``            differentiable; what a training step calls
* ``window_attention_forward``    -> (out, log-sum-exp)
* ``window_attention_backward``   -> (dq, dk, dv)
* ``PagedAttention``              plan of a serving loop: ``append`` writes a
  chunk's K/V to the cache pages, ``attend`` reads them

Mask: token i of a sequence with q_len new tokens and kv_len keys stands at
p = i + kv_len - q_len and sees key j iff j <= p and (p - j < window or
j < sinks).  A token that sees no key gives 0 and a log-sum-exp of -inf.

Layouts: q, out (batch, tokens, heads_q, head_dim); k, v (batch, tokens,
heads_kv, head_dim); heads_q a multiple of heads_kv; float16 or bfloat16;
head_dim 64 or 128.  Any strides whose rows of head_dim are contiguous and
16-byte aligned are read in place (slices of a fused projection, transposed
views); others are copied first.

P and dS enter the tensor cores in the inputs' type (every sum is fp32).  With
float16, dS below 2^-24 vanishes: scale the loss, as for any float16 training.

Everything runs on torch's current stream and, but for making a plan, never
synchronises.  A refused
argument raises ``KernelBuildError`` with the library's reason, before
anything is launched; a launch that fails raises ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import importlib

import torch

from . import _lib
from .runner import KernelBuildError

_ops = None  # the native binding, once loaded


def _native():
    """The binding (csrc/py_ops.cpp); raises KernelBuildError if it is not
    built: there is no fallback."""
    global _ops
    if _ops is None:
        try:
            abi = _lib.load().gpo_abi_version()
            ops = importlib.import_module(__package__ + "._ops")
            if ops.ABI_VERSION != abi:
                raise _lib.LibraryMissing(f"_ops.so is built for ABI {ops.ABI_VERSION}, "
                                          f"libgpo.so has {abi}")
        except (_lib.LibraryMissing, ImportError) as e:
            raise KernelBuildError(str(e), log=str(e)) from e
        ops.set_refused(KernelBuildError)
        _ops = ops
    return _ops


class _NoGradient(torch.autograd.Function):
    """Results (in a list, which torch does not look into) of a call that has
    no gradient, for inputs that need one."""

    @staticmethod
    def forward(ctx, call, results, *inputs):
        ctx.call = call
        return tuple(r.detach() for r in results)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.call} has no gradient; window_attention is the differentiable "
                           "form (call under torch.no_grad() where none is wanted)")


def window_attention_forward(q, k, v, *, window: int | None = None, sinks: int = 0,
                             scale: float | None = None, out=None, lse=None):
    """(out, lse): attention of q over k, v, and each row's log-sum-exp of
    scaled scores, fp32 (batch, q_len, heads_q).  ``out`` and ``lse`` may name
    the tensors to write.  Not differentiable (``window_attention`` is): a
    backward pass that reaches the results raises."""
    results = (_ops or _native()).window_forward(q, k, v, window, sinks, scale, out, lse)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _NoGradient.apply("window_attention_forward", [*results], q, k, v)
    return results


def window_attention_backward(dout, q, k, v, out, lse, *, window: int | None = None,
                              sinks: int = 0, scale: float | None = None, grads=None):
    """(dq, dk, dv) from the output's gradient and what the forward returned.
    ``grads`` may name the three tensors to write.

    Sums run in a fixed order: the same inputs give the same bits.  Not
    differentiable once more.
    """
    results = (_ops or _native()).window_backward(dout, q, k, v, out, lse, window, sinks, scale,
                                                  grads)
    if torch.is_grad_enabled() and (dout.requires_grad or q.requires_grad or k.requires_grad
                                    or v.requires_grad):
        return _NoGradient.apply("window_attention_backward", [*results], dout, q, k, v)
    return results


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale):
        out, lse = window_attention_forward(q, k, v, window=window, sinks=sinks, scale=scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.mask = {"window": window, "sinks": sinks, "scale": scale}
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        return (*window_attention_backward(dout, *ctx.saved_tensors, **ctx.mask), None, None, None)


def window_attention(q, k, v, *, window: int | None = None, sinks: int = 0,
                     scale: float | None = None) -> torch.Tensor:
    """Differentiable attention of q (batch, q_len, heads_q, head_dim) over
    k, v (batch, kv_len, heads_kv, head_dim)."""
    return _WindowAttention.apply(q, k, v, window, sinks, scale)


class PagedAttention:
    """Plan of attention over a paged K/V cache: fixed heads, page size, mask
    and the most sequences and new tokens per sequence of a call.

    The cache is two tensors (num_pages, page_size, heads_kv, head_dim).
    Per call, ``page_table`` (int32, seqs x width) names the page of every
    ``page_size`` slots of a sequence, ``q_start`` (int32, seqs + 1) the first
    row of each sequence in the packed rows, and ``kv_len`` (int32, seqs) its
    keys, new tokens included.  All stay on the device and are not read by
    the host; a sequence whose lengths do not fit the buffers is skipped and
    reported by ``runner.check_device_status``.  Page table entries behind a
    sequence's last key, and those of pages no token sees any more, are not
    read as pages.  An entry outside the cache is not followed: ``append`` does
    not write its rows, ``attend`` takes its keys and values as zeros and
    reports it.

    ``max_q`` also decides how the kernels split the work: next to a plan for
    chunks, one with ``max_q=1`` serves single tokens up to a quarter faster,
    over the same cache.

    The plan owns the kernels' workspace: calls of one plan have to follow
    one another, on a stream or ordered by events; concurrent streams need a
    plan each.  Any stream may make the first call.  Making a plan waits for
    its workspace (not for queued work), calls never wait.
    After a reported timeout of a device-side wait, make a new plan.
    """

    def __init__(self, *, heads_q: int, heads_kv: int, head_dim: int, page_size: int,
                 max_seqs: int, max_q: int, dtype: torch.dtype, window: int | None = None,
                 sinks: int = 0, scale: float | None = None, device=None) -> None:
        device = torch.device("cuda" if device is None else device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self._plan = _native().Plan(heads_q, heads_kv, head_dim, page_size, max_seqs, max_q,
                                    dtype, window, sinks, scale, device)

    def append(self, k, v, k_pages, v_pages, page_table, q_start, kv_len) -> None:
        """Write the new tokens' rows k, v (tokens, heads_kv, head_dim) to the
        last slots of their sequences: token i to kv_len - q_len + i.  The
        cache holds values: nothing is passed back through it."""
        self._plan.append(k, v, k_pages, v_pages, page_table, q_start, kv_len)

    def attend(self, q, k_pages, v_pages, page_table, q_start, kv_len, out=None,
               lse=None) -> torch.Tensor:
        """Attention of the new tokens q (tokens, heads_q, head_dim) over
        their sequences' pages; the tokens' own K/V are in the cache already.
        ``out`` may name the tensor to write, ``lse`` (fp32, tokens x heads_q)
        one for the log-sum-exp.  Not differentiable: a backward pass that
        reaches the result raises."""
        result = self._plan.attend(q, k_pages, v_pages, page_table, q_start, kv_len, out, lse)
        if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad
                                        or v_pages.requires_grad):
            return _NoGradient.apply("PagedAttention.attend", [result], q, k_pages, v_pages)[0]
        return result


# ------------------------------------------------------- runner.build_callable
# Candidates of these operators are fixed by their problem: a config holds
# dtype, window (0: none) and sinks, and the library picks the variant.  The
# shapes are (batch, q_len, kv_len, heads_q, heads_kv, head_dim) and, paged,
# (seqs, max_q, page_size, heads_q, heads_kv, head_dim).
OPERATOR_INPUTS = {
    "attention_window": ("q", "k", "v"),
    "attention_window_grad": ("dout", "q", "k", "v", "out", "lse"),
    "attention_paged": ("q", "k_pages", "v_pages", "page_table", "q_start", "kv_len"),
    "cache_append": ("k", "v", "k_pages", "v_pages", "page_table", "q_start", "kv_len"),
}
_KERNELS = {"attention_window_grad": "attn_grad_kernel", "cache_append": "cache_append_kernel"}


def kernel_name(task: str, shape, config: dict, tokens: int = 0) -> str:
    """The kernel instance that a call launches, as the library chooses it;
    ``tokens``: the rows of q of a paged call."""
    if task in _KERNELS:
        return _KERNELS[task]
    dtype = _lib.DTYPE_IDS[str(config.get("dtype", "bfloat16"))]
    mask = (int(config.get("window", 0)), int(config.get("sinks", 0)), 0.0, 0)
    if task == "attention_window":
        b, q_len, kv_len, hq, hk, dim = shape
        query, args = "gpo_window_kernel", _lib.GpoWindowArgs(dtype, dim, hq, hk, b, q_len, kv_len,
                                                              *mask)
    else:
        seqs, max_q, page_size, hq, hk, dim = shape
        query, args = "gpo_paged_kernel", _lib.GpoPagedArgs(dtype, dim, hq, hk, seqs, tokens, max_q,
                                                            0, page_size, 0, 0, *mask)
    name = ctypes.create_string_buffer(256)
    rc = getattr(_lib.load(), query)(args, name, 256)
    if rc != _lib.OK:
        raise KernelBuildError(f"{task}: {name.value.decode()}")
    return name.value.decode()


def operator_call(task: str, shape, config: dict, inputs):
    """(fn, description, launch record) of one operator: ``fn`` launches on
    torch's current stream and returns outputs that are allocated here."""
    names = OPERATOR_INPUTS[task]
    if len(inputs) != len(names):
        raise KernelBuildError(f"{task} takes {len(names)} inputs {names}, got {len(inputs)}")
    t = dict(zip(names, inputs))
    want = str(config.get("dtype", "bfloat16"))
    dtype = {"float16": torch.float16, "bfloat16": torch.bfloat16}.get(want)
    if dtype is None:
        raise KernelBuildError(f"{task}: dtype must be float16 or bfloat16, got {want!r}")
    if len(shape) != 6:
        raise KernelBuildError(f"{task}: shape needs 6 values, got {tuple(shape)}")
    for name in names:
        if not isinstance(t[name], torch.Tensor) or not t[name].is_cuda:
            raise KernelBuildError("inputs must be CUDA tensors")
    first = t[names[0]]
    if first.dtype is not dtype:
        raise KernelBuildError(f"input dtype {first.dtype} does not match config dtype {dtype}")
    mask = {"window": int(config.get("window", 0)) or None, "sinks": int(config.get("sinks", 0))}
    if task.startswith("attention_window"):
        b, q_len, kv_len, hq, hk, dim = shape
        for name, s in (("q", (b, q_len, hq, dim)), ("k", (b, kv_len, hk, dim))):
            if tuple(t[name].shape) != s:
                raise KernelBuildError(f"{name} has shape {tuple(t[name].shape)}, expected {s}")
        if task == "attention_window":
            out = t["q"].new_empty(t["q"].shape)
            lse = out.new_empty(out.shape[:3], dtype=torch.float32)

            def fn():
                return window_attention_forward(*inputs, out=out, lse=lse, **mask)[0]
        else:
            grads = tuple(t[n].new_empty(t[n].shape) for n in ("q", "k", "v"))

            def fn():
                return window_attention_backward(*inputs, grads=grads, **mask)
    else:
        seqs, max_q, page_size, hq, hk, dim = shape
        plan = PagedAttention(heads_q=hq, heads_kv=hk, head_dim=dim, page_size=page_size,
                              max_seqs=seqs, max_q=max_q, dtype=dtype, device=first.device, **mask)
        if task == "attention_paged":
            out = first.new_empty(first.shape)

            def fn():
                return plan.attend(*inputs, out=out)
        else:
            def fn():
                plan.append(*inputs)
                return t["k_pages"], t["v_pages"]
    kernel = kernel_name(task, shape, config, first.shape[0])
    return fn, f"b200 {kernel}", {"kernel": kernel, **config}
