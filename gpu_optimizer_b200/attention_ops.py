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

Everything runs on torch's current stream and never synchronises.  A refused
argument raises ``KernelBuildError`` with the library's reason, before
anything is launched; a launch that fails raises ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from .runner import KernelBuildError

_DTYPE_IDS = {torch.float16: _lib.DTYPE_IDS["float16"], torch.bfloat16: _lib.DTYPE_IDS["bfloat16"]}

# A call's records are packed in one go: field by field costs more than the
# launch.  (ptr, stride_batch, stride_token, stride_head) per tensor.
_HEADS = "Q3q"
_WINDOW = struct.Struct("<4i5qfi" + 4 * _HEADS + "Q" + 4 * _HEADS + "QQ")
_NO_HEADS = (0, 0, 0, 0)
_PAGED_SIZES = struct.Struct("<qq")             # num_seqs, tokens
_PAGED_PAGES = struct.Struct("<q")              # num_pages
_PAGED_TABLE = struct.Struct("<qq")             # table_width, table_stride
_PAGED_HEADS = struct.Struct("<" + 2 * _HEADS)  # q, out / k_pages, v_pages / k_new, v_new
_PAGED_PTRS = struct.Struct("<4Q")              # page_table, q_start, kv_len, lse
assert _WINDOW.size == ctypes.sizeof(_lib.GpoWindowArgs)


def _library():
    try:
        return _lib.load()
    except _lib.LibraryMissing as e:
        raise KernelBuildError(str(e), log=str(e)) from e


def _refused(name: str, rc: int, log) -> None:
    why = log.value.decode(errors="replace")
    text = f"{name}: {_lib.status_name(rc)}: {why}"
    if rc in (_lib.BAD_ARGS, _lib.BAD_CONFIG):
        raise KernelBuildError(text, log=why)
    raise RuntimeError(text)


def _launch(name: str, args, device: torch.device) -> None:
    """Call a launch entry point on ``device``'s current torch stream."""
    fn = getattr(_library(), name)
    index = device.index
    log = ctypes.create_string_buffer(256)
    if torch._C._cuda_getDevice() == index:
        rc = fn(args, torch._C._cuda_getCurrentRawStream(index), log, 256)
    else:
        with torch.cuda.device(index):
            rc = fn(args, torch._C._cuda_getCurrentRawStream(index), log, 256)
    if rc != _lib.OK:
        _refused(name, rc, log)


def _workspace_bytes(name: str, args) -> int:
    log = ctypes.create_string_buffer(256)
    size = ctypes.c_uint64(0)
    rc = getattr(_library(), name)(args, size, log, 256)
    if rc != _lib.OK:
        _refused(name, rc, log)
    return size.value


def _check(name: str, t: torch.Tensor, dims: int, dtype: torch.dtype,
           device: torch.device) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise KernelBuildError(f"{name} must be a CUDA tensor")
    if t.dim() != dims:
        raise KernelBuildError(f"{name} must have {dims} dimensions, got {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise KernelBuildError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise KernelBuildError(f"{name} is on {t.device}, expected {device}")


def _in_place(t: torch.Tensor) -> bool:
    """Whether the kernels can address ``t``'s rows where they are."""
    *steps, last = t.stride()
    if last == 1 and t.data_ptr() & 15 == 0:
        if all(s & 7 == 0 for s in steps):
            return True
        return all(s & 7 == 0 for n, s in zip(t.shape, steps) if n > 1)
    return t.numel() == 0


def _readable(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy where its rows cannot be read in place: rows that are
    not contiguous, or a start or stride off the 16-byte grid."""
    return t if _in_place(t) else t.clone(memory_format=torch.contiguous_format)


def _heads(t: torch.Tensor) -> tuple:
    """gpo_heads fields of a (batch, token, head, dim) tensor, or of packed
    (token, head, dim) rows."""
    s = t.stride()
    if len(s) == 4:
        return t.data_ptr(), s[0], s[1], s[2]
    return t.data_ptr(), 0, s[0], s[1]


def _mask(window, sinks: int, scale) -> tuple:
    """window, sinks and scale fields."""
    if window is not None and window < 1:
        raise KernelBuildError(f"window must be at least 1 (or None), got {window}")
    if sinks < 0:
        raise KernelBuildError(f"sinks must not be negative, got {sinks}")
    if scale is not None and not scale > 0:
        raise KernelBuildError(f"scale must be positive, got {scale}")
    return (0 if window is None else min(int(window), 1 << 40), min(int(sinks), 1 << 40),
            0.0 if scale is None else float(scale))


def _window_sizes(q, k, v, window, sinks, scale) -> tuple:
    """Leading fields of a gpo_window_args, after checks of q, k and v."""
    if not isinstance(q, torch.Tensor) or q.dtype not in _DTYPE_IDS:
        raise KernelBuildError("q must be a float16 or bfloat16 CUDA tensor")
    dtype, device = q.dtype, q.device
    _check("q", q, 4, dtype, device)
    _check("k", k, 4, dtype, device)
    _check("v", v, 4, dtype, device)
    b, q_len, heads_q, dim = q.shape
    kb, kv_len, heads_kv, kdim = ks = k.shape
    if ks != v.shape or kb != b or kdim != dim:
        raise KernelBuildError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} "
                               "do not belong together")
    return (_DTYPE_IDS[dtype], dim, heads_q, heads_kv, b, q_len, kv_len,
            *_mask(window, sinks, scale), 0)


def _window_args(sizes, q, k, v, out, lse, grads=4 * _NO_HEADS, workspace=(0, 0)):
    a = _lib.GpoWindowArgs()
    _WINDOW.pack_into(a, 0, *sizes, *_heads(q), *_heads(k), *_heads(v), *_heads(out),
                      lse.data_ptr(), *grads, *workspace)
    return a


def _written(name: str, t: torch.Tensor, shape, dtype, device) -> None:
    _check(name, t, len(shape), dtype, device)
    if t.shape != shape or not (t.is_contiguous() if dtype is torch.float32 else _in_place(t)):
        raise KernelBuildError(f"{name} must have shape {tuple(shape)}, its rows contiguous and "
                               f"16-byte aligned")


def window_attention_forward(q, k, v, *, window: int | None = None, sinks: int = 0,
                             scale: float | None = None, out=None, lse=None):
    """(out, lse): attention of q over k, v, and each row's log-sum-exp of
    scaled scores, fp32 (batch, q_len, heads_q).  ``out`` and ``lse`` may name
    the tensors to write."""
    sizes = _window_sizes(q, k, v, window, sinks, scale)
    q, k, v = _readable(q), _readable(k), _readable(v)
    if out is None:
        out = q.new_empty(q.shape)
    else:
        _written("out", out, q.shape, q.dtype, q.device)
    if lse is None:
        lse = q.new_empty(q.shape[:3], dtype=torch.float32)
    else:
        _written("lse", lse, q.shape[:3], torch.float32, q.device)
    _launch("gpo_window_attention", _window_args(sizes, q, k, v, out, lse), q.device)
    return out, lse


def window_attention_backward(dout, q, k, v, out, lse, *, window: int | None = None,
                              sinks: int = 0, scale: float | None = None, grads=None):
    """(dq, dk, dv) from the output's gradient and what the forward returned.
    ``grads`` may name the three tensors to write.

    Sums run in a fixed order: the same inputs give the same bits.
    """
    sizes = _window_sizes(q, k, v, window, sinks, scale)
    shape, device = q.shape, q.device
    for name, t in (("out", out), ("dout", dout)):
        _check(name, t, 4, q.dtype, device)
        if t.shape != shape:
            raise KernelBuildError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    _check("lse", lse, 3, torch.float32, device)
    if lse.shape != shape[:3]:
        raise KernelBuildError(f"lse has shape {tuple(lse.shape)}, expected {tuple(shape[:3])}")
    q, k, v, out, dout = (_readable(q), _readable(k), _readable(v), _readable(out),
                          _readable(dout))
    lse = lse.contiguous()
    if grads is None:
        dq, dk, dv = q.new_empty(shape), q.new_empty(k.shape), q.new_empty(k.shape)
    else:
        dq, dk, dv = grads
        for name, t, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
            _written(name, t, like.shape, q.dtype, device)
    grads = (*_heads(dout), *_heads(dq), *_heads(dk), *_heads(dv))
    size = _workspace_bytes("gpo_window_workspace", _window_args(sizes, q, k, v, out, lse))
    work = torch.empty(max(1, size), dtype=torch.uint8, device=device)
    a = _window_args(sizes, q, k, v, out, lse, grads, (work.data_ptr(), size))
    _launch("gpo_window_attention_grad", a, device)
    return dq, dk, dv


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale):
        out, lse = window_attention_forward(q, k, v, window=window, sinks=sinks, scale=scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.mask = {"window": window, "sinks": sinks, "scale": scale}
        return out

    @staticmethod
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
    keys, new tokens included.  Both stay on the device and are not read by
    the host; a sequence whose lengths do not fit the buffers is skipped and
    reported by ``runner.check_device_status``.  Page table entries behind a
    sequence's last key, and those of pages no token sees any more, are not
    read as pages.

    The plan owns the kernels' workspace: calls of one plan have to follow
    one another on a stream; concurrent streams need a plan each.
    """

    def __init__(self, *, heads_q: int, heads_kv: int, head_dim: int, page_size: int,
                 max_seqs: int, max_q: int, dtype: torch.dtype, window: int | None = None,
                 sinks: int = 0, scale: float | None = None, device=None) -> None:
        if dtype not in _DTYPE_IDS:
            raise KernelBuildError(f"dtype must be float16 or bfloat16, got {dtype}")
        if max_seqs < 1 or max_q < 1:
            raise KernelBuildError("max_seqs and max_q must be at least 1")
        self.dtype, self.heads_q, self.heads_kv, self.head_dim = dtype, heads_q, heads_kv, head_dim
        self.page_size, self.max_seqs, self.max_q = page_size, max_seqs, max_q
        device = torch.device("cuda" if device is None else device)
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        win, sink, factor = _mask(window, sinks, scale)
        a = self._args = _lib.GpoPagedArgs(
            dtype=_DTYPE_IDS[dtype], head_dim=head_dim, heads_q=heads_q, heads_kv=heads_kv,
            page_size=page_size, max_q=max_q, window=win, sinks=sink, scale=factor,
            num_seqs=max_seqs, tokens=max_seqs * max_q)
        size = _workspace_bytes("gpo_paged_workspace", a)
        self._work = torch.zeros(max(1, size), dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes = self._work.data_ptr(), size
        self._page_shape = (page_size, heads_kv, head_dim)

    def _fill(self, rows, k_pages, v_pages, page_table, q_start, kv_len, lse=0):
        a, dtype, device = self._args, self.dtype, self.device
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            _check(name, t, 4, dtype, device)
            if t.shape[1:] != self._page_shape:
                raise KernelBuildError(f"{name} has shape {tuple(t.shape)}, expected (pages, "
                                       f"{', '.join(map(str, self._page_shape))})")
            if not _in_place(t):
                raise KernelBuildError(f"{name}: rows must be contiguous and 16-byte aligned")
        pages = k_pages.shape[0]
        if pages != v_pages.shape[0]:
            raise KernelBuildError("k_pages and v_pages have different numbers of pages")
        _check("page_table", page_table, 2, torch.int32, device)
        _check("q_start", q_start, 1, torch.int32, device)
        _check("kv_len", kv_len, 1, torch.int32, device)
        seqs, width = page_table.shape
        if seqs > self.max_seqs or q_start.shape[0] != seqs + 1 or kv_len.shape[0] != seqs:
            raise KernelBuildError(
                f"{seqs} sequences in page_table, {q_start.shape[0] - 1} in q_start, "
                f"{kv_len.shape[0]} in kv_len; at most {self.max_seqs}")
        row, step = page_table.stride()
        if (width > 1 and step != 1) or not q_start.is_contiguous() \
                or not kv_len.is_contiguous():
            raise KernelBuildError("page_table rows, q_start and kv_len must be contiguous")
        at = _lib.GpoPagedArgs
        _PAGED_SIZES.pack_into(a, at.num_seqs.offset, seqs, rows)
        _PAGED_PAGES.pack_into(a, at.num_pages.offset, pages)
        _PAGED_TABLE.pack_into(a, at.table_width.offset, width, row)
        _PAGED_HEADS.pack_into(a, at.k_pages.offset, *_heads(k_pages), *_heads(v_pages))
        _PAGED_PTRS.pack_into(a, at.page_table.offset, page_table.data_ptr(), q_start.data_ptr(),
                              kv_len.data_ptr(), lse)
        return a

    def append(self, k, v, k_pages, v_pages, page_table, q_start, kv_len) -> None:
        """Write the new tokens' rows k, v (tokens, heads_kv, head_dim) to the
        last slots of their sequences: token i to kv_len - q_len + i."""
        for name, t in (("k", k), ("v", v)):
            _check(name, t, 3, self.dtype, self.device)
            if t.shape[1:] != (self.heads_kv, self.head_dim) or t.shape[0] != k.shape[0]:
                raise KernelBuildError(f"{name} has shape {tuple(t.shape)}, expected (tokens, "
                                       f"{self.heads_kv}, {self.head_dim})")
        k, v = _readable(k), _readable(v)
        a = self._fill(k.shape[0], k_pages, v_pages, page_table, q_start, kv_len)
        _PAGED_HEADS.pack_into(a, _lib.GpoPagedArgs.k_new.offset, *_heads(k), *_heads(v))
        _launch("gpo_cache_append", a, self.device)

    def attend(self, q, k_pages, v_pages, page_table, q_start, kv_len, out=None,
               lse=None) -> torch.Tensor:
        """Attention of the new tokens q (tokens, heads_q, head_dim) over
        their sequences' pages; the tokens' own K/V are in the cache already.
        ``out`` may name the tensor to write, ``lse`` (fp32, tokens x heads_q)
        one for the log-sum-exp."""
        _check("q", q, 3, self.dtype, self.device)
        if q.shape[1:] != (self.heads_q, self.head_dim):
            raise KernelBuildError(f"q has shape {tuple(q.shape)}, expected (tokens, "
                                   f"{self.heads_q}, {self.head_dim})")
        q = _readable(q)
        if out is None:
            out = q.new_empty(q.shape)
        else:
            _written("out", out, q.shape, self.dtype, self.device)
        if lse is not None:
            _written("lse", lse, q.shape[:2], torch.float32, self.device)
        a = self._fill(q.shape[0], k_pages, v_pages, page_table, q_start, kv_len,
                       0 if lse is None else lse.data_ptr())
        _PAGED_HEADS.pack_into(a, _lib.GpoPagedArgs.q.offset, *_heads(q), *_heads(out))
        _launch("gpo_paged_attention", a, self.device)
        return out


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
_KERNELS = {"attention_window": "attn_fwd_kernel<dense>",
            "attention_window_grad": "attn_grad_kernel",
            "attention_paged": "attn_fwd_kernel<paged>",
            "cache_append": "cache_append_kernel"}


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
    return fn, f"b200 {_KERNELS[task]}", {"kernel": _KERNELS[task], **config}
