"""Plain 64-bit forms of the window / paged attention operators and the error
bounds their 16-bit kernels must keep (imported by the tests of the operators).

Bounds.  u is the unit roundoff of the element type (2^-8 bfloat16, 2^-11
float16: half a unit in the last place of 1).  A kernel
rounds P (and dS) to the element type as an MMA operand and rounds each output
once; everything else is fp32.  R = 3e-4 covers the fp32 part relative to the
sum of the terms' magnitudes: scores of 128 fp32 products (2^-24 * 128 each way
on |s| <= 30 is 2.3e-4 in the exponent at the very worst), exponentials
(7.5e-5), sums.  With A = P |V|:
    |out - ref| <= (u + R) A + u |ref|
    |dv  - ref| <= (u + R) P^T |dO| + u |ref|
dS is P * (dP - delta), delta from the rounded output: with a = sum |dO| |O|
and b = |dO| |V|^T,
    |dS - ref|  <= (u + R) |dS| + P * (u a + R (a + b))  =: E
    |dq - ref|  <= scale E |K| + R scale |dS| |K| + u |ref|, dk likewise.
float16 has a smallest normal of 2^-14: what is below it is rounded to
multiples of 2^-24, which adds 2^-25 per P and dS, and to each output.
"""

import math

import torch

R = 3e-4


def unit(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11


def tiny(dtype):
    return 0.0 if dtype == torch.bfloat16 else 2.0 ** -25


def visible(q_len, kv_len, window, sinks, device="cpu"):
    p = torch.arange(q_len, device=device)[:, None] + (kv_len - q_len)
    j = torch.arange(kv_len, device=device)[None, :]
    see = j <= p
    if window is not None:
        see &= (p - j < window) | (j < sinks)
    return see


def head(q, k, v, see, scale, dout=None):
    """One head in 64 bits: out, lse and their bounds' magnitudes (and the
    gradients with theirs)."""
    q, k, v = q.double(), k.double(), v.double()
    s = (q @ k.T * scale).masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full((q.shape[0],), -math.inf,
                                                              dtype=torch.float64, device=q.device)
    p = torch.where(see, torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[:, None]), 0.0)
    out = p @ v
    r = {"out": out, "lse": lse, "A": p @ v.abs(), "V": see.double() @ v.abs()}
    if dout is None:
        return r
    do = dout.double()
    dp = do @ v.T
    ds = torch.where(see, p * (dp - (do * out).sum(-1, keepdim=True)), 0.0)
    a = (do.abs() * out.abs()).sum(-1, keepdim=True)
    b = do.abs() @ v.abs().T
    return {**r, "p": p, "ds": ds, "a": a, "b": b, "do": do, "q": q, "k": k,
            "dq": ds @ k * scale, "dk": ds.T @ q * scale, "dv": p.T @ do}


def bounds(r, dtype, scale=1.0):
    """Element bounds of a head's outputs (dk, dv: of its share of the sums,
    the output rounding excluded)."""
    u, t = unit(dtype), tiny(dtype)
    e = {"out": (u + R) * r["A"] + u * r["out"].abs() + t * r["V"]}
    if "ds" in r:
        see = (r["p"] > 0).double()
        es = (u + R) * r["ds"].abs() + r["p"] * (u * r["a"] + R * (r["a"] + r["b"])) + t * see
        e["dq"] = scale * (es @ r["k"].abs() + R * r["ds"].abs() @ r["k"].abs()) + u * r["dq"].abs()
        e["dk"] = scale * (es.T @ r["q"].abs() + R * r["ds"].abs().T @ r["q"].abs())
        e["dv"] = ((u + R) * r["p"] + t * see).T @ r["do"].abs()
    return e


def within(name, got, want, bound):
    off = (got.double() - want).abs() - bound - tiny(got.dtype)
    worst = off.max().item() if off.numel() else -1.0
    assert not torch.isnan(got).any(), f"{name}: NaN"
    assert worst <= 1e-12, f"{name}: {worst:.3e} over its bound"
