"""Measured cases of the attention operators: window attention with sinks
(forward, and forward + backward as in a training step), attention of a
chunk of new tokens over a paged K/V cache (single tokens included), and the
append of a chunk's K/V to the pages.

``run`` computes a case in its plain form (elementary torch operations in 32
bits, rounded once at the end) or, with ``own`` true, through this package's
operators.  Both read the same state.

The mask of every case: query token i of a sequence with q new tokens and n
keys stands at position p = n - q + i and sees key j iff j <= p and
(p - j < window or j < sinks); window 0 means no window.  A query that sees
nothing gives 0 (and a log-sum-exp of -inf).
"""

import math
import random

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


# ------------------------------------------------------------------- cases
def _window(name, batch, q_len, kv_len, heads_q, heads_kv, dim, window, sinks, dtype,
            train, fused):
    return {"name": name, "op": "train" if train else "window", "batch": batch, "q_len": q_len,
            "kv_len": kv_len, "heads_q": heads_q, "heads_kv": heads_kv, "dim": dim,
            "window": window, "sinks": sinks, "dtype": dtype, "fused": fused}


def _paged(name, op, seqs, q_max, kv_max, spread, page, heads_q, heads_kv, dim, window, sinks,
           dtype, lengths):
    return {"name": name, "op": op, "seqs": seqs, "q_max": q_max, "kv_max": kv_max,
            "spread": spread, "page": page, "heads_q": heads_q, "heads_kv": heads_kv,
            "dim": dim, "window": window, "sinks": sinks, "dtype": dtype, "lengths": lengths}


def listed():
    return [
        # a short prompt of a small model: the call's latency counts
        _window("window_short", 2, 257, 257, 8, 2, 64, 128, 4, "bfloat16", False, True),
        # prompt of a long-context model: window of 1024, four sinks, grouped heads
        _window("window_long", 1, 8192, 8192, 32, 8, 128, 1024, 4, "bfloat16", False, True),
        # fine-tuning step on short ragged samples, three query heads per kv head
        _window("train_ragged", 3, 333, 333, 6, 2, 64, 100, 2, "float16", True, False),
        # pre-training step of the long-context model
        _window("train_long", 1, 8192, 8192, 32, 8, 128, 1024, 4, "bfloat16", True, True),
        # pre-training step without a window (plain causal), one kv head per query head
        _window("train_causal", 2, 4096, 4096, 16, 16, 128, 0, 0, "bfloat16", True, False),
        # one user's next token: the smallest serving call
        _paged("decode_one", "paged", 1, 1, 777, 0.0, 16, 32, 8, 128, 0, 0, "bfloat16", 1),
        # next tokens of a full batch with sequences of all ages
        _paged("decode_batch", "paged", 64, 1, 8192, 0.9, 64, 32, 8, 128, 0, 0, "bfloat16", 2),
        # next tokens over two very long contexts
        _paged("decode_long", "paged", 2, 1, 131071, 0.1, 128, 32, 4, 128, 0, 0, "float16", 3),
        # chunked prefill: 512 new tokens of four sequences over their caches
        _paged("chunk_prefill", "paged", 4, 512, 8192, 0.3, 16, 32, 8, 128, 0, 0, "bfloat16", 4),
        # mixed batch (single tokens and chunks) of a window model with sinks
        _paged("chunk_window", "paged", 12, 300, 6000, 0.8, 32, 14, 2, 64, 1024, 4, "float16", 5),
        # the decode batch's new K/V into the cache
        _paged("append_tokens", "append", 64, 1, 2048, 0.9, 64, 32, 8, 128, 0, 0, "bfloat16", 6),
        # a prompt chunk's K/V of eight sequences into the cache
        _paged("append_chunk", "append", 8, 1024, 4096, 0.5, 16, 32, 8, 128, 0, 0, "bfloat16", 7),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("window", "window", "train", "train", "paged", "paged", "paged", "append"))
    dtype = rng.choice(("bfloat16", "float16"))
    dim = rng.choice((64, 128))
    heads_kv = rng.choice((1, 2, 4, 8))
    heads_q = heads_kv * rng.choice((1, 2, 3, 4, 4, 5, 6, 7, 8))
    sinks = rng.choice((0, 1, 4, 4, 16, 130))
    if op in ("window", "train"):
        batch = rng.choice((1, 1, 2, 3, 4))
        # the plain form holds every score in 32 bits, the largest listed case 2^31 of them
        most = min(8192, int(math.sqrt(2**31 / (batch * heads_q))))
        q_len = _log(rng, 1, most)
        kv_len = q_len
        if rng.random() < 0.3:  # a prefix in front of the queries, or fewer keys than queries
            kv_len = max(1, min(most, int(q_len * rng.choice((0.5, 0.9, 1.3, 2.0)))))
        window = rng.choice((0, 1)) * _log(rng, 1, 4096)
        # and no more visible pairs than the largest listed case has
        cap = max(1, 2**28 // (batch * heads_q * q_len))
        if cap < kv_len // 2 + 1:
            window = min(window or cap, cap)
            sinks = min(sinks, 4)
        return _window("", batch, q_len, kv_len, heads_q, heads_kv, dim, window, sinks, dtype,
                       op == "train", rng.random() < 0.5 and kv_len == q_len)
    seqs = _log(rng, 1, 64)
    page = rng.choice((8, 16, 16, 32, 48, 64, 128, 256))
    kv_most = max(64, min(131072, 2**29 // (seqs * heads_kv * dim)))
    kv_max = _log(rng, 1, kv_most)
    if op == "append":
        kv_max = min(kv_max, 4096)
        q_max = min(kv_max, rng.choice((1, _log(rng, 1, 1024))))
    else:
        pairs = 2**29 // (seqs * heads_q * kv_max)
        q_max = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, min(kv_max, pairs, 2048)))
    window = rng.choice((0, 0, 1)) * _log(rng, 1, 4096)
    return _paged("", op, seqs, q_max, kv_max, rng.choice((0.0, 0.5, 1.0)), page, heads_q,
                  heads_kv, dim, window, sinks, dtype, rng.randrange(1 << 30))


def _lengths(case):
    """(new tokens, keys) of each sequence: the first has the case's largest;
    the others lose up to the case's spread of it, and a batch whose spread
    is nearly whole holds single tokens and idle slots too."""
    r = random.Random(case["lengths"])
    q, n = [], []
    for b in range(case["seqs"]):
        f = 1.0 if b == 0 else 1.0 - case["spread"] * r.random()
        keys = max(1, int(case["kv_max"] * f))
        new = max(1, min(keys, int(case["q_max"] * (1.0 if b == 0 else 1.0 - case["spread"] * r.random()))))
        if b and case["spread"] >= 0.75:
            k = r.random()
            if k < 0.3:
                new = 1
            elif k < 0.34:
                new = keys = 0
        q.append(new)
        n.append(keys)
    return q, n


def _seen(q, n, window, sinks):
    """(visible pairs, keys seen by any query) of one sequence and one head."""
    pairs, low, first_p = 0, None, n - q
    window = window or n + q + 1
    for p in range(max(0, first_p), n):
        lo = max(0, p - window + 1)
        if low is None:
            low = lo
        pairs += p - lo + 1 + min(lo, sinks)
    if low is None:
        return 0, 0
    return pairs, n - low + min(low, sinks)


def work(case):
    hq, hk, d, es = case["heads_q"], case["heads_kv"], case["dim"], 2
    if case["op"] in ("window", "train"):
        b, q, n = case["batch"], case["q_len"], case["kv_len"]
        pairs, _ = _seen(q, n, case["window"], case["sinks"])
        qb, kb = b * q * hq * d * es, b * n * hk * d * es
        lse = b * q * hq * 4
        if case["op"] == "window":
            return {"bytes": 2 * qb + 2 * kb + lse, "flops": 4 * d * b * hq * pairs}
        # q, k, v and the output's gradient in; output, log-sum-exp and three gradients out
        return {"bytes": 4 * qb + 4 * kb + lse, "flops": 14 * d * b * hq * pairs}
    qs, ns = _lengths(case)
    if case["op"] == "append":
        return {"bytes": 4 * sum(qs) * hk * d * es + 4 * sum(q // case["page"] + 1 for q in qs),
                "flops": 0}
    pairs = keys = 0
    for q, n in zip(qs, ns):
        p, k = _seen(q, n, case["window"], case["sinks"])
        pairs, keys = pairs + p, keys + k
    return {"bytes": 2 * sum(qs) * hq * d * es + 2 * keys * hk * d * es, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    hq, hk, d = case["heads_q"], case["heads_kv"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    if case["op"] in ("window", "train"):
        b, q, n = case["batch"], case["q_len"], case["kv_len"]
        if case["fused"]:  # one projection's output, split by heads: strided views
            qkv = normal(b, q, hq + 2 * hk, d)
            s = {"q": qkv[:, :, :hq], "k": qkv[:, :, hq:hq + hk], "v": qkv[:, :, hq + hk:]}
        else:
            s = {"q": normal(b, q, hq, d), "k": normal(b, n, hk, d), "v": normal(b, n, hk, d)}
        if case["op"] == "train":
            s["dout"] = normal(b, q, hq, d)
        return s
    qs, ns = _lengths(case)
    page, seqs = case["page"], case["seqs"]
    per_seq = [-(-n // page) for n in ns]
    width = max(1, -(-case["kv_max"] // page))
    # pages in no order, a few of them free; entries past a sequence's pages are -1
    pages = sum(per_seq) + 7
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(per_seq):
        table[i, :k] = order[at:at + k]
        at += k
    start = [0]
    for q in qs:
        start.append(start[-1] + q)
    s = {"table": table.cuda(),
         "start": torch.tensor(start, dtype=torch.int32).cuda(),
         "kv_len": torch.tensor(ns, dtype=torch.int32).cuda(),
         "k_pages": normal(pages, page, hk, d), "v_pages": normal(pages, page, hk, d)}
    if case["op"] == "append":
        s["k"], s["v"] = normal(start[-1], hk, d), normal(start[-1], hk, d)
        return s
    # slots that no token has been written to hold whatever was there
    for i, (n, k) in enumerate(zip(ns, per_seq)):
        if n % page:
            last = int(table[i, k - 1])
            s["k_pages"][last, n % page:] = math.nan
            s["v_pages"][last, n % page:] = math.nan
    s["q"] = normal(start[-1], hq, d)
    return s


def prepare(case, seed):
    state = {"case": case, "tokens": 0, **_inputs(case, seed)}
    if case["op"] in ("paged", "append"):
        state["tokens"] = sum(_lengths(case)[0])
        if own:  # the plan (with its workspace) that a serving program keeps
            from gpu_optimizer_b200.attention_ops import PagedAttention

            state["plan"] = PagedAttention(
                heads_q=case["heads_q"], heads_kv=case["heads_kv"], head_dim=case["dim"],
                page_size=case["page"], max_seqs=case["seqs"], max_q=case["q_max"],
                dtype=_DTYPES[case["dtype"]], window=case["window"] or None,
                sinks=case["sinks"])
    return state


# ------------------------------------------------------------- plain forms
def _visible(pos, keys, kv_len, window, sinks):
    see = (keys <= pos) & (keys < kv_len)
    if window:
        see &= (pos - keys < window) | (keys < sinks)
    return see


def _softmax(s, see):
    """exp(s - max) over the visible keys, its sum and the log-sum-exp."""
    s = s.masked_fill_(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    m0 = m.masked_fill(m == -math.inf, 0.0)
    p = s.sub_(m0).exp_()
    total = p.sum(-1, keepdim=True)
    return p, total, (m0 + total.log()).squeeze(-1)


def _plain_window(st):
    case, dt = st["case"], st["q"].dtype
    b, q, n = case["batch"], case["q_len"], case["kv_len"]
    hk, d = case["heads_kv"], case["dim"]
    g = case["heads_q"] // hk
    scale = 1.0 / math.sqrt(d)
    dev = st["q"].device

    def heads(x):  # (b, t, h, d) -> (b, hk, h/hk, t, d)
        return x.float().reshape(b, x.shape[1], hk, -1, d).permute(0, 2, 3, 1, 4)

    def tokens(x):  # back, rounded
        return x.permute(0, 3, 1, 2, 4).reshape(b, x.shape[3], -1, d).to(dt)

    qf, kf, vf = heads(st["q"]), heads(st["k"]), heads(st["v"])
    pos = torch.arange(q, device=dev)[:, None] + (n - q)
    see = _visible(pos, torch.arange(n, device=dev), n, case["window"], case["sinks"])
    p, total, lse = _softmax((qf * scale) @ kf.transpose(-1, -2), see)
    p = p.div_(total.masked_fill(total == 0, 1.0))
    out = p @ vf
    res = {"out": tokens(out), "lse": lse.reshape(b, hk * g, q).transpose(1, 2).contiguous()}
    if case["op"] == "train":
        do = heads(st["dout"])
        res["dv"] = tokens((p.transpose(-1, -2) @ do).sum(2, keepdim=True))
        ds = (do @ vf.transpose(-1, -2)).sub_((do * out).sum(-1, keepdim=True)).mul_(p)
        res["dq"] = tokens(ds @ kf * scale)
        res["dk"] = tokens((ds.transpose(-1, -2) @ qf).sum(2, keepdim=True) * scale)
    return res


def _token_rows(st):
    """Sequence and place in it of every new token."""
    t = torch.arange(st["tokens"], device="cuda")
    seq = torch.searchsorted(st["start"], t.to(torch.int32), right=True) - 1
    return seq, t - st["start"][seq]


def _plain_paged(st):
    case, dt = st["case"], st["q"].dtype
    hk, d, page = case["heads_kv"], case["dim"], case["page"]
    seqs, qm = case["seqs"], case["q_max"]
    scale = 1.0 / math.sqrt(d)
    start, kv_len, table = st["start"].long(), st["kv_len"].long(), st["table"].long()
    width = table.shape[1] * page
    rows = (start[:-1, None] + torch.arange(qm, device="cuda")).clamp(max=max(0, st["tokens"] - 1))
    qf = st["q"][rows].float().reshape(seqs, qm, hk, -1, d).permute(0, 2, 3, 1, 4)
    g = qf.shape[2]
    keys = torch.arange(width, device="cuda")
    there = (keys < kv_len[:, None])[:, None, :, None]

    def cache(pages):  # (seqs, hk, width, d), nothing where no token was written
        x = pages[table.clamp(min=0)].reshape(seqs, width, hk, d).transpose(1, 2).float()
        return x.masked_fill_(~there, 0.0)

    kf, vf = cache(st["k_pages"]), cache(st["v_pages"])
    pos = (kv_len - (start[1:] - start[:-1]))[:, None] + torch.arange(qm, device="cuda")
    see = _visible(pos[:, :, None], keys, kv_len[:, None, None], case["window"], case["sinks"])
    s = (qf * scale).reshape(seqs, hk, g * qm, d) @ kf.transpose(-1, -2)
    p, total, _ = _softmax(s.reshape(seqs, hk, g, qm, width), see[:, None, None])
    out = p.reshape(seqs, hk, g * qm, width) @ vf
    out = out.reshape(seqs, hk, g, qm, d) / total.masked_fill(total == 0, 1.0)
    seq, at = _token_rows(st)
    return {"out": out.permute(0, 3, 1, 2, 4)[seq, at].reshape(-1, hk * g, d).to(dt)}


def _plain_append(st):
    seq, at = _token_rows(st)
    q_len = st["start"][1:] - st["start"][:-1]
    slot = (st["kv_len"] - q_len)[seq] + at
    page = st["table"].long()[seq, slot // st["case"]["page"]].long()
    st["k_pages"][page, slot % st["case"]["page"]] = st["k"]
    st["v_pages"][page, slot % st["case"]["page"]] = st["v"]
    return {"k_pages": st["k_pages"], "v_pages": st["v_pages"]}


# --------------------------------------------------------------------- run
def _own_window(st):
    from gpu_optimizer_b200 import attention_ops as ops

    case = st["case"]
    mask = {"window": case["window"] or None, "sinks": case["sinks"]}
    out, lse = ops.window_attention_forward(st["q"], st["k"], st["v"], **mask)
    if case["op"] == "window":
        return {"out": out, "lse": lse}
    dq, dk, dv = ops.window_attention_backward(st["dout"], st["q"], st["k"], st["v"], out, lse,
                                               **mask)
    return {"out": out, "lse": lse, "dv": dv, "dq": dq, "dk": dk}


def run(state):
    op = state["case"]["op"]
    if op in ("window", "train"):
        return _own_window(state) if own else _plain_window(state)
    if not own:
        return _plain_append(state) if op == "append" else _plain_paged(state)
    where = (state["k_pages"], state["v_pages"], state["table"], state["start"], state["kv_len"])
    if op == "append":
        state["plan"].append(state["k"], state["v"], *where)
        return {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}
    return {"out": state["plan"].attend(state["q"], *where)}


# ------------------------------------------------------------------- exact
def _exact_head(q, k, v, p0, window, sinks, dout=None):
    """One head in 64 bits: softmax over each row's visible keys, and the
    products' gradients by the chain rule through the normalised weights."""
    d = q.shape[-1]
    n = k.shape[0]
    at = torch.arange(q.shape[0], device=q.device)[:, None] + p0
    j = torch.arange(n, device=q.device)[None, :]
    dist = at - j
    hidden = dist < 0
    if window:
        hidden |= (dist >= window) & (j >= sinks)
    a = torch.einsum("id,jd->ij", q, k).mul_(d ** -0.5)
    a[hidden] = -math.inf
    lse = torch.logsumexp(a, 1)
    w = torch.exp(a - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None])
    o = torch.einsum("ij,jd->id", w, v)
    if dout is None:
        return o, lse
    dw = torch.einsum("id,jd->ij", dout, v)
    da = w * (dw - (w * dw).sum(1, keepdim=True)) * d ** -0.5
    return (o, lse, torch.einsum("ij,jd->id", da, k), torch.einsum("ij,id->jd", da, q),
            torch.einsum("ij,id->jd", w, dout))


def exact(case, seed):
    s = _inputs(case, seed)
    hk, d = case["heads_kv"], case["dim"]
    g = case["heads_q"] // hk
    f64 = {"dtype": torch.float64, "device": "cuda"}
    if case["op"] in ("window", "train"):
        q, k, v = (s[x].double() for x in "qkv")
        do = s["dout"].double() if case["op"] == "train" else None
        out, lse = torch.zeros(q.shape, **f64), torch.zeros(q.shape[:3], **f64)
        dq, dk, dv = torch.zeros(q.shape, **f64), torch.zeros(k.shape, **f64), torch.zeros(k.shape, **f64)
        for b in range(case["batch"]):
            for h in range(case["heads_q"]):
                r = _exact_head(q[b, :, h], k[b, :, h // g], v[b, :, h // g],
                                case["kv_len"] - case["q_len"], case["window"], case["sinks"],
                                None if do is None else do[b, :, h])
                out[b, :, h], lse[b, :, h] = r[0], r[1]
                if do is not None:
                    dq[b, :, h] = r[2]
                    dk[b, :, h // g] += r[3]
                    dv[b, :, h // g] += r[4]
        if do is None:
            return {"out": out, "lse": lse}
        return {"out": out, "lse": lse, "dv": dv, "dq": dq, "dk": dk}
    qs, ns = _lengths(case)
    start, table, page = s["start"].tolist(), s["table"].tolist(), case["page"]
    if case["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        for b, (q, n) in enumerate(zip(qs, ns)):
            slots = torch.arange(n - q, n)
            at = torch.tensor(table[b])[slots // page].long(), slots % page
            kp[at[0], at[1]] = s["k"][start[b]:start[b + 1]].double()
            vp[at[0], at[1]] = s["v"][start[b]:start[b + 1]].double()
        return {"k_pages": kp, "v_pages": vp}
    out = torch.zeros(s["q"].shape, **f64)
    for b, (q, n) in enumerate(zip(qs, ns)):
        if not q:
            continue
        ids = torch.tensor(table[b][: -(-n // page)], device="cuda").long()
        for h in range(hk):
            k = s["k_pages"][ids, :, h].reshape(-1, d)[:n].double()
            v = s["v_pages"][ids, :, h].reshape(-1, d)[:n].double()
            for e in range(h * g, (h + 1) * g):
                out[start[b]:start[b + 1], e] = _exact_head(
                    s["q"][start[b]:start[b + 1], e].double(), k, v, n - q, case["window"],
                    case["sinks"])[0]
    return {"out": out}
