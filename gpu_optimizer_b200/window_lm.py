"""Example: a small language model with sliding-window attention, trained and
then served from a paged K/V cache.

``python -m gpu_optimizer_b200.window_lm [--steps N]`` trains a two-layer
model on sequences that repeat with a fixed period (the window is longer than
the period, the sinks hold the start token), then serves a batch of prompts:
prompt chunks first, single tokens after, every sequence at its own length.
Both halves use the same mask: ``window_attention`` in training,
``PagedAttention.append`` / ``attend`` in serving.  It prints the loss, how
often the served tokens continue the pattern, and how far the served logits
are from those of one dense pass over the same tokens.
"""

from __future__ import annotations

import argparse

import torch
import torch.nn.functional as F

from .attention_ops import PagedAttention, window_attention
from .runner import check_device_status


class WindowLM:
    """Token embedding, pre-norm attention + MLP layers, tied output."""

    def __init__(self, vocab=64, layers=2, heads_q=4, heads_kv=2, head_dim=64, window=24, sinks=2,
                 dtype=torch.bfloat16, seed=0) -> None:
        self.heads_q, self.heads_kv, self.head_dim = heads_q, heads_kv, head_dim
        self.mask = {"window": window, "sinks": sinks}
        self.dtype = dtype
        width = heads_q * head_dim
        g = torch.Generator().manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g) * cols ** -0.5).cuda().requires_grad_()

        self.embed = weight(vocab, width)
        # a layer's qkv, output, and the MLP's two projections; fp32 masters
        self.layers = [{"qkv": weight((heads_q + 2 * heads_kv) * head_dim, width),
                        "out": weight(width, width), "up": weight(2 * width, width),
                        "down": weight(width, 2 * width)} for _ in range(layers)]

    def parameters(self):
        return [self.embed, *(w for layer in self.layers for w in layer.values())]

    def _rotate(self, x, pos):
        """Rotary positions on (..., head, dim) with one position per row."""
        half = self.head_dim // 2
        freq = 100.0 ** (-torch.arange(half, device=x.device) / half)
        a = pos[..., None, None].float() * freq
        x1, x2 = x.float()[..., :half], x.float()[..., half:]
        c, s = a.cos(), a.sin()
        return torch.cat((x1 * c - x2 * s, x1 * s + x2 * c), -1).to(self.dtype)

    def _qkv(self, layer, x, pos):
        h = F.rms_norm(x, x.shape[-1:]).to(self.dtype)
        qkv = (h @ layer["qkv"].to(self.dtype).t()).unflatten(-1, (-1, self.head_dim))
        q, k, v = qkv.split((self.heads_q, self.heads_kv, self.heads_kv), -2)
        return self._rotate(q, pos), self._rotate(k, pos), v

    def _rest(self, layer, x, attended):
        x = x + attended.flatten(-2) @ layer["out"].to(self.dtype).t()
        h = F.rms_norm(x, x.shape[-1:]).to(self.dtype)
        return x + F.gelu(h @ layer["up"].to(self.dtype).t()) @ layer["down"].to(self.dtype).t()

    def _logits(self, x):
        return F.rms_norm(x, x.shape[-1:]).to(self.dtype).float() @ self.embed.t()

    def forward(self, tokens):
        """Logits of (batch, length) tokens in one dense pass."""
        pos = torch.arange(tokens.shape[1], device=tokens.device).expand(tokens.shape)
        x = self.embed[tokens].to(self.dtype)
        for layer in self.layers:
            q, k, v = self._qkv(layer, x, pos)
            x = self._rest(layer, x, window_attention(q, k, v, **self.mask))
        return self._logits(x)


class Server:
    """Sequences of a WindowLM over one paged cache per layer."""

    def __init__(self, model: WindowLM, max_seqs=8, max_len=256, max_chunk=32, page_size=16):
        self.m = model
        per_seq = -(-max_len // page_size)
        shape = (max_seqs * per_seq, page_size, model.heads_kv, model.head_dim)
        self.k = [torch.empty(shape, dtype=model.dtype, device="cuda") for _ in model.layers]
        self.v = [torch.empty(shape, dtype=model.dtype, device="cuda") for _ in model.layers]
        # any assignment of pages will do; here they are handed out at random
        self.table = torch.randperm(shape[0]).to(torch.int32).view(max_seqs, per_seq).cuda()
        self.length = torch.zeros(max_seqs, dtype=torch.int32, device="cuda")
        self.plan = PagedAttention(heads_q=model.heads_q, heads_kv=model.heads_kv,
                                   head_dim=model.head_dim, page_size=page_size,
                                   max_seqs=max_seqs, max_q=max_chunk, dtype=model.dtype,
                                   **model.mask)

    @torch.no_grad()
    def step(self, chunks):
        """Logits of each sequence's new tokens (a list of 1-D tensors, one
        per sequence, empty for an idle one), appended to the cache."""
        counts = torch.tensor([0] + [len(c) for c in chunks], device="cuda")
        start = counts.cumsum(0).to(torch.int32)
        tokens = torch.cat(chunks)
        pos = torch.cat([n + torch.arange(len(c), device="cuda")
                         for n, c in zip(self.length, chunks)])
        self.length += counts[1:].to(torch.int32)
        x = self.m.embed[tokens].to(self.m.dtype)
        for layer, k_pages, v_pages in zip(self.m.layers, self.k, self.v):
            q, k, v = self.m._qkv(layer, x, pos)
            where = (k_pages, v_pages, self.table, start, self.length)
            self.plan.append(k, v, *where)
            x = self.m._rest(layer, x, self.plan.attend(q, *where))
        return self.m._logits(x).split([len(c) for c in chunks])


def pattern(batch, length, period, vocab, generator):
    """Start token 0, then a random word of ``period`` tokens over and over."""
    word = torch.randint(1, vocab, (batch, period), generator=generator)
    body = word.repeat(1, -(-length // period))[:, :length - 1]
    return torch.cat((torch.zeros(batch, 1, dtype=torch.long), body), 1).cuda()


def main(steps=300, seed=0) -> dict:
    g = torch.Generator().manual_seed(seed)
    model = WindowLM(seed=seed)
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3, fused=True)
    loss = None
    for i in range(steps):
        tokens = pattern(32, 96, 9, 64, g)
        logits = model.forward(tokens)
        loss = F.cross_entropy(logits[:, 16:-1].flatten(0, 1), tokens[:, 17:].flatten())
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        if i % 50 == 0 or i == steps - 1:
            print(f"step {i}: loss {loss.item():.4f}", flush=True)
    # serve prompts of different lengths, in chunks, then token by token
    truth = pattern(8, 140, 9, 64, g)
    prompts = [40 + 7 * i for i in range(8)]
    server, seen = Server(model), [[] for _ in prompts]
    fed, nxt = [0] * 8, [None] * 8
    while min(fed) < 130:
        chunks = []
        for b, n in enumerate(prompts):
            if fed[b] >= 130:
                chunk = truth[b, :0]
            elif fed[b] < n:
                chunk = truth[b, fed[b]:min(n, fed[b] + 32)]
            else:
                chunk = nxt[b]
            seen[b].append(chunk)
            fed[b] += len(chunk)
            chunks.append(chunk)
        for b, out in enumerate(server.step(chunks)):
            if len(out):
                nxt[b] = out[-1:].argmax(-1)
                seen[b][-1] = (chunks[b], out)
    right = total = 0
    far = 0.0
    for b, n in enumerate(prompts):
        parts = [s for s in seen[b] if isinstance(s, tuple)]
        tokens = torch.cat([s[0] for s in parts])
        served = torch.cat([s[1] for s in parts])
        right += (tokens[n:130] == truth[b, n:130]).sum().item()
        total += 130 - n
        with torch.no_grad():
            dense = model.forward(tokens[None])[0]
        far = max(far, ((served - dense).norm() / dense.norm()).item())
    check_device_status()
    result = {"loss": loss.item(), "continued": right / total, "logits_rel": far}
    print(f"served {total} tokens: {result['continued']:.1%} continue the pattern; "
          f"logits {far:.2e} from the dense pass", flush=True)
    return result


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--steps", type=int, default=300)
    main(ap.parse_args().steps)
