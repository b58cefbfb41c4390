"""Speculative decoding of several sessions over one paged 8-bit KV cache per layer.

    python examples/speculate.py [--sessions 8] [--tokens 64] [--drafts 4] ...

A random-weight transformer (its dense products are torch's) is decoded with the paged operators of
sx: every step drafts a few tokens per session with a cheap model (the target without its layers),
runs the target once over them, and keeps what verification accepts:

    Pages.extend -> kv8_append -> kv8_attn (each layer) -> probs -> verify -> Pages.truncate

Prompts enter through the same two calls, packed, whatever their lengths.
"""
import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "ai-research_b200"))
import sx  # noqa: E402


def rms(x, eps=1e-6):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps)).to(x.dtype)


class Target:
    """layers x (attention over the paged cache, feed forward) between an embedding and a head."""

    def __init__(self, eng, pages, layers=4, hidden=1024, q_heads=16, kv_heads=8, head_dim=64, vocab=32000,
                 num_pages=256, page_tokens=64, window=0, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.eng, self.pages, self.page_tokens, self.vocab = eng, pages, page_tokens, vocab
        self.q_heads, self.kv_heads, self.head_dim, self.window = q_heads, kv_heads, head_dim, window

        def w(*shape):
            return (torch.randn(*shape, device="cuda", generator=g) * shape[0] ** -0.5).bfloat16()

        self.embed = torch.randn(vocab, hidden, device="cuda", generator=g).bfloat16()
        self.head = w(hidden, vocab)
        kv = kv_heads * head_dim
        self.layers = [dict(q=w(hidden, q_heads * head_dim), k=w(hidden, kv), v=w(hidden, kv), o=0.3 * w(q_heads * head_dim, hidden),
                            up=w(hidden, 2 * hidden), down=0.3 * w(2 * hidden, hidden)) for _ in range(layers)]
        self.gain = torch.ones(head_dim, device="cuda")
        self.inv_freq = torch.from_numpy(sx.rope_inv_freq(head_dim, 10000.0).copy()).cuda()
        blocks = num_pages * kv_heads * (page_tokens // 16)
        self.data = [torch.zeros(blocks * 2 * 16 * head_dim, dtype=torch.uint8, device="cuda") for _ in self.layers]
        self.scale = [torch.zeros(blocks * 2, device="cuda") for _ in self.layers]

    def rows(self, tokens, news):
        """Final hidden rows of packed new tokens, news[b] of them for sequence b (the pages are there)."""
        n = int(sum(news))
        start = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device="cuda")
        lens = torch.tensor([self.pages.length(b) if k else 0 for b, k in enumerate(news)], dtype=torch.int32, device="cuda")
        table = torch.from_numpy(self.pages.table().view(np.int32)).cuda()
        x = self.embed[tokens]
        for layer, data, scale in zip(self.layers, self.data, self.scale):
            cache = sx.KV8(data, scale, table, self.page_tokens, self.kv_heads, self.head_dim)
            h = rms(x)
            q, k, v = h @ layer["q"], h @ layer["k"], h @ layer["v"]
            self.eng.kv8_append(cache, sx.DTYPE_BF16, q, k, v, q, start, lens, n, self.q_heads, self.inv_freq, self.head_dim,
                                q_norm_w=self.gain, k_norm_w=self.gain)
            out = torch.empty_like(q)
            self.eng.kv8_attn(cache, sx.DTYPE_BF16, q, out, start, lens, n, self.q_heads, self.head_dim ** -0.5, window=self.window)
            x = x + out @ layer["o"]
            x = x + torch.nn.functional.gelu(rms(x) @ layer["up"]) @ layer["down"]
        return x

    def logits(self, x):
        return 3.0 * (rms(x) @ self.head).float()


def generate(eng, target, prompts, tokens, drafts=4, temperature=1.0, seed=1):
    """Samples `tokens` tokens after every prompt.  Returns them and how many drafts were accepted
    of how many."""
    pages, seqs, vocab = target.pages, len(prompts), target.vocab
    gen = torch.Generator(device="cuda").manual_seed(seed)
    uniform = lambda *shape: torch.rand(*shape, device="cuda", generator=gen)  # noqa: E731
    empty = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
    accepted, one = (torch.empty(seqs, dtype=torch.int32, device="cuda") for _ in range(2))
    p, q = empty(seqs, drafts + 1, vocab), empty(seqs, max(drafts, 1), vocab)
    tok = torch.zeros(seqs, max(drafts, 1), dtype=torch.int32, device="cuda")
    out = torch.empty(seqs, drafts + 1, dtype=torch.int32, device="cuda")

    # prompts: all but their last token enter the cache
    news = [len(t) - 1 for t in prompts]
    for b, n in enumerate(news):
        pages.extend(b, n)
    if sum(news):
        target.rows(torch.cat([torch.as_tensor(t[:-1], device="cuda") for t in prompts]), news)
    last = torch.tensor([int(t[-1]) for t in prompts], device="cuda")
    got, hits, tried = [[] for _ in prompts], 0, 0
    while min(len(t) for t in got) < tokens:
        # draft: the target without its layers, one token at a time; verify draws when nothing is drafted
        seq, token = [last], last
        draw = torch.empty(seqs, 1, dtype=torch.int32, device="cuda")
        for i in range(drafts):
            row = empty(seqs, vocab)
            eng.probs(target.logits(target.embed[token]), row, seqs, vocab, temperature)
            eng.verify(row, None, None, None, uniform(seqs), draw, one, seqs, 0, vocab)
            q[:, i], tok[:, i] = row, draw[:, 0]
            token = draw[:, 0].long()
            seq.append(token)
        # the target over the last token and its drafts
        for b in range(seqs):
            pages.extend(b, pages.length(b) + drafts + 1)
        x = target.rows(torch.stack(seq, 1).reshape(-1), [drafts + 1] * seqs)
        eng.probs(target.logits(x), p, seqs * (drafts + 1), vocab, temperature)
        eng.verify(p, q if drafts else None, tok if drafts else None, uniform(seqs, drafts) if drafts else None, uniform(seqs),
                   out, accepted, seqs, drafts, vocab)
        # what was refused leaves the cache
        kept, ids = accepted.tolist(), out.tolist()
        for b, n in enumerate(kept):
            pages.truncate(b, pages.length(b) - (drafts - n))
            got[b] += ids[b][:n + 1]
        last = out.long().gather(1, accepted.long()[:, None])[:, 0]
        hits += sum(kept)
        tried += drafts * seqs
    return [t[:tokens] for t in got], hits, tried


def main(argv=None):
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument("--sessions", type=int, default=8)
    a.add_argument("--tokens", type=int, default=64)
    a.add_argument("--drafts", type=int, default=4)
    a.add_argument("--temperature", type=float, default=1.0)
    a.add_argument("--prompt", type=int, default=300, help="longest prompt; lengths are drawn up to it")
    a = a.parse_args(argv)
    rng = np.random.default_rng(0)
    lens = rng.integers(1, a.prompt + 1, a.sessions)
    # (a lucky session runs ahead of the slowest by `drafts` tokens a step)
    per = -(-(a.prompt + (a.tokens + 1) * (a.drafts + 1)) // 64)
    eng = sx.Engine(0)
    eng.set_stream(sx.STREAM_LEGACY)
    pages = sx.Pages(per * a.sessions, 64, a.sessions, per)
    target = Target(eng, pages, num_pages=per * a.sessions)
    prompts = [rng.integers(0, target.vocab, n) for n in lens]
    start = time.perf_counter()
    got, hits, tried = generate(eng, target, prompts, a.tokens, a.drafts, a.temperature)
    eng.sync()
    seconds = time.perf_counter() - start
    print(f"{a.sessions} sessions x {a.tokens} tokens in {seconds:.2f} s; {hits} of {tried} drafts accepted; first session: {got[0][:12]}")
    pages.close()
    eng.close()


if __name__ == "__main__":
    main()
