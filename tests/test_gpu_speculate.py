"""The example of speculative decoding: what its cache holds at the end is what its tokens say."""
import importlib.util
import os

import numpy as np
import pytest

import sx

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

spec = importlib.util.spec_from_file_location("speculate", os.path.join(os.path.dirname(__file__), "..", "examples", "speculate.py"))
speculate = importlib.util.module_from_spec(spec)
spec.loader.exec_module(speculate)


def dense_rows(target, tokens):
    """Final rows of one sequence by plain attention in f32, nothing quantised."""
    d, hq, hkv = target.head_dim, target.q_heads, target.kv_heads
    n = len(tokens)
    pos = torch.arange(n, device="cuda").float()[:, None] * target.inv_freq
    cos, sin = pos.cos()[:, None], pos.sin()[:, None]

    def turn(x):
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    x = target.embed[tokens]
    seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    for layer in target.layers:
        h = speculate.rms(x)
        q, k, v = ((h @ layer[w]).float().view(n, -1, d) for w in "qkv")
        q, k = turn(speculate.rms(q)), turn(speculate.rms(k))
        k, v = k.repeat_interleave(hq // hkv, 1), v.repeat_interleave(hq // hkv, 1)
        s = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
        o = torch.einsum("hqk,khd->qhd", s.masked_fill(~seen, -torch.inf).softmax(-1), v).reshape(n, -1).bfloat16()
        x = x + o @ layer["o"]
        x = x + torch.nn.functional.gelu(speculate.rms(x) @ layer["up"]) @ layer["down"]
    return x


@pytest.mark.parametrize("drafts,temperature", [(0, 1.0), (1, 0.7), (4, 1.0)])
def test_speculate(drafts, temperature):
    eng = sx.Engine(0)
    eng.set_stream(sx.STREAM_LEGACY)
    lens, tokens, page, per = [1, 2, 17, 100, 200], 24, 16, 24
    pages = sx.Pages(per * len(lens), page, len(lens), per)
    target = speculate.Target(eng, pages, layers=2, hidden=256, q_heads=8, kv_heads=2, head_dim=64, vocab=1000,
                              num_pages=per * len(lens), page_tokens=page)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1000, n) for n in lens]
    got, hits, tried = speculate.generate(eng, target, prompts, tokens, drafts, temperature)
    eng.sync()
    assert all(len(t) == tokens and all(0 <= x < 1000 for x in t) for t in got)
    assert 0 <= hits <= tried and (drafts == 0 or hits > 0)
    # The next step's rows from the cache are those of a plain forward pass over the same tokens, up to
    # 8-bit keys and values: their error is at most 2^-4 of each element, 2^-6 of a row as a rule, and
    # the residual stream takes a third of it in, twice.
    for b, prompt in enumerate(prompts):
        n = pages.length(b)
        seq = np.concatenate([prompt, got[b]])[:n]
        if len(seq) < n:
            continue  # (more tokens were accepted than asked for)
        pages.truncate(b, n - 1)
        pages.extend(b, n)
        news = [0] * len(prompts)
        news[b] = 1
        row = target.rows(torch.as_tensor(seq[-1:], device="cuda"), news)[0].float()
        want = dense_rows(target, torch.as_tensor(seq, device="cuda"))[-1].float()
        assert (row - want).norm() <= 0.05 * want.norm()
    eng.sync()
    for b in range(len(prompts)):
        pages.truncate(b, 0)
    assert pages.free_count == per * len(lens)
    pages.close()
    eng.close()


@pytest.mark.parametrize("drafts,temperature", [(0, 1.0), (1, 0.7), (4, 1.0)])
def test_speculate_every_session_against_plain_attention(drafts, temperature):
    """What the cache holds for every session, cut to the tokens asked for, gives the next row of a plain
    forward pass over them (the bound is that of the test above)."""
    eng = sx.Engine(0)
    eng.set_stream(sx.STREAM_LEGACY)
    lens, tokens, page, per = [1, 2, 17, 100, 200], 24, 16, 24
    pages = sx.Pages(per * len(lens), page, len(lens), per)
    target = speculate.Target(eng, pages, layers=2, hidden=256, q_heads=8, kv_heads=2, head_dim=64, vocab=1000,
                              num_pages=per * len(lens), page_tokens=page)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1000, n) for n in lens]
    got, hits, tried = speculate.generate(eng, target, prompts, tokens, drafts, temperature)
    eng.sync()
    compared = 0
    for b, prompt in enumerate(prompts):
        seq = np.concatenate([prompt, got[b]])
        # the cache holds all but the newest token at least; more where a lucky session ran ahead
        n = min(pages.length(b), len(seq))
        assert n >= len(seq) - 1
        pages.truncate(b, n - 1)
        pages.extend(b, n)
        news = [0] * len(prompts)
        news[b] = 1
        row = target.rows(torch.as_tensor(seq[n - 1:n], device="cuda"), news)[0].float()
        want = dense_rows(target, torch.as_tensor(seq[:n], device="cuda"))[-1].float()
        assert (row - want).norm() <= 0.05 * want.norm()
        compared += 1
    assert compared == len(prompts)
    eng.sync()
    pages.close()
    eng.close()
