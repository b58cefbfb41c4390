"""The operators of speculative decoding over a paged 8-bit KV cache: cases, inputs, plain forms.

Four operators, each once as elementary torch operations in 32 bits and once as the call of the
library (``own``):

* ``append``  q / k RMS norm, position rotation, and the new keys and values quantised into the
              pages of an e4m3 cache with one power-of-two scale per 16 tokens and kv head;
* ``attn``    attention of one or many new rows per sequence over that cache;
* ``probs``   logits to probabilities at a temperature;
* ``verify``  acceptance of drafted tokens and the draw of the next one from given random numbers.

Layout of the cache.  ``data`` is uint8 [pages][kv heads][page / 16][2][16 D]: for every 16 tokens
a K record and a V record of 16 D e4m3 bytes.  Token t (0..15) and element d of a K record sit at
byte 512 (d / 32) + 16 (4 (t % 8) + (d % 32) / 8) + 8 (t / 8) + d % 8, of a V record at
512 (d / 32) + 16 (4 ((d % 32) / 4) + (t % 8) / 2) + 4 (d % 4) + t % 2 + 2 (t / 8).  ``scale`` is
f32 [pages][kv heads][page / 16][2]; a stored value is e4m3 times its scale.
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0
SCALE_EXP = 60  # scales are 2^-60 .. 2^60
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
ROPE_THETA = 1.0e6
EPS = 1e-6


# ------------------------------------------------------------------------------------ cases
def listed():
    base = {"q_heads": 16, "kv_heads": 8, "dim": 256, "rot": 64, "page": 64}
    one = {"q_heads": 8, "kv_heads": 1, "dim": 256, "rot": 64, "page": 64}
    return [
        # one decoded token of each of 8 sessions, 12B head layout: the append of every step
        dict(base, name="append_step", op="append", seqs=8, new=1, ctx=100000, dtype="f32", lens=1),
        # 64 packed prompts of 16 to 512 tokens enter the cache
        dict(base, name="append_prompts", op="append", seqs=64, new=512, ctx=0, dtype="bf16", lens=2),
        # one session on a ring-sized context: launch and merge latency
        dict(one, name="attn_one", op="attn", seqs=1, new=1, ctx=639, window=0, dtype="f32", lens=3),
        # a full decode batch, ragged contexts up to 8k: streaming the cache
        dict(base, name="attn_step", op="attn", seqs=64, new=1, ctx=8191, window=0, dtype="bf16", lens=4),
        # one session with a very long context: one token's work split over the whole GPU
        dict(base, name="attn_long", op="attn", seqs=1, new=1, ctx=131070, window=0, dim=128, dtype="f32", lens=5),
        # a token and four drafts per session, 8 q heads on 1 kv head: 40 rows share each key
        dict(one, name="attn_drafts", op="attn", seqs=32, new=5, ctx=16000, window=0, dtype="bf16", lens=6),
        # sliding-window layer of 16 sessions far into their contexts; old pages are released
        dict(base, name="attn_window", op="attn", seqs=16, new=1, ctx=100000, window=512, dtype="f32", lens=7),
        # ragged prompt chunks, each behind a context that is already cached
        dict(base, name="attn_prompts", op="attn", seqs=4, new=4096, ctx=4096, window=0, dim=128, dtype="bf16", lens=8),
        # sampling probabilities of one token
        dict(name="probs_one", op="probs", rows=1, vocab=262144, temperature=0.8),
        # the target's probabilities of a token and four drafts in 8 sessions
        dict(name="probs_drafts", op="probs", rows=40, vocab=262144, temperature=1.0),
        # verification for one session, and for a batch of them
        dict(name="verify_one", op="verify", seqs=1, drafts=4, vocab=262144, draft_probs=True),
        dict(name="verify_batch", op="verify", seqs=64, drafts=4, vocab=262144, draft_probs=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "attn", "attn", "attn", "attn", "probs", "verify"])
    if op == "probs":
        return dict(op=op, rows=_log(rng, 1, 40), vocab=_log(rng, 1000, 262144), temperature=round(rng.uniform(0.3, 1.5), 2))
    if op == "verify":
        return dict(op=op, seqs=_log(rng, 1, 64), drafts=rng.randint(1, 4), vocab=_log(rng, 1000, 262144), draft_probs=rng.random() < 0.7)
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128, 128, 256, 256, 512])
    case = dict(op=op, q_heads=kv * rng.choice([1, 2, 3, 4, 8] if kv < 4 else [1, 2]), kv_heads=kv, dim=dim,
                rot=rng.choice([dim, dim // 2, 32]), page=rng.choice([16, 32, 64, 128]),
                dtype=rng.choice(["f32", "bf16"]), lens=rng.randrange(1 << 20))
    if op == "append":
        seqs = _log(rng, 1, 64)
        return dict(case, seqs=seqs, new=rng.choice([1, rng.randint(2, 9), _log(rng, 10, 512)]), ctx=rng.choice([0, _log(rng, 1, 100000)]))
    kind = rng.choice(["step", "step", "drafts", "window", "prompt"])
    if kind == "prompt":
        new = _log(rng, 16, 2048)
        return dict(case, seqs=rng.randint(1, 4), new=new, ctx=rng.choice([0, _log(rng, 1, 4096)]), window=rng.choice([0, 0, _log(rng, 16, 1024)]))
    seqs = _log(rng, 1, 64)
    ctx = _log(rng, 1, 131070 // seqs)
    new = rng.randint(2, 8) if kind == "drafts" else 1
    return dict(case, seqs=seqs, new=new, ctx=ctx, window=_log(rng, 16, 1024) if kind == "window" else 0)


def _lengths(case):
    """New tokens and cached-before tokens of each sequence: part of the case, not of the seed."""
    rng = random.Random(case["lens"])
    n, ctx, ragged = [], [], case["new"] > 16
    for b in range(case["seqs"]):
        n.append(case["new"] if b == 0 or not ragged else rng.randint(min(16, case["new"]), case["new"]))
        ctx.append(case["ctx"] if b == 0 else rng.randint(0, case["ctx"]))
    return n, ctx


def work(case):
    if case["op"] == "probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 8 * n, "flops": 4 * n}
    if case["op"] == "verify":
        # one row pair per sequence for the residual, and two values per drafted token
        b, k, v = case["seqs"], case["drafts"], case["vocab"]
        rows = 2 if case["draft_probs"] else 1
        return {"bytes": b * rows * 4 * v + b * k * 16 + b * (k + 3) * 4, "flops": 2 * b * v}
    n, ctx = _lengths(case)
    t, d, es = sum(n), case["dim"], 4 if case["dtype"] == "f32" else 2
    hq, hkv = case["q_heads"], case["kv_heads"]
    if case["op"] == "append":
        return {"bytes": t * d * (2 * hq * es + 2 * hkv * es + 2 * hkv) + t * hkv, "flops": 8 * t * d * (hq + 2 * hkv)}
    keys = pairs = 0
    for nb, cb in zip(n, ctx):
        w = case["window"] or 1 << 40
        keys += min(nb + cb, w + nb - 1)
        full = max(0, min(nb, w - cb))  # rows that see their whole past
        pairs += full * cb + full * (full + 1) // 2 + (nb - full) * w
    return {"bytes": keys * hkv * (2 * d + 0.5) + 2 * t * hq * d * es, "flops": 4 * d * hq * pairs}


# ----------------------------------------------------------------------------------- inputs
def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e, within the scales' range."""
    bits = amax.view(torch.int32)
    e = (bits >> 23) - 127 - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)
    return e.clamp(-SCALE_EXP, SCALE_EXP)


def _e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _pack(k, v):
    """[..., 16, D] bytes of K and V -> [..., 2, 16 D] records."""
    lead, d = k.shape[:-2], k.shape[-1]
    m = len(lead)
    k = k.reshape(*lead, 2, 8, d // 32, 4, 8)  # h g p c j
    k = k.permute(*range(m), m + 2, m + 1, m + 3, m, m + 4).reshape(*lead, 16 * d)
    v = v.reshape(*lead, 2, 4, 2, d // 32, 8, 4)  # h c u p g i
    v = v.permute(*range(m), m + 3, m + 4, m + 1, m + 5, m, m + 2).reshape(*lead, 16 * d)
    return torch.stack((k, v), -2)


def _unpack(data, d):
    """[..., 2, 16 D] records -> K and V bytes [..., 16, D]."""
    lead = data.shape[:-2]
    m = len(lead)
    k = data[..., 0, :].reshape(*lead, d // 32, 8, 4, 2, 8)  # p g c h j
    k = k.permute(*range(m), m + 3, m + 1, m, m + 2, m + 4).reshape(*lead, 16, d)
    v = data[..., 1, :].reshape(*lead, d // 32, 8, 4, 4, 2, 2)  # p g c i h u
    v = v.permute(*range(m), m + 4, m + 2, m + 5, m, m + 1, m + 3).reshape(*lead, 16, d)
    return k, v


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(case, g, need):
    """Pages for `need` [(first, last) page] of each sequence, in shuffled order, filled with
    quantised normal values whose spread differs by block; table entries outside are -1."""
    d, hkv, nb = case["dim"], case["kv_heads"], case["page"] // 16
    pages = sum(hi - lo for lo, hi in need)
    width = max(hi for _, hi in need)
    order = list(range(pages))
    random.Random(case["lens"] + 1).shuffle(order)
    rows, at = [], 0
    for lo, hi in need:
        rows.append([-1] * lo + order[at:at + hi - lo] + [-1] * (width - hi))
        at += hi - lo
    data = torch.empty(pages, hkv, nb, 2, 16 * d, dtype=torch.uint8, device="cuda")
    scale = torch.empty(pages, hkv, nb, 2, device="cuda")
    step = max(1, (1 << 27) // (hkv * nb * 16 * d))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        x = torch.randn(2, n, hkv, nb, 16, d, device="cuda", generator=g)
        x *= torch.randn(2, n, hkv, nb, 1, 1, device="cuda", generator=g).mul_(0.5).exp2_()
        s = torch.ldexp(torch.ones((), device="cuda"), _exponent(x.abs().amax((-1, -2))))
        x = _e4m3(x.div_(s[..., None, None])).view(torch.uint8)
        data[i:i + n] = _pack(x[0], x[1])
        scale[i:i + n] = s.permute(1, 2, 3, 0)
    return data, scale, torch.tensor(rows, dtype=torch.int32, device="cuda")


def _rows(n, ctx):
    start = [0]
    for x in n:
        start.append(start[-1] + x)
    put = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return put(start), put([a + b for a, b in zip(n, ctx)])


def prepare(case, seed):
    g = _gen(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if case["op"] == "probs":
        z = rand(case["rows"], case["vocab"]) * 3
        return {"case": case, "logits": z, "probs": torch.empty_like(z)}
    if case["op"] == "verify":
        b, k, v = case["seqs"], case["drafts"], case["vocab"]
        z = rand(b, k + 1, v) * 3
        p = torch.softmax(z, -1)
        if case["draft_probs"]:
            q = torch.softmax(z[:, :k] + 0.7 * rand(b, k, v), -1)
            u = torch.rand(b, k, 1, device="cuda", generator=g)
            tokens = torch.searchsorted(q.double().cumsum(-1), u.double()).clamp(max=v - 1)[..., 0]
        else:
            q, tokens = None, z[:, :k].argmax(-1)
        return {"case": case, "target": p, "draft": q, "tokens": tokens.to(torch.int32),
                "u_accept": torch.rand(b, k, device="cuda", generator=g), "u_sample": torch.rand(b, device="cuda", generator=g),
                "out": torch.empty(b, k + 1, dtype=torch.int32, device="cuda"), "accepted": torch.empty(b, dtype=torch.int32, device="cuda")}
    n, ctx = _lengths(case)
    start, kv_len = _rows(n, ctx)
    t, d, hq, hkv, page, dt = sum(n), case["dim"], case["q_heads"], case["kv_heads"], case["page"], DTYPES[case["dtype"]]
    state = {"case": case, "start": start, "kv_len": kv_len, "tokens": t, "most": max(n)}
    last = [-(-(a + b) // page) for a, b in zip(n, ctx)]
    if case["op"] == "append":
        data, scale, table = _cache(case, g, [(b // page, hi) for b, hi in zip(ctx, last)])
        qkv = (rand(t, (hq + 2 * hkv) * d) * 2).to(dt)  # one projection's rows: q | k | v
        freq = torch.tensor([ROPE_THETA ** (-2 * i / case["rot"]) for i in range(case["rot"] // 2)], dtype=torch.float64)
        return dict(state, data=data, scale=scale, table=table, q=qkv[:, :hq * d], k=qkv[:, hq * d:(hq + hkv) * d], v=qkv[:, (hq + hkv) * d:],
                    q_norm=1 + 0.1 * rand(d), k_norm=1 + 0.1 * rand(d), inv_freq=freq.float().cuda(), q_out=torch.empty(t, hq * d, dtype=dt, device="cuda"))
    first = [max(0, b - (case["window"] or 1 << 40) + 1) // page for b in ctx]
    data, scale, table = _cache(case, g, list(zip(first, last)))
    q = rand(t, hq * d).to(dt)
    return dict(state, data=data, scale=scale, table=table, q=q, out=torch.empty_like(q), qk_scale=d ** -0.5)


# -------------------------------------------------------------------------- the plain forms
def _norm(x, w):
    x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))
    return x if w is None else x * w


def _rotate(x, pos, inv_freq):
    """x [T, heads, D]; the first 2 len(inv_freq) elements in pairs (i, i + half)."""
    half = inv_freq.numel()
    a = (pos.float()[:, None] * inv_freq)[:, None, :]
    c, s = torch.cos(a), torch.sin(a)
    x0, x1 = x[..., :half], x[..., half:2 * half]
    return torch.cat((x0 * c - x1 * s, x0 * s + x1 * c, x[..., 2 * half:]), -1)


def _positions(s):
    """Sequence and position of each row."""
    row = torch.arange(s["tokens"], device="cuda")
    seq = (row[:, None] >= s["start"][None, 1:]).sum(-1)
    return seq, s["kv_len"][seq].long() - s["start"][seq + 1] + row


def _plain_append(s):
    case = s["case"]
    d, hq, hkv, page = case["dim"], case["q_heads"], case["kv_heads"], case["page"]
    seq, pos = _positions(s)
    q = _rotate(_norm(s["q"].float().reshape(-1, hq, d), s["q_norm"]), pos, s["inv_freq"])
    k = _rotate(_norm(s["k"].float().reshape(-1, hkv, d), s["k_norm"]), pos, s["inv_freq"])
    v = _norm(s["v"].float().reshape(-1, hkv, d), None)
    # block of each row, [pages * page / 16] blocks in all
    blk = s["table"][seq, pos // page].long() * (page // 16) + pos % page // 16
    nblk = s["data"].shape[0] * (page // 16)
    new = torch.stack((k, v), 2)  # T, kv, 2, D
    top = torch.zeros(nblk, hkv, 2, device="cuda").scatter_reduce_(0, blk[:, None, None].expand(-1, hkv, 2), new.abs().amax(-1), "amax")
    fresh = torch.zeros(nblk, dtype=torch.bool, device="cuda").index_fill_(0, blk[pos % 16 == 0], True)
    old_scale = s["scale"].transpose(1, 2).reshape(nblk, hkv, 2)
    old_e = torch.where(fresh[:, None, None], -SCALE_EXP, _exponent(old_scale * E4M3_MAX))
    e = torch.maximum(old_e, _exponent(top))
    scale = torch.ldexp(torch.ones((), device="cuda"), e)
    # what was there, at the new scale; a block whose first token is new starts empty
    old = torch.stack(_unpack(s["data"].transpose(1, 2).reshape(nblk, hkv, 2, 16 * d), d), 2)  # nblk, kv, 2, 16, D
    old = old.view(torch.float8_e4m3fn).float() * (old_scale / scale)[..., None, None]
    old = torch.where(fresh[:, None, None, None, None], 0.0, old)
    vals = _e4m3(old).view(torch.uint8)
    vals[blk, :, :, pos % 16] = _e4m3(new / scale[blk][..., None]).view(torch.uint8)
    data = _pack(vals[:, :, 0], vals[:, :, 1]).reshape(-1, page // 16, hkv, 2, 16 * d).transpose(1, 2).contiguous()
    scale = scale.reshape(-1, page // 16, hkv, 2).transpose(1, 2).contiguous()
    return {"data": data.view(torch.float8_e4m3fn), "scale": scale, "q": q.reshape(-1, hq * d).to(s["q"].dtype)}


def _plain_attn(s):
    case = s["case"]
    d, hq, hkv, page, window = case["dim"], case["q_heads"], case["kv_heads"], case["page"], case["window"]
    b, n, rep = case["seqs"], s["most"], hq // hkv
    count, kv_len = s["start"].diff().long(), s["kv_len"].long()
    # the pages that rows of a sequence can see
    width = s["table"].shape[1]
    lo = ((kv_len - count - window + 1).clamp(min=0) // page) if window else torch.zeros_like(kv_len)
    width = min(width, (window + n - 2) // page + 2) if window else width
    at = lo[:, None] + torch.arange(width, device="cuda")
    ids = torch.gather(s["table"].long(), 1, at.clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    k, v = _unpack(s["data"][ids].transpose(1, 2), d)  # b, kv, width, page / 16, 16, D
    sc = s["scale"][ids].transpose(1, 2)
    k = (k.view(torch.float8_e4m3fn).float() * sc[..., 0, None, None]).reshape(b, hkv, width * page, d)
    v = (v.view(torch.float8_e4m3fn).float() * sc[..., 1, None, None]).reshape(b, hkv, width * page, d)
    # rows padded to the longest sequence
    i = torch.arange(n, device="cuda")
    row = (s["start"][:-1, None].long() + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[row].reshape(b, n, hkv, rep, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, rep * n, d)
    z = (q @ k.transpose(-1, -2)).reshape(b, hkv, rep, n, -1) * s["qk_scale"]
    key = (lo[:, None] * page + torch.arange(width * page, device="cuda"))[:, None, :]
    pos = (kv_len - count)[:, None, None] + i[:, None]
    seen = (key <= pos) & (key < kv_len[:, None, None])
    if window:
        seen &= key > pos - window
    z = torch.where(seen[:, None, None], z, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    p /= p.sum(-1, keepdim=True).clamp(min=1e-38)
    out = (p.reshape(b, hkv, rep * n, -1) @ v).reshape(b, hkv, rep, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, hq * d)
    return out[i < count[:, None]].to(s["q"].dtype)


def _plain_probs(s):
    z = s["logits"] / s["case"]["temperature"]
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-38)


def _plain_verify(s):
    p, q, tok = s["target"], s["draft"], s["tokens"].long()
    b, k, v = p.shape[0], tok.shape[1], p.shape[2]
    p_tok = p[:, :k].gather(-1, tok[..., None])[..., 0]
    q_tok = torch.ones_like(p_tok) if q is None else q.gather(-1, tok[..., None])[..., 0]
    ok = (s["u_accept"] * q_tok < p_tok).to(torch.int32)
    m = ok.cumprod(-1).sum(-1)  # drafts accepted
    at = torch.arange(b, device="cuda")
    rest = p[at, m]
    cut = m.clamp(max=k - 1)
    if q is None:
        less = rest.scatter(-1, tok[at, cut][:, None], 0.0)
    else:
        less = rest - q[at, cut]
    less = torch.where((m < k)[:, None], less, rest)
    # probabilities as multiples of 2^-38: sums are exact and do not depend on their order
    whole = lambda w: (torch.where(w > 0, w.clamp(max=1.0), 0.0) * 2.0 ** 38).to(torch.int64)  # noqa: E731
    w = whole(less)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, whole(rest))
    c = w.cumsum(-1)
    total = c[:, -1]
    u = (s["u_sample"] * 2.0 ** 24).to(torch.int64)
    goal = (total >> 24) * u + (((total & 0xFFFFFF) * u) >> 24)
    drawn = torch.where(total > 0, (c <= goal[:, None]).sum(-1), -1)
    i = torch.arange(k + 1, device="cuda")
    out = torch.where(i < m[:, None], torch.cat((tok, tok[:, :1]), 1), torch.where(i == m[:, None], drawn[:, None], -1))
    return {"tokens": out.to(torch.int32), "accepted": m.to(torch.int32)}


# ------------------------------------------------------------------------ the library's calls
_held = {}


def _engine():
    if not _held:
        import os
        import sys

        sys.path.append(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ai-research_b200"))
        import sx

        e = sx.Engine(0)
        e.set_stream(torch.cuda.current_stream().cuda_stream or sx.STREAM_LEGACY)
        _held.update(sx=sx, engine=e)
    return _held["sx"], _held["engine"]


def _own(s):
    sx, e = _engine()
    case = s["case"]
    op = case["op"]
    if op == "probs":
        e.probs(s["logits"], s["probs"], case["rows"], case["vocab"], temperature=case["temperature"])
        return s["probs"]
    if op == "verify":
        e.verify(s["target"], s["draft"], s["tokens"], s["u_accept"], s["u_sample"], s["out"], s["accepted"],
                 case["seqs"], case["drafts"], case["vocab"])
        return {"tokens": s["out"], "accepted": s["accepted"]}
    cache = sx.KV8(s["data"], s["scale"], s["table"], case["page"], case["kv_heads"], case["dim"])
    dt = sx.DTYPE_F32 if case["dtype"] == "f32" else sx.DTYPE_BF16
    if op == "append":
        e.kv8_append(cache, dt, s["q"], s["k"], s["v"], s["q_out"], s["start"], s["kv_len"], s["tokens"], case["q_heads"],
                     s["inv_freq"], case["rot"], q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], v_norm=True, eps=EPS,
                     q_ld=s["q"].stride(0), k_ld=s["k"].stride(0), v_ld=s["v"].stride(0))
        return {"data": s["data"].view(torch.float8_e4m3fn), "scale": s["scale"], "q": s["q_out"]}
    e.kv8_attn(cache, dt, s["q"], s["out"], s["start"], s["kv_len"], s["tokens"], case["q_heads"], s["qk_scale"], window=case["window"])
    return s["out"]


_PLAIN = {"append": _plain_append, "attn": _plain_attn, "probs": _plain_probs, "verify": _plain_verify}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------------------- 64-bit definitions
def _grid(x):
    """x (f64) to the nearest e4m3 number, ties to the even one."""
    a = x.abs().clamp(max=E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign(torch.round(a / step) * step, x)


def _table64():
    """Values of the 256 e4m3 codes."""
    out = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        val = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        out.append(math.nan if c & 127 == 127 else -val if c & 128 else val)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _places(d):
    """Byte of (token, element) in a K and in a V record."""
    t, e = torch.arange(16, device="cuda")[:, None], torch.arange(d, device="cuda")[None]
    in_k = 512 * (e // 32) + 16 * (4 * (t % 8) + e % 32 // 8) + 8 * (t // 8) + e % 8
    in_v = 512 * (e // 32) + 16 * (4 * (e % 32 // 4) + t % 8 // 2) + 4 * (e % 4) + t % 2 + 2 * (t // 8)
    return in_k.reshape(-1), in_v.reshape(-1)


def _exact_append(s):
    case = s["case"]
    d, hq, hkv, page, rot = case["dim"], case["q_heads"], case["kv_heads"], case["page"], case["rot"]
    in_k, in_v = _places(d)
    codes = _table64()
    data, scale = codes[s["data"].long()], s["scale"].double()
    start, kv_len, table = s["start"].tolist(), s["kv_len"].tolist(), s["table"].tolist()
    q_out = torch.empty(s["tokens"], hq, d, dtype=torch.float64, device="cuda")
    for b in range(case["seqs"]):
        r0, r1 = start[b], start[b + 1]
        n, first = r1 - r0, kv_len[b] - (r1 - r0)
        pos = torch.arange(first, kv_len[b], device="cuda")
        # the rotation's angle is the 32-bit product of position and frequency, by definition
        ang = (pos.float()[:, None] * s["inv_freq"][None]).double()
        turn = torch.polar(torch.ones_like(ang), ang)[:, None]

        def normed(x, w):
            x = x[r0:r1].double().reshape(n, -1, d)
            x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt()
            return x if w is None else x * w.double()

        def turned(x):
            y = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot].contiguous()) * turn
            return torch.cat((y.real, y.imag, x[..., rot:]), -1)

        q_out[r0:r1] = turned(normed(s["q"], s["q_norm"]))
        kv = (turned(normed(s["k"], s["k_norm"])), normed(s["v"], None))
        for j0 in range(first // 16, -(-kv_len[b] // 16)):
            page_id, slot = table[b][j0 * 16 // page], j0 % (page // 16)
            lo, hi = max(first, j0 * 16), min(kv_len[b], j0 * 16 + 16)
            for which, place in ((0, in_k), (1, in_v)):
                new = kv[which][lo - first:hi - first].transpose(0, 1)  # kv, tokens, D
                old = data[page_id, :, slot, which][:, place].reshape(hkv, 16, d)
                was = scale[page_id, :, slot, which].clone()
                if lo == j0 * 16:
                    old, was = torch.zeros_like(old), torch.full_like(was, 2.0 ** -SCALE_EXP)
                fit = torch.exp2(torch.ceil(torch.log2(new.abs().amax((-1, -2)).clamp(min=1e-300) / E4M3_MAX)).clamp(-SCALE_EXP, SCALE_EXP))
                now = torch.maximum(was, fit)
                old = _grid(old * (was / now)[:, None, None])
                old[:, lo - j0 * 16:hi - j0 * 16] = _grid(new / now[:, None, None])
                data[page_id, :, slot, which] = torch.empty_like(data[page_id, :, slot, which]).index_copy_(1, place, old.reshape(hkv, -1))
                scale[page_id, :, slot, which] = now
    return {"data": data, "scale": scale, "q": q_out.reshape(-1, hq * d)}


def _exact_attn(s):
    case = s["case"]
    d, hq, hkv, page = case["dim"], case["q_heads"], case["kv_heads"], case["page"]
    in_k, in_v = _places(d)
    codes = _table64()
    start, kv_len, table = s["start"].tolist(), s["kv_len"].tolist(), s["table"].tolist()
    out = torch.zeros(s["tokens"], hq, d, dtype=torch.float64, device="cuda")
    for b in range(case["seqs"]):
        r0, r1, total = start[b], start[b + 1], kv_len[b]
        first = total - (r1 - r0)
        begin = max(0, first - case["window"] + 1) // page * page if case["window"] else 0
        ids = table[b][begin // page:-(-total // page)]
        pos = torch.arange(first, total, device="cuda")[:, None]
        key = torch.arange(begin, total, device="cuda")[None]
        hidden = key > pos
        if case["window"]:
            hidden |= pos - key >= case["window"]
        for h in range(hkv):
            rec = s["data"][ids, h]  # pages, page / 16, 2, 16 D
            sc = s["scale"][ids, h].double().repeat_interleave(16, 1)
            k, v = (codes[rec[:, :, w][..., place].long()].reshape(-1, d)[:total - begin] for w, place in ((0, in_k), (1, in_v)))
            ks, vs = (sc[..., w].reshape(-1, 1)[:total - begin] for w in (0, 1))
            for g in range(h * hq // hkv, (h + 1) * hq // hkv):
                z = s["q"][r0:r1, g * d:(g + 1) * d].double() @ (k * ks).T * s["qk_scale"]
                out[r0:r1, g] = torch.softmax(z.masked_fill_(hidden, -math.inf), -1) @ (v * vs)
    return out.reshape(-1, hq * d)


def exact(case, seed):
    """run()'s outputs in 64 bits; verify's are whole numbers and have none."""
    if case["op"] == "verify":
        return None
    s = prepare(case, seed)
    if case["op"] == "probs":
        return torch.softmax(s["logits"].double() / case["temperature"], -1)
    return _exact_append(s) if case["op"] == "append" else _exact_attn(s)
