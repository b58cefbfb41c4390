"""Logits to probabilities and verification of drafted tokens, against 64-bit and whole-number
restatements."""
import math

import numpy as np
import pytest

import sx

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def eng():
    e = sx.Engine(0)
    e.set_stream(sx.STREAM_LEGACY)
    yield e
    e.close()


# --------------------------------------------------------------------------------- probabilities
def check_probs(eng, z, temperature=1.0, ld=None, inplace=False):
    rows, n = z.shape
    ld = ld or n
    buf = torch.full((rows, ld), 9.0, device="cuda")
    buf[:, :n] = z
    out = buf if inplace else torch.full((rows, ld), 9.0, device="cuda")
    eng.probs(buf, out, rows, n, temperature=temperature, logits_ld=ld, probs_ld=ld)
    eng.sync()
    assert (out[:, n:] == 9.0).all()
    t = np.float32(temperature).item()
    want = torch.softmax(z.double() / t, -1)
    want = torch.where((z == -math.inf).all(-1, keepdim=True), 0.0, want)
    got = out[:, :n].double()
    assert torch.equal(got.isnan(), want.isnan())
    # the exponent's error is 2^-23 of its size, exp's and the sum's a few ulps; below the normal
    # range nothing is promised
    x = ((z.double() - z.double().amax(-1, keepdim=True)) / t).abs().clamp(max=200).nan_to_num(0.0)
    tol = want * (x * 2.0 ** -22 + 2.0 ** -20) + 2.0 ** -126
    bad = ~(((got - want).abs() <= tol) | want.isnan())
    assert not bad.any(), (int(bad.sum()), float((got - want).abs().max()))


@pytest.mark.parametrize("n", [1, 2, 31, 33, 1000, 4097, 32001, 151937, 262144, 300001])
@pytest.mark.parametrize("rows", [1, 3])
def test_probs_sizes(eng, n, rows):
    check_probs(eng, torch.randn(rows, n, device="cuda") * 4, 0.7)


@pytest.mark.parametrize("temperature", [1e-3, 0.1, 1.0, 50.0])
def test_probs_temperature_and_range(eng, temperature):
    check_probs(eng, torch.randn(4, 5001, device="cuda") * 20, temperature)
    check_probs(eng, torch.randn(4, 5001, device="cuda") * 1e30, temperature)


def test_probs_many_rows(eng):
    check_probs(eng, torch.randn(3000, 257, device="cuda"))


@pytest.mark.parametrize("n,ld", [(1000, 1003), (4096, 4100), (262143, 262147), (70001, 80000)])
def test_probs_strides_and_in_place(eng, n, ld):
    z = torch.randn(3, n, device="cuda") * 3
    check_probs(eng, z, 0.9, ld)
    check_probs(eng, z, 0.9, ld, inplace=True)


@pytest.mark.parametrize("n", [7, 5000, 262144])
def test_probs_special_values(eng, n):
    z = torch.randn(6, n, device="cuda")
    z[0] = -math.inf
    z[1, : n // 2] = -math.inf
    z[2, n // 3] = math.nan
    z[3, n // 2] = math.inf
    z[4] = torch.finfo(torch.float32).min
    z[5, n - 1] = 3e38
    check_probs(eng, z)


@pytest.mark.parametrize("n,rows,ld", [(65537, 40, 65537), (131072, 60, 131076), (262144, 20, 262147), (300001, 20, 300004)])
def test_probs_many_long_rows(eng, n, rows, ld):
    z = torch.randn(rows, n, device="cuda") * 3
    z[1] = -math.inf
    z[2, : n // 2] = -math.inf
    z[3, n // 3] = math.nan
    z[4, n - 1] = math.inf
    z[5] = torch.finfo(torch.float32).min
    check_probs(eng, z, 0.8, ld)
    check_probs(eng, z, 0.8, ld, inplace=True)


def test_probs_many_long_rows_repeat_in_a_graph(eng):
    z = torch.randn(24, 262144, device="cuda")
    want, out = torch.empty_like(z), torch.empty_like(z)
    eng.probs(z, want, 24, 262144)
    eng.sync()
    s = torch.cuda.Stream()
    try:
        with torch.cuda.stream(s):
            eng.set_stream(s.cuda_stream)
            eng.probs(z, out, 24, 262144)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                for _ in range(4):
                    eng.probs(z, out, 24, 262144)
            for _ in range(3):
                out.zero_()
                g.replay()
                s.synchronize()
                assert torch.equal(out, want)
    finally:
        eng.set_stream(sx.STREAM_LEGACY)


@pytest.mark.parametrize("rows,n", [(3000, 65537), (40, (1 << 24) - 3)])
def test_probs_more_rows_than_one_pass_holds(eng, rows, n):
    """Row by row against a softmax in 64 bits, at places of every pass over the rows."""
    z = torch.randn(rows, 4096, device="cuda")
    z = z.repeat(1, -(-n // 4096))[:, :n].contiguous()
    z[:, -1] = torch.arange(rows, device="cuda") % 7
    out = torch.empty_like(z)
    eng.probs(z, out, rows, n)
    eng.sync()
    for r in list(range(0, rows, max(1, rows // 40))) + [rows - 1]:
        want = torch.softmax(z[r].double(), -1)
        assert ((out[r] - want).abs() <= want * 2.0 ** -19).all(), r


@pytest.mark.parametrize("rows,n", [(1, (1 << 24) - 3), (2, 3_000_001), (24, (1 << 24) - 3)])
def test_probs_long_rows_that_repeat_themselves(eng, rows, n):
    """Equal parts err alike, and a plain chain of additions with them: 512 of 2^-25 in one pass, 64 in two."""
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(rows, 4096, device="cuda", generator=g).repeat(1, -(-n // 4096))[:, :n].contiguous()
    out = torch.empty_like(z)
    eng.probs(z, out, rows, n)
    eng.sync()
    for r in range(rows):
        want = torch.softmax(z[r].double(), -1)
        # the sum alone: what all of a row's probabilities have in common
        assert abs(float(((out[r] - want) / want).mean())) <= 2.0 ** -21, r


def test_probs_beside_attention(eng):
    """Captured in two graphs, long rows' probabilities and an attention that is cut over CTAs may run at
    the same time: they work in memory of their own."""
    d, n = 128, 6000
    data = torch.randint(0, 120, (n // 16, 2, 1, 2, 16 * d), dtype=torch.uint8, device="cuda")
    scale = torch.full((n // 16, 2, 1, 2), 2.0 ** -6, device="cuda")
    table = torch.arange(n // 16, dtype=torch.int32, device="cuda")[None]
    cache = sx.KV8(data, scale, table, 16, 2, d)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    z = torch.randn(24, 262144, device="cuda")
    for new in (1, 100):
        q = torch.randn(new, 8 * d, device="cuda")
        start, kv_len, out, p = ints(0, new), ints(n), torch.empty_like(q), torch.empty_like(z)
        eng.kv8_attn(cache, sx.DTYPE_F32, q, out, start, kv_len, new, 8, d ** -0.5)
        eng.probs(z, p, 24, 262144)
        eng.sync()
        want_out, want_p = out.clone(), p.clone()
        streams, graphs = [torch.cuda.Stream() for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
        try:
            for s, g, call in zip(streams, graphs, (lambda: eng.kv8_attn(cache, sx.DTYPE_F32, q, out, start, kv_len, new, 8, d ** -0.5),
                                                    lambda: eng.probs(z, p, 24, 262144))):
                with torch.cuda.graph(g, stream=s):
                    eng.set_stream(s.cuda_stream)
                    for _ in range(20):
                        call()
        finally:
            eng.set_stream(sx.STREAM_LEGACY)
        for _ in range(5):
            out.zero_()
            p.zero_()
            torch.cuda.synchronize()
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want_out) and torch.equal(p, want_p)


def test_probs_refusals(eng):
    z = torch.zeros(2, 8, device="cuda")
    for kw in (dict(logits=None), dict(probs=None), dict(n=0), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan),
               dict(temperature=math.inf), dict(logits_ld=7), dict(probs_ld=7), dict(n=(1 << 24) + 1), dict(probs=z, probs_ld=16)):
        a = dict(logits=z, probs=torch.empty_like(z), rows=2, n=8)
        a.update(kw)
        with pytest.raises(sx.SxError) as e:
            eng.probs(a.pop("logits"), a.pop("probs"), a.pop("rows"), a.pop("n"), **a)
        assert e.value.status == sx.SX_ERR_INVALID, kw
    eng.probs(z, z, 0, 8)


# ----------------------------------------------------------------------------------- verification
def whole(w):
    w = np.where(w > 0, np.minimum(w, np.float32(1)), np.float32(0)).astype(np.float32)
    return np.floor(w.astype(np.float64) * 2.0 ** 38).astype(object)


def want_verify(p, q, tok, ua, us, nd):
    """One sequence in Python integers."""
    m = 0
    while m < nd:
        x = int(tok[m])
        qx = np.float32(1) if q is None else q[m, x]
        if x >= p.shape[1] or not np.float32(ua[m]) * qx < p[m, x]:
            break
        m += 1
    if m < nd and q is not None:
        w = p[m] - q[m]
    else:
        w = p[m].copy()
        if m < nd and tok[m] < len(w):
            w[int(tok[m])] = 0
    w = whole(w)
    if w.sum() == 0:
        w = whole(p[m])
    total = int(w.sum())
    drawn = sx.NO_TOKEN
    if total:
        goal = total * int(np.floor(np.float64(us) * 2 ** 24)) >> 24
        c = 0
        for i, x in enumerate(w):
            c += int(x)
            if c > goal:
                drawn = i
                break
    out = [int(t) for t in tok[:m]] + [drawn]
    return m, out + [sx.NO_TOKEN] * (len(tok) + 1 - len(out))


def run_verify(eng, p, q, tok, ua, us, n_draft=None, ld=0):
    b, k1, v = p.shape
    k = k1 - 1

    def rows(x):
        if x is None or not ld:
            return x
        y = torch.full((*x.shape[:2], ld), 0.5, device="cuda")
        y[..., :v] = x
        return y

    out = torch.full((b, k1), 77, dtype=torch.int32, device="cuda")
    acc = torch.full((b,), 77, dtype=torch.int32, device="cuda")
    eng.verify(rows(p), rows(q), tok, ua, us, out, acc, b, k, v, n_draft=n_draft, target_ld=ld, draft_ld=ld)
    eng.sync()
    return out.cpu().numpy().view(np.uint32), acc.cpu().numpy()


def check_verify(eng, p, q, tok, ua, us, n_draft=None, ld=0):
    out, acc = run_verify(eng, p, q, tok, ua, us, n_draft, ld)
    b, k1, _ = p.shape
    pn, qn = p.cpu().numpy(), None if q is None else q.cpu().numpy()
    tn, an, un = tok.cpu().numpy(), ua.cpu().numpy(), us.cpu().numpy()
    for i in range(b):
        nd = k1 - 1 if n_draft is None else int(n_draft[i])
        m, want = want_verify(pn[i], None if qn is None else qn[i], tn[i], an[i], un[i], nd)
        assert int(acc[i]) == m and out[i].tolist() == want, (i, int(acc[i]), m, out[i].tolist(), want)
    return out, acc


def drawn_inputs(b, k, v, seed, spread=3.0, noise=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(b, k + 1, v, device="cuda", generator=g) * spread
    p = torch.softmax(z, -1)
    q = torch.softmax(z[:, :k] + noise * torch.randn(b, k, v, device="cuda", generator=g), -1)
    u = torch.rand(b, k, 1, device="cuda", generator=g)
    tok = torch.searchsorted(q.double().cumsum(-1), u.double()).clamp(max=v - 1)[..., 0].to(torch.int32)
    return p, q, tok, torch.rand(b, k, device="cuda", generator=g), torch.rand(b, device="cuda", generator=g)


@pytest.mark.parametrize("v", [1, 2, 5, 33, 1000, 4099, 32001])
@pytest.mark.parametrize("b,k", [(1, 1), (7, 3), (3, 8)])
def test_verify_against_integers(eng, v, b, k):
    p, q, tok, ua, us = drawn_inputs(b, k, v, v + b)
    check_verify(eng, p, q, tok, ua, us)
    check_verify(eng, p, None, tok, ua, us)


def test_verify_large_vocabulary(eng):
    p, q, tok, ua, us = drawn_inputs(2, 3, 262144, 5)
    check_verify(eng, p, q, tok, ua, us)


@pytest.mark.parametrize("ld", [1001, 1004, 1100])
def test_verify_strides(eng, ld):
    p, q, tok, ua, us = drawn_inputs(5, 3, 1000, 6)
    check_verify(eng, p, q, tok, ua, us, ld=ld)


def test_verify_every_place_of_refusal_and_extreme_draws(eng):
    b, k, v = 5, 4, 777
    for u_s in (0.0, 1 - 2.0 ** -24, 0.5):
        p, q, tok, _, us = drawn_inputs(b, k, v, 8)
        us[:] = u_s
        ua = torch.zeros(b, k, device="cuda")
        for i in range(b):  # sequence i refuses place i; the last accepts all
            p[i, torch.arange(k), tok[i].long()] += 0.25
            if i < k:
                ua[i, i] = 1.0
                q[i, i, int(tok[i, i])] = 1.0
                p[i, i, int(tok[i, i])] = 0.125
        out, acc = check_verify(eng, p, q, tok, ua, us)
        assert acc.tolist() == list(range(b))


def test_verify_ragged_and_no_drafts(eng):
    p, q, tok, ua, us = drawn_inputs(6, 3, 501, 9)
    nd = torch.tensor([0, 1, 2, 3, 0, 2], dtype=torch.int32, device="cuda")
    check_verify(eng, p, q, tok, ua, us, n_draft=nd)
    out, acc = run_verify(eng, p[:, :1].contiguous(), None, torch.empty(6, 0, dtype=torch.int32, device="cuda"), torch.empty(6, 0, device="cuda"), us)
    assert acc.tolist() == [0] * 6
    for i in range(6):
        assert out[i].tolist() == want_verify(p[i, :1].cpu().numpy(), None, [], [], float(us[i]), 0)[1]


def test_verify_degenerate_rows(eng):
    """Equal distributions, no weight at all, NaN, a draft the draft model gives no probability."""
    v, k = 100, 2
    p, q, tok, ua, us = drawn_inputs(6, k, v, 10)
    ua[:] = 0.999999
    q[0], q[1] = p[0, :k], p[1, :k]
    ua[0] = 1.0  # u q < p fails at equality: the difference is empty, the row itself is drawn from
    p[2] = 0.0
    p[3] = math.nan
    q[4] = 0.0
    p[5, :, 50:] = math.nan
    out, acc = check_verify(eng, p, q, tok, ua, us)
    assert out[2, 0] == sx.NO_TOKEN and out[3, 0] == sx.NO_TOKEN and acc[2] == acc[3] == 0
    p[:] = 5.0  # weights saturate at 1
    check_verify(eng, p, q, tok, ua, us)
    p[:] = math.inf
    check_verify(eng, p, None, tok, ua, us)


def test_verify_bad_tokens_are_refused_and_reported(eng):
    p, q, tok, ua, us = drawn_inputs(2, 2, 50, 11)
    ua[:] = 0.0
    tok[1, 1] = 50
    out, acc = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for dq in (q, None):
        eng.verify(p, dq, tok, ua, us, out, acc, 2, 2, 50)
        with pytest.raises(sx.SxError) as e:
            eng.sync()
        assert e.value.status == sx.SX_ERR_DEVICE
        assert acc.tolist() == [2, 1] and 0 <= int(out[1, 1]) < 50
    tok[1, 1] = 3
    eng.verify(p, q, tok, ua, us, out, acc, 2, 2, 50, n_draft=torch.tensor([3, 1], dtype=torch.int32, device="cuda"))
    with pytest.raises(sx.SxError):
        eng.sync()
    assert acc.tolist() == [2, 1]


def test_verify_keeps_the_target_distribution(eng):
    """The first token out is distributed as the target's row, whatever the draft proposes."""
    v, n = 8, 1 << 18
    g = torch.Generator(device="cuda").manual_seed(3)
    p1, q1 = (torch.softmax(2 * torch.randn(v, device="cuda", generator=g), -1) for _ in range(2))
    tok = torch.multinomial(q1, n, replacement=True, generator=g).to(torch.int32).reshape(n, 1)
    p, q = p1.expand(n, 2, v).contiguous(), q1.expand(n, 1, v).contiguous()
    out, acc = torch.empty(n, 2, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    eng.verify(p, q, tok, torch.rand(n, 1, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g), out, acc, n, 1, v)
    eng.sync()
    freq = torch.bincount(out[:, 0].long(), minlength=v).double() / n
    sigma = (p1.double() * (1 - p1.double()) / n).sqrt()
    assert ((freq - p1.double()).abs() <= 5 * sigma).all()
    rate = float(torch.minimum(p1, q1).sum())
    assert abs(float(acc.double().mean()) - rate) <= 5 * math.sqrt(rate * (1 - rate) / n)


def test_verify_and_probs_in_a_graph(eng):
    z = torch.randn(6, 4000, device="cuda")
    p, _, tok, ua, us = drawn_inputs(2, 2, 4000, 12)
    probs = torch.empty_like(z)
    out, acc = torch.empty(2, 3, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        eng.set_stream(s.cuda_stream)
        eng.probs(z, probs, 6, 4000)
        eng.verify(probs, None, tok, ua, us, out, acc, 2, 2, 4000)
    eng.set_stream(sx.STREAM_LEGACY)
    for seed in (1, 2):
        z.copy_(torch.randn(6, 4000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        check_probs(eng, z)
        p = torch.empty_like(z)
        eng.probs(z, p, 6, 4000)
        want_out, want_acc = run_verify(eng, p.reshape(2, 3, 4000), None, tok, ua, us)
        assert np.array_equal(out.cpu().numpy().view(np.uint32), want_out) and acc.tolist() == want_acc.tolist()


@pytest.mark.parametrize("v", [1, 100, 32001])
@pytest.mark.parametrize("u,counts_as", [(1.0, 1 - 2.0 ** -24), (1.5, 1 - 2.0 ** -24), (math.inf, 1 - 2.0 ** -24), (-1.0, 0.0), (-0.0, 0.0), (math.nan, 0.0)])
def test_verify_draws_with_any_number(eng, v, u, counts_as):
    """u outside [0, 1) draws the nearest token: every place of out is written."""
    p, q, tok, ua, us = drawn_inputs(3, 2, v, 13)
    us[:] = counts_as
    want = check_verify(eng, p, q, tok, ua, us)
    us[:] = u
    got = run_verify(eng, p, q, tok, ua, us)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_verify_refusals(eng):
    p, q, tok, ua, us = drawn_inputs(2, 2, 50, 11)
    out, acc = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    good = [p, q, tok, ua, us, out, acc, 2, 2, 50]
    for at, val in ((0, None), (2, None), (3, None), (4, None), (5, None), (6, None), (9, 0), (9, (1 << 24) + 1), (8, 2000)):
        a = list(good)
        a[at] = val
        with pytest.raises(sx.SxError) as e:
            eng.verify(*a)
        assert e.value.status == sx.SX_ERR_INVALID, at
    for ld in (dict(target_ld=49), dict(draft_ld=49)):
        with pytest.raises(sx.SxError):
            eng.verify(*good, **ld)
    good[7] = 0
    eng.verify(*good)
