"""The feed-forward block in 8-bit whole numbers against whole-number and 64-bit restatements.

Tolerances count roundings: half a step of f32 is 2^-24 of a value (F below), of bf16 2^-8."""
import math

import pytest

import sx

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F, HALF_BF16 = 2.0 ** -24, 2.0 ** -8
TYPES = {torch.float32: sx.DTYPE_F32, torch.bfloat16: sx.DTYPE_BF16, torch.int8: sx.DTYPE_I8}
JUNK = 77


@pytest.fixture(scope="module")
def eng():
    e = sx.Engine(0)
    e.set_stream(sx.STREAM_LEGACY)
    yield e
    e.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def wide(rows, n, ld, dtype):
    """[rows][n] inside a buffer of stride ld whose other elements are JUNK."""
    buf = torch.full((rows, ld), JUNK, dtype=dtype, device="cuda")
    return buf, buf[:, :n]


# ------------------------------------------------------------------------------------ products
def operands(t, n, k, seed, x_ld=0, w_ld=0, gated=False, lo=-127):
    g = gen(seed)

    def codes(rows, ld):
        buf, v = wide(rows, k, ld or k, torch.int8)
        v.copy_(torch.randint(lo, 128, (rows, k), device="cuda", generator=g, dtype=torch.int32))
        return v, torch.rand(rows, device="cuda", generator=g) * 0.02 / math.sqrt(k) + 1e-5

    return [codes(t, x_ld)] + [codes(n, w_ld) for _ in range(2 if gated else 1)]


def sums(x, w):
    """Whole numbers below 2^53: exact in f64 whatever the order."""
    return x.double() @ w.double().T


def rounding(dtype):
    return HALF_BF16 if dtype == torch.bfloat16 else 0.0


def check_gemm(eng, t, n, k, dtype=torch.float32, seed=0, x_ld=0, w_ld=0, y_ld=0, lo=-127, y_off=0):
    (x, xs), (w, ws) = operands(t, n, k, seed, x_ld, w_ld, lo=lo)
    ld = y_ld or n
    buf = torch.full((t * ld + y_off,), JUNK, dtype=dtype, device="cuda")
    y = buf[y_off:].view(t, ld)
    eng.gemm_i8(x, xs, w, ws, TYPES[dtype], y, t, n, k, x_ld=x.stride(0), w_ld=w.stride(0), y_ld=ld)
    eng.sync()
    assert (y[:, n:] == JUNK).all() and (buf[:y_off] == JUNK).all()
    want = sums(x, w) * xs.double()[:, None] * ws.double()
    # the sum, and its products with the two scales, are rounded to f32; then to the type
    tol = want.abs() * (3.01 * F + rounding(dtype))
    err = (y[:, :n].double() - want).abs()
    assert (err <= tol).all(), (int((err > tol).sum()), float((err / want.abs().clamp(min=1e-30)).max()))


def gelu(g):
    return g / (1 + torch.exp(-2 * 0.7978845608 * (g + 0.044715 * g ** 3)))


def check_gate_up(eng, t, n, k, dtype=torch.float32, seed=0, x_ld=0, w_ld=0, y_ld=0, scale=1.0):
    (x, xs), (wg, gs), (wu, us) = operands(t, n, k, seed, x_ld, w_ld, gated=True)
    xs = xs * scale
    buf, y = wide(t, n, y_ld or n, dtype)
    eng.gate_up_i8(x, xs, wg, gs, wu, us, TYPES[dtype], buf, t, n, k, x_ld=x.stride(0), w_ld=wg.stride(0), y_ld=y_ld)
    eng.sync()
    assert (buf[:, n:] == JUNK).all()
    g = sums(x, wg) * xs.double()[:, None] * gs.double()
    u = sums(x, wu) * xs.double()[:, None] * us.double()
    want = gelu(g) * u
    # g and u err by 3 F; z = c (g + 0.044715 g^3) by 14 F of itself; e^-2z by that (absolute 28 F |z|) and by
    # 2 + 1.173 |2 z| ulps of 2 F; the sum, the quotient (2 ulps) and the last product by F, 4 F and F; u 3 F
    z = (0.7978845608 * (g + 0.044715 * g ** 3)).abs()
    tol = want.abs() * ((18 + 33 * z) * F + rounding(dtype)) + (g * u).abs() * 2.0 ** -125 + 2.0 ** -149
    err = (y.double() - want).abs()
    assert (err <= tol).all(), (int((err > tol).sum()), float((err / tol.clamp(min=1e-300)).max()))


SIZES = [(1, 1, 16), (1, 64, 64), (2, 100, 48), (3, 129, 400), (5, 37, 1552), (7, 16, 32), (8, 3840, 256), (9, 511, 144), (15, 2050, 784),
         (16, 1000, 512), (17, 127, 128), (31, 257, 272), (33, 640, 2064), (64, 128, 128), (65, 4099, 160), (100, 1, 96), (127, 300, 1024),
         (128, 256, 3840), (129, 385, 640), (200, 1537, 1040), (256, 256, 256), (257, 513, 128), (300, 77, 6144), (511, 1023, 336),
         (640, 512, 15360), (1000, 3000, 176), (2049, 130, 1536)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,n,k", SIZES)
def test_gemm_sizes(eng, t, n, k, dtype):
    check_gemm(eng, t, n, k, dtype, seed=t + n + k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,n,k", SIZES)
def test_gate_up_sizes(eng, t, n, k, dtype):
    check_gate_up(eng, t, n, k, dtype, seed=t + n + k)


@pytest.mark.parametrize("t", list(range(1, 41)) + [48, 56, 72, 96, 160, 384])
def test_every_small_number_of_rows(eng, t):
    check_gemm(eng, t, 333, 720, seed=t)
    check_gate_up(eng, t, 207, 720, torch.bfloat16, seed=t)


# more tiles than run at a time, with few, some and many left over; many groups of rows; many short rows of weights
MANY = [(2560, 2048, 64), (2600, 2400, 208), (9000, 600, 64), (5000, 4100, 96), (300, 40000, 80), (8, 33000, 528), (16, 30000, 272),
        (20, 33000, 144), (17000, 64, 64), (1, 70000, 32), (130, 20000, 400), (33000, 40, 48), (1100, 5000, 2064), (700, 900, 131056)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,n,k", MANY)
def test_many_tiles(eng, t, n, k, dtype):
    check_gemm(eng, t, n, k, dtype, seed=t)
    if k < 10000:
        check_gate_up(eng, t, (n + 1) // 2, k, dtype, seed=t)


@pytest.mark.parametrize("t,ld", [(3, 1 << 31), (40, 1 << 27), (300, 1 << 24)])
def test_offsets_past_32_bits(eng, t, ld):
    """Rows of x and y that lie further apart than 32 bits reach."""
    n, k, x_ld = 200, 144, ld + 16
    (x, xs), (w, ws), (wu, us) = operands(t, n, k, 8, gated=True)
    far = torch.empty(t * x_ld, dtype=torch.int8, device="cuda").view(t, x_ld)
    far[:, :k] = x
    want, got = torch.empty(t, n, dtype=torch.bfloat16, device="cuda"), torch.empty(t * (ld + 8), dtype=torch.bfloat16, device="cuda").view(t, ld + 8)
    eng.gemm_i8(x, xs, w, ws, sx.DTYPE_BF16, want, t, n, k)
    eng.gemm_i8(far, xs, w, ws, sx.DTYPE_BF16, got, t, n, k, x_ld=x_ld, y_ld=ld + 8)
    eng.sync()
    assert torch.equal(got[:, :n], want)
    eng.gate_up_i8(x, xs, w, ws, wu, us, sx.DTYPE_BF16, want, t, n, k)
    eng.gate_up_i8(far, xs, w, ws, wu, us, sx.DTYPE_BF16, got, t, n, k, x_ld=x_ld, y_ld=ld + 8)
    eng.sync()
    assert torch.equal(got[:, :n], want)
    del got
    # weights
    far_w = far if t <= n else far[:n]
    rows = far_w.shape[0]
    far_w[:, :k] = w[:rows]
    want, got = torch.empty(t, rows, device="cuda"), torch.empty(t, rows, device="cuda")
    eng.gemm_i8(x, xs, w, ws, sx.DTYPE_F32, want, t, rows, k)
    eng.gemm_i8(x, xs, far_w, ws, sx.DTYPE_F32, got, t, rows, k, w_ld=x_ld)
    eng.sync()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,n,k", [(1, 100, 144), (6, 333, 1040), (40, 130, 272), (300, 200, 400), (700, 601, 144)])
def test_strides(eng, t, n, k, dtype):
    """Rows inside wider buffers, whose other bytes are not used and not written."""
    for extra in (0, 1, 2, 3, 8, 11):
        check_gemm(eng, t, n, k, dtype, x_ld=k + 48, w_ld=k + 16, y_ld=n + extra)
        check_gate_up(eng, t, n, k, dtype, x_ld=k + 16, w_ld=k + 112, y_ld=n + extra)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,n,k", [(300, 1, 64), (2600, 2401, 208), (5000, 2045, 96), (1100, 4999, 272), (4097, 1023, 1040)])
def test_rows_that_begin_aligned_and_end_anywhere(eng, t, n, k, dtype):
    """Rows 16 bytes apart or a multiple: nothing is written between a row's end and the next."""
    for extra in (0, 8):
        check_gemm(eng, t, n, k, dtype, seed=n, y_ld=(n + 7) // 8 * 8 + extra)
        check_gate_up(eng, t, n, k, dtype, seed=n, y_ld=(n + 7) // 8 * 8 + extra)


@pytest.mark.parametrize("off", [1, 2, 4, 6])
@pytest.mark.parametrize("t,n", [(3, 64), (64, 256), (300, 512)])
def test_unaligned_outputs(eng, t, n, off):
    check_gemm(eng, t, n, 256, torch.float32, y_off=off)
    check_gemm(eng, t, n, 256, torch.bfloat16, y_off=off)


@pytest.mark.parametrize("t", [1, 8, 24, 130])
def test_long_sums_and_every_code(eng, t):
    """Sums of up to 2^31 - 2^18 in size: codes of -128 alone, over the longest row."""
    k = 131056
    x = torch.full((t, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((40, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    w[2, ::2] = 127
    one = torch.ones(max(t, 40), device="cuda")
    y = torch.empty(t, 40, device="cuda")
    eng.gemm_i8(x, one, w, one, sx.DTYPE_F32, y, t, 40, k)
    eng.sync()
    assert torch.equal(y, sums(x, w).float())
    check_gemm(eng, t, 50, k, lo=-128)


def test_gate_range(eng):
    """Gates from far below (whose product is -0 or tiny) to far above."""
    for scale in (1e-30, 1e-3, 1.0, 30.0, 1e3, 1e6):
        check_gate_up(eng, 5, 129, 512, scale=scale)
        check_gate_up(eng, 50, 129, 512, scale=scale)


@pytest.mark.parametrize("t,n", [(4, 70), (40, 300), (400, 300)])
def test_rows_of_nan_infinity_and_zero(eng, t, n):
    """What a scale is reaches its own row or column and no other."""
    k = 320
    (x, xs), (w, ws), (wu, us) = operands(t, n, k, 3, gated=True)
    clean = torch.empty(t, n, device="cuda"), torch.empty(t, n, device="cuda")
    eng.gemm_i8(x, xs, w, ws, sx.DTYPE_F32, clean[0], t, n, k)
    eng.gate_up_i8(x, xs, w, ws, wu, us, sx.DTYPE_F32, clean[1], t, n, k)
    xs[0], xs[2], ws[5], ws[7], x[3] = math.nan, 0.0, math.nan, math.inf, 0
    got = torch.empty(t, n, device="cuda"), torch.empty(t, n, device="cuda")
    eng.gemm_i8(x, xs, w, ws, sx.DTYPE_F32, got[0], t, n, k)
    eng.gate_up_i8(x, xs, w, ws, wu, us, sx.DTYPE_F32, got[1], t, n, k)
    eng.sync()
    rows, cols = [i for i in range(t) if i not in (0, 2, 3)], [j for j in range(n) if j not in (5, 7)]
    for c, g in zip(clean, got):
        assert g[0].isnan().all() and g[:, 5].isnan().all()
        assert (g[2:4][:, cols] == 0).all()
        assert torch.equal(g[rows][:, cols], c[rows][:, cols])


# --------------------------------------------------------------------------------- quantisation
def codes_of(u):
    """Codes as the header defines them, in f32 (each operation rounded once)."""
    top = u.abs().amax(-1, keepdim=True)
    bad = ~(top < math.inf)
    top = torch.where((top >= 2.0 ** -100) & ~bad, top, 0.0)
    mul = torch.where(top > 0, torch.full_like(top, 127.0) / top, 0.0)  # (a number over a tensor is rounded twice)
    q = torch.where(bad, 0.0, torch.round(u * mul)).to(torch.int8)
    return q, torch.where(bad, math.nan, top.double() / 127)[:, 0]


def mean_tol(n):
    """Of 1 / sqrt(mean + eps): a sum of positive terms errs by as many half steps as it has levels, half of it
    in the root; then mean, root, quotient and what they are multiplied with."""
    return (n / 1024 + 64) * F


def check_quantize(eng, x, w=None, eps=1e-6, x_ld=0, q_ld=0):
    rows, n = x.shape
    xb, xv = wide(rows, n, x_ld or n, x.dtype)
    xv.copy_(x)
    qb, q = wide(rows, n, q_ld or n, torch.int8)
    scale = torch.full((rows + 1,), 9.0, device="cuda")
    eng.quantize_i8(TYPES[x.dtype], xb, qb, scale, rows, n, norm_w=w, eps=eps, x_ld=x_ld, q_ld=q_ld)
    eng.sync()
    u = x.float() if w is None else x.float() * w
    want_q, want = codes_of(u)
    if w is not None:
        sq = x.double().square().sum(-1)
        lost = ~(x.float().square().sum(-1) < math.inf)  # (none of the rows here is at the border)
        want = torch.where(lost, math.nan, want / (sq / n + eps).sqrt())
        want_q[lost] = 0
    assert torch.equal(q, want_q)
    assert (qb[:, n:] == JUNK).all() and scale[rows] == 9.0
    got = scale[:rows].double()
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    assert ((got - want).abs() <= want.abs() * (mean_tol(n) if w is not None else 2 * F))[ok].all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
@pytest.mark.parametrize("n", [16, 32, 240, 256, 272, 1040, 1536, 3840, 4112, 8192, 15360, 16400, 32784, 131056])
def test_quantize_sizes(eng, n, norm, dtype):
    g = gen(n)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    for rows in (1, 5, 130 if n < 20000 else 3):
        check_quantize(eng, (rand(rows, n) * rand(rows, 1).exp()).to(dtype), 1 + 0.2 * rand(n) if norm else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(297, 16), (299, 256), (1001, 272), (333, 512), (301, 784), (303, 1024), (305, 1040), (307, 2048), (309, 2064), (5001, 1552),
                                    (5003, 3840), (311, 8192), (313, 8208), (315, 16400)])
def test_many_rows(eng, rows, n, dtype):
    """Rows as warps and as CTAs, with every number of elements a thread."""
    g = gen(rows)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = (rand(rows, n) * rand(rows, 1).exp()).to(dtype)
    x[5], x[7, 3], x[9, n - 1], x[11] = 0, math.nan, math.inf, 1
    check_quantize(eng, x)
    check_quantize(eng, x, 1 + 0.2 * rand(n))
    x[[7, 9]] = 0
    for y_type in (torch.float32, torch.bfloat16, torch.int8, None):
        check_norm(eng, rand(rows, n), x, 1 + 0.2 * rand(n), 1 + 0.2 * rand(n), 0.5, y_type)


def test_quantize_many_rows_and_strides(eng):
    x = torch.randn(20011, 48, device="cuda", generator=gen(1))
    check_quantize(eng, x, torch.rand(48, device="cuda"), x_ld=56, q_ld=80)
    check_quantize(eng, x.bfloat16(), x_ld=56, q_ld=64)
    check_quantize(eng, torch.randn(77, 4096, device="cuda"), x_ld=4100, q_ld=4112)


@pytest.mark.parametrize("n", [64, 3840, 40000])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_quantize_special_rows(eng, n, norm):
    x = torch.randn(12, n, device="cuda", generator=gen(2))
    x[0] = 0
    x[1, n // 2] = math.nan
    x[2, n - 1] = math.inf
    x[3, 3] = -math.inf
    x[4] *= 1e-32  # under 2^-100
    x[5] *= 1e-29  # not under it
    x[6] *= 1e30   # squares pass f32
    x[7] = -1.0    # all codes -127
    x[8] = 0
    x[8, 5] = 3e-3
    x[9, 7] = 1e4  # one value dominates
    x[10] *= 1e-42  # subnormal
    x[11] = torch.arange(n, device="cuda") % 255 - 127.0  # halves and borders: codes are the values
    check_quantize(eng, x, torch.ones(n, device="cuda") if norm else None)
    if norm:
        w = torch.ones(n, device="cuda")
        w[4] = math.nan
        check_quantize(eng, x, w)


def test_quantize_eps_zero(eng):
    check_quantize(eng, torch.randn(3, 256, device="cuda"), torch.ones(256, device="cuda"), eps=0.0)


# ---------------------------------------------------------------------------------- seam of norms
def check_norm(eng, x, r, post, pre, scalar, y_type, eps=1e-6, lds=(0, 0, 0, 0), in_place=False):
    rows, n = x.shape
    xb, xv = wide(rows, n, lds[0] or n, torch.float32)
    rb, rv = wide(rows, n, lds[1] or n, r.dtype)
    xv.copy_(x)
    rv.copy_(r)
    ob, ov = (xb, xv) if in_place else wide(rows, n, lds[2] or n, torch.float32)
    yb, yv = wide(rows, n, lds[3] or n, y_type) if y_type is not None else (None, None)
    scale = torch.full((rows + 1,), 9.0, device="cuda") if y_type == torch.int8 else None
    eng.residual_norm(xb, TYPES[r.dtype], rb, ob, TYPES.get(y_type, 0), yb, rows, n, post_w=post, pre_w=pre, scalar=scalar, eps=eps,
                      y_scale=scale, x_ld=lds[0], r_ld=lds[1], x_out_ld=lds[0] if in_place else lds[2], y_ld=lds[3])
    eng.sync()
    assert (ob[:, n:] == JUNK).all() and (rv == r).logical_or(r.isnan()).all()
    rd, m = r.double(), mean_tol(n)
    h = rd if post is None else rd / (rd.square().sum(-1, keepdim=True) / n + eps).sqrt() * post.double()
    s = float(torch.tensor(scalar, dtype=torch.float32))
    want = (x.double() + h) * s
    e_x = (h.abs() * (m if post is not None else 0) + (x.double() + h).abs() * 2 * F) * abs(s)  # of x_out
    assert torch.equal(ov.isnan(), want.isnan())
    fine = ~want.isnan().any(-1)
    assert ((ov.double() - want).abs() <= e_x + 2.0 ** -140)[fine].all()
    if y_type is None:
        return
    assert (yb[:, n:] == JUNK).all()
    # y from the x_out that was written: its own roundings alone
    xo = ov.double()
    inv = 1 / (xo.square().sum(-1, keepdim=True) / n + eps).sqrt()
    if y_type == torch.int8:
        q, step = codes_of(ov * pre)
        assert torch.equal(yv, q) and scale[rows] == 9.0
        step = step * inv[:, 0]
        assert torch.equal(scale[:rows].isnan(), step.isnan())
        assert ((scale[:rows].double() - step).abs() <= step * m)[~step.isnan()].all()
        return
    y = xo * inv * pre.double()
    assert torch.equal(yv.isnan(), y.isnan())
    assert ((yv.double() - y).abs() <= y.abs() * (m + rounding(y_type)) + 2.0 ** -140)[~y.isnan()].all()


@pytest.mark.parametrize("r_type", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("y_type", [torch.float32, torch.bfloat16, torch.int8, None], ids=["yf32", "ybf16", "yi8", "none"])
@pytest.mark.parametrize("n", [16, 256, 272, 1536, 3840, 8208, 15360, 32784, 131056])
def test_norm_sizes(eng, n, y_type, r_type):
    g = gen(n)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    for rows in (1, 7, 150 if n < 20000 else 2):
        for post in (1 + 0.2 * rand(n), None):
            check_norm(eng, rand(rows, n) * rand(rows, 1).exp(), (3 * rand(rows, n)).to(r_type), post, 1 + 0.2 * rand(n), 0.875, y_type)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n", [64, 3840, 40000])
def test_norm_strides_and_in_place(eng, n, in_place):
    g = gen(n)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    for y_type, r_type in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.int8, torch.bfloat16), (None, torch.float32)):
        check_norm(eng, rand(9, n), rand(9, n).to(r_type), rand(n), rand(n), -1.5, y_type, lds=(n + 4, n + 8, n + 12, n + 16), in_place=in_place)


@pytest.mark.parametrize("n", [64, 3840, 40000])
@pytest.mark.parametrize("y_type", [torch.float32, torch.int8], ids=["yf32", "yi8"])
def test_norm_special_rows(eng, n, y_type):
    g = gen(4)
    x, r = (torch.randn(7, n, device="cuda", generator=g) for _ in range(2))
    x[0] = 0
    r[0] = 0
    r[1] = 0
    x[2, 3] = math.nan
    r[3, n - 1] = math.nan
    x[4] *= 1e-34
    r[4] = 0
    x[5, n // 2] = 1e5
    check_norm(eng, x, r, torch.ones(n, device="cuda"), torch.ones(n, device="cuda"), 1.0, y_type)


@pytest.mark.parametrize("rows,ld", [(3, 1 << 31), (700, 1 << 23)])
def test_rows_past_32_bits(eng, rows, ld):
    n = 96
    g = gen(rows)
    x = torch.randn(rows, n, device="cuda", generator=g).bfloat16()
    w = 1 + 0.1 * torch.randn(n, device="cuda", generator=g)
    far = torch.empty(rows * (ld + 8), dtype=torch.bfloat16, device="cuda").view(rows, ld + 8)
    far[:, :n] = x
    q, qf = torch.empty(rows, n, dtype=torch.int8, device="cuda"), torch.empty(rows * (ld + 16), dtype=torch.int8, device="cuda").view(rows, ld + 16)
    s, sf = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    eng.quantize_i8(sx.DTYPE_BF16, x, q, s, rows, n, norm_w=w)
    eng.quantize_i8(sx.DTYPE_BF16, far, qf, sf, rows, n, norm_w=w, x_ld=ld + 8, q_ld=ld + 16)
    eng.sync()
    assert torch.equal(qf[:, :n], q) and torch.equal(s, sf)
    xr = torch.randn(rows, n, device="cuda", generator=g)
    out, y, yf = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, dtype=torch.bfloat16, device="cuda"), far
    eng.residual_norm(xr, sx.DTYPE_BF16, x, out, sx.DTYPE_BF16, y, rows, n, post_w=w, pre_w=w)
    first = out.clone()
    eng.residual_norm(xr, sx.DTYPE_BF16, x, out, sx.DTYPE_BF16, yf, rows, n, post_w=w, pre_w=w, y_ld=ld + 8)
    eng.sync()
    assert torch.equal(yf[:, :n], y) and torch.equal(out, first)


# ---------------------------------------------------------------------- streams, graphs, a whole block
def test_no_rows(eng):
    one = torch.zeros(64, device="cuda")
    codes = torch.zeros(64, dtype=torch.int8, device="cuda")
    eng.quantize_i8(sx.DTYPE_F32, one, codes, one, 0, 64)
    eng.residual_norm(one, sx.DTYPE_F32, one, one, sx.DTYPE_F32, None, 0, 64)
    eng.gemm_i8(codes, one, codes, one, sx.DTYPE_F32, one, 0, 1, 64)
    eng.gate_up_i8(codes, one, codes, one, codes, one, sx.DTYPE_F32, one, 0, 1, 64)
    eng.sync()
    assert (one == 0).all() and (codes == 0).all()


class Block:
    """A feed-forward block: quantised weights, and its buffers for t tokens."""

    def __init__(self, eng, t, hidden, inter, seed):
        g = gen(seed)
        self.eng, self.t, self.hidden, self.inter = eng, t, hidden, inter
        self.x = torch.randn(t, hidden, device="cuda", generator=g)
        self.attn = torch.randn(t, hidden, device="cuda", generator=g)
        self.gain = [1 + 0.1 * torch.randn(hidden, device="cuda", generator=g) for _ in range(4)]
        self.w = {}
        for name, n, k in (("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter)):
            full = (torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k)).bfloat16()
            q, s = torch.empty(n, k, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
            eng.quantize_i8(sx.DTYPE_BF16, full, q, s, n, k)
            self.w[name] = q, s, full
        empty = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
        self.q, self.qs = empty(t, hidden, dtype=torch.int8), empty(t)
        self.h, self.hq, self.hs = empty(t, inter, dtype=torch.bfloat16), empty(t, inter, dtype=torch.int8), empty(t)
        self.out, self.x1, self.x2, self.y = empty(t, hidden), empty(t, hidden), empty(t, hidden), empty(t, hidden)

    def run(self):
        e, t, hidden, inter = self.eng, self.t, self.hidden, self.inter
        e.residual_norm(self.x, sx.DTYPE_F32, self.attn, self.x1, sx.DTYPE_I8, self.q, t, hidden, post_w=self.gain[0], pre_w=self.gain[1], y_scale=self.qs)
        e.gate_up_i8(self.q, self.qs, *self.w["gate"][:2], *self.w["up"][:2], sx.DTYPE_BF16, self.h, t, inter, hidden)
        e.quantize_i8(sx.DTYPE_BF16, self.h, self.hq, self.hs, t, inter)
        e.gemm_i8(self.hq, self.hs, *self.w["down"][:2], sx.DTYPE_F32, self.out, t, hidden, inter)
        e.residual_norm(self.x1, sx.DTYPE_F32, self.out, self.x2, sx.DTYPE_F32, self.y, t, hidden, post_w=self.gain[2], pre_w=self.gain[3], scalar=0.5)

    def want(self):
        """The block with the same codes, in 64 bits from each call's own inputs on."""
        rms = lambda v: v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
        deq = lambda q, s: q.double() * s.double()[:, None]  # noqa: E731
        x1 = self.x.double() + rms(self.attn.double()) * self.gain[0].double()
        a = deq(self.q, self.qs)
        h = gelu(a @ deq(*self.w["gate"][:2]).T) * (a @ deq(*self.w["up"][:2]).T)
        b = deq(self.hq, self.hs)
        out = b @ deq(*self.w["down"][:2]).T
        x2 = (x1 + rms(out) * self.gain[2].double()) * 0.5
        return x1, rms(x1) * self.gain[1].double(), a, h, b, out, rms(x2) * self.gain[3].double()


def near(got, want, tol):
    err, size = float((got.double() - want).norm()), float(want.norm())
    assert err <= tol * size, (err / size, tol)


@pytest.mark.parametrize("t", [1, 8, 40, 700])
def test_a_block(eng, t):
    b = Block(eng, t, 1536, 6144, t)
    b.run()
    eng.sync()
    x1, y1, a, h, hq, out, y = b.want()
    near(b.x1, x1, 1e-6)
    near(b.h, h, HALF_BF16)
    near(b.out, out, 1e-6)
    near(b.y, y, 1e-5)
    # a code is off by at most half a step, a step is the row's largest value / 127
    assert ((a - y1).abs() <= y1.abs().amax(-1, keepdim=True) / 127 * 0.501).all()
    assert ((hq - b.h.double()).abs() <= b.h.double().abs().amax(-1, keepdim=True) / 127 * 0.501).all()
    # and with the weights as they were before, the block is what 8 bits leave of it: each of the six
    # operands' codes rounds by 0.29 steps, a step about 1/30 of the operand's size: 1 % each
    full = {k: v[2].double() for k, v in b.w.items()}
    g = gelu(y1 @ full["gate"].T) * (y1 @ full["up"].T)
    near(b.out, g @ full["down"].T, 0.05)


@pytest.mark.parametrize("t", [1, 16, 50, 300])
def test_captured_and_replayed(eng, t):
    """A captured block replays on new inputs; two captures replayed on streams of their own do not meet."""
    blocks = [Block(eng, t, 512, 1040, s) for s in (1, 2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in blocks]
    try:
        for b, s in zip(blocks, streams):
            eng.set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                b.run()
                s.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    b.run()
                graphs.append(g)
    finally:
        eng.set_stream(sx.STREAM_LEGACY)
    torch.cuda.synchronize()
    for b in blocks:
        b.x.normal_(generator=gen(7 + t))
        b.attn.normal_(generator=gen(8 + t))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    replayed = [(b.x1.clone(), b.h.clone(), b.out.clone(), b.y.clone()) for b in blocks]
    for b, r in zip(blocks, replayed):
        b.run()
        eng.sync()
        for x, y in zip((b.x1, b.h, b.out, b.y), r):
            assert torch.equal(x, y)


def test_calls_on_two_engines_at_once():
    """Two engines' calls run beside one another: no memory is shared."""
    engines = [sx.Engine(0) for _ in range(2)]
    try:
        blocks = [Block(e, t, 1024, 2048, t) for e, t in zip(engines, (9, 130))]
        for e in engines:
            e.sync()
        torch.cuda.synchronize()
        alone = []
        for e, b in zip(engines, blocks):
            b.run()
            e.sync()
            alone.append((b.h.clone(), b.out.clone(), b.y.clone()))
        for b in blocks:
            b.h.zero_(), b.out.zero_(), b.y.zero_()
        torch.cuda.synchronize()
        for _ in range(30):
            for b in blocks:
                b.run()
        for e in engines:
            e.sync()
        for b, want in zip(blocks, alone):
            for x, y in zip((b.h, b.out, b.y), want):
                assert torch.equal(x, y)
    finally:
        for e in engines:
            e.close()


def test_repeats_bit_for_bit(eng):
    for t in (3, 60, 600):
        (x, xs), (w, ws) = operands(t, 900, 1200, t)
        first = torch.empty(t, 900, device="cuda")
        eng.gemm_i8(x, xs, w, ws, sx.DTYPE_F32, first, t, 900, 1200)
        for _ in range(5):
            y = torch.empty(t, 900, device="cuda")
            eng.gemm_i8(x, xs, w, ws, sx.DTYPE_F32, y, t, 900, 1200)
            eng.sync()
            assert torch.equal(y, first)


def test_rows_do_not_depend_on_their_batch(eng):
    """A row of a product is the same alone and among others: sums are whole numbers."""
    (x, xs), (w, ws), (wu, us) = operands(400, 650, 720, 5, gated=True)
    y, z = torch.empty(400, 650, device="cuda"), torch.empty(400, 650, device="cuda")
    eng.gemm_i8(x, xs, w, ws, sx.DTYPE_F32, y, 400, 650, 720)
    eng.gate_up_i8(x, xs, w, ws, wu, us, sx.DTYPE_F32, z, 400, 650, 720)
    for t in (1, 8, 17, 130):
        a, b = torch.empty(t, 650, device="cuda"), torch.empty(t, 650, device="cuda")
        eng.gemm_i8(x, xs, w, ws, sx.DTYPE_F32, a, t, 650, 720)
        eng.gate_up_i8(x, xs, w, ws, wu, us, sx.DTYPE_F32, b, t, 650, 720)
        eng.sync()
        assert torch.equal(a, y[:t]) and torch.equal(b, z[:t])


# rows as CTAs with every number of elements a thread, and as warps
LAYOUTS = [(9, 64), (9, 3840), (9, 8208), (9, 15360), (9, 40000), (305, 64), (305, 512), (305, 1024), (305, 2048), (305, 8192), (305, 8208), (305, 16400)]


def seam(eng, x, r, post, pre, y_type, scalar=0.875, eps=1e-6):
    rows, n = x.shape
    out, scale = torch.empty(rows, n, device="cuda"), torch.empty(rows, device="cuda") if y_type == torch.int8 else None
    y = None if y_type is None else torch.full((rows, n), JUNK, dtype=y_type, device="cuda")
    eng.residual_norm(x, TYPES[r.dtype], r, out, TYPES.get(y_type, 0), y, rows, n, post_w=post, pre_w=pre, scalar=scalar, eps=eps, y_scale=scale)
    eng.sync()
    return out, y, scale


def only_nan(y, scale):
    """Rows of no value: floats that are NaN, or codes 0 with the scale NaN."""
    return y.isnan().all() if scale is None else (y == 0).all() and scale.isnan().all()


@pytest.mark.parametrize("r_type", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,n", LAYOUTS)
def test_norm_of_squares_past_f32(eng, rows, n, r_type):
    """A norm of squares whose sum f32 does not hold is NaN, whatever it is written as, and no other row's."""
    g = gen(n)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    clean = rand(rows, n), rand(rows, n).to(r_type)
    clean[1][rows - 1] *= 1e16  # (not past it)
    clean[0][rows - 2] *= 1e16
    post, pre = 1 + 0.2 * rand(n), 1 + 0.2 * rand(n)
    x, r = (v.clone() for v in clean)
    r[0] *= 1e30
    r[1, n // 3] = 1e20
    r[2, 5] = math.inf
    x[3] *= 1e30
    x[4, n - 1] = -1e25
    x[5, 7] = -math.inf
    for y_type in (torch.float32, torch.bfloat16, torch.int8, None):
        for w in (post, None):
            check_norm(eng, *clean, w, pre, 0.875, y_type)
            want, want_y, want_scale = seam(eng, *clean, w, pre, y_type)
            out, y, scale = seam(eng, x, r, w, pre, y_type)
            assert torch.equal(out[6:], want[6:])
            if w is not None:
                assert out[:3].isnan().all()
                assert torch.equal(out[5].isinf(), x[5].isinf()) and torch.equal(out[5, 8:], want[5, 8:])
            else:
                assert torch.equal(out[:6], (x[:6] + r[:6].float()) * 0.875)
            assert ((out[3:5] - x[3:5] * 0.875).abs() <= x[3:5].abs() * 2 * F + (want[3:5] - clean[0][3:5] * 0.875).abs() + 1e-6).all()
            if y_type is None:
                continue
            assert torch.equal(y[6:], want_y[6:]) and only_nan(y[:6], None if scale is None else scale[:6])
            if scale is not None:
                assert torch.equal(scale[6:], want_scale[6:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,n", LAYOUTS)
def test_squares_below_f32(eng, rows, n, dtype):
    """Rows whose squares are nothing in f32: any eps of a normal number is enough for them; with less they are NaN (codes,
    where values are below 2^-100: zeros)."""
    g = gen(n)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    post, pre, zeros, ones = 1 + 0.2 * rand(n), 1 + 0.2 * rand(n), torch.zeros(rows, n, device="cuda"), torch.ones(rows, n, device="cuda")
    x = rand(rows, n)
    x[:3] *= torch.tensor([1e-15, 1e-17, 1e-18], device="cuda")[:, None]
    x[rows - 1] *= 1e-18
    for eps in (0.0, 1e-40):
        check_quantize(eng, x.to(dtype), pre, eps=eps)
        for y_type in (torch.float32, torch.bfloat16, torch.int8, None):
            check_norm(eng, x, zeros.to(dtype), None, pre, 0.5, y_type, eps=eps)
            check_norm(eng, zeros, x.to(dtype), post, pre, 0.5, y_type, eps=eps)
    small = x.clone()
    small[3:7] = rand(4, n) * torch.tensor([1e-20, 1e-25, 1e-29, 1e-36], device="cuda")[:, None]
    small[7] = 0
    for eps in (2.0 ** -126, 1e-30):
        check_quantize(eng, small.to(dtype), pre, eps=eps)
        for y_type in (torch.float32, torch.bfloat16, torch.int8, None):
            check_norm(eng, small, zeros.to(dtype), None, pre, 0.5, y_type, eps=eps)
            check_norm(eng, ones, small.to(dtype), post, pre, 0.5, y_type, eps=eps)
    for eps in (0.0, 1e-41):
        q, scale = torch.full((rows, n), JUNK, dtype=torch.int8, device="cuda"), torch.full((rows,), 9.0, device="cuda")
        eng.quantize_i8(TYPES[dtype], small.to(dtype), q, scale, rows, n, norm_w=pre, eps=eps)
        eng.sync()
        assert scale[3:6].isnan().all() and (q[6:8] == 0).all() and (scale[6:8] == 0).all()
        assert scale[:3].isfinite().all() and scale[8:].isfinite().all() and (q[8:].abs().amax(-1) == 127).all()
        for y_type in (torch.float32, torch.bfloat16, torch.int8):
            out, y, scale = seam(eng, small, zeros.to(dtype), None, pre, y_type, eps=eps)
            assert torch.equal(out, small * 0.875)
            if scale is None:
                assert only_nan(y[3:8], None) and y[:3].isfinite().all() and y[8:].isfinite().all()
            else:
                assert scale[3:6].isnan().all() and (y[6:8] == 0).all() and (scale[6:8] == 0).all()
                assert scale[:3].isfinite().all() and scale[8:].isfinite().all()
            out = seam(eng, ones, small.to(dtype), post, pre, y_type, eps=eps)[0]
            assert out[3:8].isnan().all() and out[:3].isfinite().all() and out[8:].isfinite().all()


@pytest.mark.parametrize("dtype,t", [(torch.float32, 4200), (torch.bfloat16, 8400)], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,y_ld", [(8200, 8200), (8201, 8208)])
def test_results_that_l2_does_not_hold(eng, t, n, y_ld, dtype):
    """More than 128 MB of y: its lines leave L2 first; whole rows, and rows that end inside 16 bytes."""
    check_gemm(eng, t, n, 80, dtype, seed=n, y_ld=y_ld)
    check_gate_up(eng, t, n, 80, dtype, seed=n, y_ld=y_ld)


@pytest.mark.parametrize("t,n", [(4, 70), (16, 70), (40, 300), (400, 300)])
def test_infinite_scales_of_columns(eng, t, n):
    """An infinite scale makes its column infinite, by the sums' signs; NaN where there is 0 to multiply."""
    k = 320
    (x, xs), (w, ws), (wu, us) = operands(t, n, k, 3, gated=True)
    x[1] = 0
    xs[2] = 0
    ws[7], us[9] = math.inf, math.inf
    y, z = torch.empty(t, n, device="cuda"), torch.empty(t, n, device="cuda")
    eng.gemm_i8(x, xs, w, ws, sx.DTYPE_F32, y, t, n, k)
    eng.gate_up_i8(x, xs, w, ws, wu, us, sx.DTYPE_F32, z, t, n, k)
    eng.sync()
    s, su = sums(x, w), sums(x, wu)
    inf = torch.tensor(math.inf, device="cuda", dtype=torch.float64)
    sign = torch.where(xs > 0, s[:, 7].sign(), 0.0)
    assert torch.equal(y[:, 7].double().nan_to_num(0.0, math.inf, -math.inf), torch.where(sign == 0, 0.0, sign * inf))
    assert torch.equal(y[:, 7].isnan(), sign == 0)
    # an infinite gate opens or, below, is infinity times nothing; an infinite `up` has the gate's sign times its own
    up = torch.where(xs > 0, su[:, 7].sign(), 0.0)
    lost = (sign <= 0) | (up == 0)
    assert torch.equal(z[:, 7].isnan(), lost) and torch.equal(z[:, 7].double()[~lost], (up * inf)[~lost])
    both = torch.where(xs > 0, s[:, 9].sign() * su[:, 9].sign(), 0.0)
    assert torch.equal(z[:, 9].isnan(), both == 0) and torch.equal(z[:, 9].double()[both != 0], (both * inf)[both != 0])
    cols = [j for j in range(n) if j not in (7, 9)]
    assert y[:, cols].isfinite().all() and z[:, cols].isfinite().all() and y[:, 9].isfinite().all()


@pytest.mark.parametrize("t", [1, 16, 50, 300])
def test_captures_with_inputs_of_their_own(eng, t):
    """Two captures of blocks whose weights are the same, replayed at once: each has its own input's results."""
    blocks = [Block(eng, t, 512, 1040, 1) for _ in range(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in blocks]
    try:
        for b, s in zip(blocks, streams):
            eng.set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                b.run()
                s.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    b.run()
                graphs.append(g)
    finally:
        eng.set_stream(sx.STREAM_LEGACY)
    torch.cuda.synchronize()
    for i, b in enumerate(blocks):
        b.x.normal_(generator=gen(100 * i + t))
        b.attn.normal_(generator=gen(100 * i + t + 50))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    replayed = [(b.x1.clone(), b.h.clone(), b.out.clone(), b.y.clone()) for b in blocks]
    for x, y in zip(*replayed):
        assert not torch.equal(x, y)
    for b, r in zip(blocks, replayed):
        b.run()
        eng.sync()
        for x, y in zip((b.x1, b.h, b.out, b.y), r):
            assert torch.equal(x, y)


@pytest.mark.parametrize("t", [1, 9, 40, 300])
def test_gates_that_are_nothing(eng, t):
    """Around g = -10 the gate leaves f32's normal numbers: off by at most 2^-126 |g u| there, and never by more below."""
    n, k = 2048, 16
    x = torch.ones(t, k, dtype=torch.int8, device="cuda")
    wg, wu = -torch.ones(n, k, dtype=torch.int8, device="cuda"), torch.ones(n, k, dtype=torch.int8, device="cuda")
    xs = torch.ones(t, device="cuda")
    gs = torch.linspace(9.0, 11.0, n, device="cuda") / 16
    us = torch.full((n,), 2.0 ** 90 / 16, device="cuda")
    y = torch.empty(t, n, device="cuda")
    eng.gate_up_i8(x, xs, wg, gs, wu, us, sx.DTYPE_F32, y, t, n, k)
    eng.sync()
    g, u = -16 * gs.double(), 2.0 ** 90
    z = (0.7978845608 * (g + 0.044715 * g ** 3)).abs()
    want = gelu(g) * u
    # (as in check_gate_up, g and u exact here but for g's own rounding; the reciprocal's 0 takes 2^-126 |g u|)
    tol = want.abs() * (18 + 33 * z) * F + (g * u).abs() * 2.0 ** -126
    assert ((y.double() - want).abs() <= tol).all()
    assert (y[:, g < -10.01] == 0).all() and (y[:, g > -9.99] != 0).all()
