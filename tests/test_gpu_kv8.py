"""The paged 8-bit KV cache: append with rotation and quantisation, and attention over it, against
restatements in 64 bits that follow the layout's byte formulas."""
import ctypes
import math

import pytest

import sx

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": (sx.DTYPE_F32, torch.float32), "bf16": (sx.DTYPE_BF16, torch.bfloat16)}


@pytest.fixture(scope="module")
def eng():
    e = sx.Engine(0)
    e.set_stream(sx.STREAM_LEGACY)
    yield e
    e.close()


# Attention of more than 16 packed rows has two forms, and the table's width decides with the rows.
BOTH_FORMS = """drafts prompts window one_long_prompt strided_rows magnitudes scales_far_apart nan_in_masked_places
nan_value_only large_values_without_weight scales_at_random chunks_beside_single_tokens rows_outside_sequences_stay bad_page_masks_and_reports prompts_repeat_bit_for_bit
repeats_bit_for_bit_on_any_stream_and_in_a_graph scale_zero_and_negative""".split()


def pytest_generate_tests(metafunc):
    if metafunc.function.__name__.removeprefix("test_attn_") in BOTH_FORMS:
        metafunc.parametrize("table_width", [0, 100000], indirect=True, ids=["narrow", "wide"])


@pytest.fixture(autouse=True)
def table_width(request):
    Cache.spare_columns = getattr(request, "param", 0)
    yield
    Cache.spare_columns = 0


# ------------------------------------------------------------------------- the cache in 64 bits
def codes():
    out = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(math.nan if c & 127 == 127 else -v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def places(d):
    t, e = torch.arange(16)[:, None], torch.arange(d)[None]
    k = 512 * (e // 32) + 16 * (4 * (t % 8) + e % 32 // 8) + 8 * (t // 8) + e % 8
    v = 512 * (e // 32) + 16 * (4 * (e % 32 // 4) + t % 8 // 2) + 4 * (e % 4) + t % 2 + 2 * (t // 8)
    return k.reshape(-1).cuda(), v.reshape(-1).cuda()


class Cache:
    """A pool with every page in use: sequences' pages in shuffled order, the rest of the table bad."""

    spare_columns = 0  # of the table: its width says how much there may be to do

    def __init__(self, lens, page, hkv, d, seed, first=None, spare=2, fill=1.0):
        g = torch.Generator().manual_seed(seed)
        self.page, self.hkv, self.d, self.lens = page, hkv, d, lens
        first = first or [0] * len(lens)
        need = [max(0, -(-n // page) - f) for n, f in zip(lens, first)]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        width = max([1] + [-(-n // page) for n in lens]) + 1 + Cache.spare_columns
        rows = []
        for n, f in zip(need, first):
            rows.append([-1] * f + [order.pop() for _ in range(n)] + [-1] * (width - n - f))
        self.table = torch.tensor(rows, dtype=torch.int32).reshape(len(lens), width).cuda()
        nb = page // 16
        x = torch.randn(self.pages, hkv, nb, 2, 16 * d, generator=g) * fill
        self.data = x.mul(64).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).cuda()
        self.scale = torch.exp2(torch.randint(-8, -4, (self.pages, hkv, nb, 2), generator=g).float()).cuda()

    def kv8(self):
        return sx.KV8(self.data, self.scale, self.table, self.page, self.hkv, self.d)

    def values(self, b, n=None, data=None, scale=None):
        """K and V of sequence b's first n tokens, f64 [n, hkv, d]."""
        n = self.lens[b] if n is None else n
        data, scale = self.data if data is None else data, self.scale if scale is None else scale
        nb = -(-n // 16)
        ids = self.table[b].long().repeat_interleave(self.page // 16)[:nb].clamp(min=0)
        slot = torch.arange(nb, device="cuda") % (self.page // 16)
        rec, sc = data[ids, :, slot], scale[ids, :, slot].double()  # nb, hkv, 2, 16 d
        out = []
        for w, p in enumerate(places(self.d)):
            val = codes()[rec[:, :, w][..., p].long()].reshape(nb, self.hkv, 16, self.d) * sc[:, :, w, None, None]
            out.append(val.transpose(1, 2).reshape(nb * 16, self.hkv, self.d)[:n])
        return out


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rows_of(news, lens):
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    return ints(start), ints(lens), start


# ------------------------------------------------------------------------------------- attention
def want_attn(cache, q, news, lens, hq, scale, window):
    out, start = torch.zeros(q.shape[0], hq, cache.d, dtype=torch.float64, device="cuda"), 0
    mass = torch.zeros_like(out)
    dz = 0.0
    for b, (n, total) in enumerate(zip(news, lens)):
        if n:
            k, v = cache.values(b, total)
            rep = hq // cache.hkv
            pos, key = torch.arange(total - n, total)[:, None].cuda(), torch.arange(total)[None].cuda()
            hide = key > pos
            if window:
                hide |= key <= pos - window
            for h in range(hq):
                x = q[start:start + n, h * cache.d:(h + 1) * cache.d].double()
                kk, vv = k[:, h // rep], v[:, h // rep]
                z = (x @ kk.T * scale).masked_fill(hide, -math.inf)
                p = torch.softmax(z, -1)
                # masked values do not count, whatever they are
                p = torch.where(hide, 0.0, p)
                vv = torch.where(hide.all(0)[:, None], 0.0, vv)
                out[start:start + n, h] = p @ vv
                mass[start:start + n, h] = p @ vv.abs()
                dz = max(dz, float((x.abs() @ kk.abs().T * abs(scale)).masked_fill(hide, 0).nan_to_num(0).max()))
        start += n
    return out.reshape(q.shape[0], -1), mass.reshape(q.shape[0], -1), dz


def tolerance(dtype, want, mass, dz, d):
    """A score errs by dz (the largest sum of |q||k| scale) times the operands' rounding -- 2^-22
    where q is split in two f16 terms, none for bf16 q, which f16 holds -- and the f32 sum's,
    which grows like sqrt(d) 2^-24; 8 times that covers the spread.  p errs by as much relatively,
    plus its own rounding (2^-22 split, 2^-11 as one f16) and the sums' 2^-20; the output's own
    rounding comes last."""
    f32 = dtype == "f32"
    score = dz * ((2.0 ** -22 if f32 else 0) + 8 * math.sqrt(d) * 2.0 ** -24)
    rel = 2 * score + (2.0 ** -22 if f32 else 2.0 ** -11) + 2.0 ** -20
    return mass * rel + want.abs() * (2.0 ** -23 if f32 else 2.0 ** -8) + 1e-30


def check_attn(eng, dtype, hq, hkv, d, page, news, lens, window=0, seed=1, pad=0, cache=None, qmul=1.0, fill=1.0):
    code, dt = DT[dtype]
    first = [max(0, n - k - window + 1) // page if window else 0 for n, k in zip(lens, news)]
    cache = cache or Cache(lens, page, hkv, d, seed, first=first, fill=fill)
    t = sum(news)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(t, hq * d + pad, device="cuda", generator=g) * qmul).to(dt)
    out = torch.full((t, hq * d + pad), 7.0, dtype=dt, device="cuda")
    start, kv_len, _ = rows_of(news, lens)
    scale = d ** -0.5
    eng.kv8_attn(cache.kv8(), code, q, out, start, kv_len, t, hq, scale, window=window, q_ld=hq * d + pad, out_ld=hq * d + pad)
    eng.sync()
    if pad:
        assert (out[:, hq * d:] == 7.0).all()
    got = out[:, :hq * d].double()
    want, mass, dz = want_attn(cache, q, news, lens, hq, scale, window)
    tol = tolerance(dtype, want, mass, dz, d)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol).max()), bad.nonzero()[:3].tolist())
    return cache, q, out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (8, 1), (6, 2), (16, 8)])
def test_attn_one_row(eng, dtype, d, hq, hkv):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 200, 513]
    check_attn(eng, dtype, hq, hkv, d, 64, [1] * len(lens), lens, seed=d + hq)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,hq,hkv,page", [(64, 8, 1, 16), (128, 5, 1, 48), (256, 16, 8, 64), (256, 8, 1, 128), (512, 4, 2, 32), (128, 64, 1, 16)])
@pytest.mark.parametrize("new", [2, 5, 8])
def test_attn_drafts(eng, dtype, d, hq, hkv, page, new):
    lens = [new, new + 1, 40, 100, 333]
    check_attn(eng, dtype, hq, hkv, d, page, [new] * len(lens), lens, seed=new)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 4), (128, 16, 8), (128, 3, 1), (256, 8, 1), (512, 2, 1)])
def test_attn_prompts(eng, dtype, d, hq, hkv):
    news, lens = [1, 130, 0, 257, 64], [90, 130, 0, 300, 1000]
    check_attn(eng, dtype, hq, hkv, d, 32, news, lens)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 5000])
@pytest.mark.parametrize("new", [1, 3, 70])
def test_attn_window(eng, dtype, window, new):
    lens = [new, 33 + new, 257, 1000, 1024]
    check_attn(eng, dtype, 8, 4, 128, 32, [new] * len(lens), lens, window=window)


@pytest.mark.parametrize("dtype,d", [("f32", 128), ("bf16", 256)])
def test_attn_long_and_ragged(eng, dtype, d):
    check_attn(eng, dtype, 8, 4, d, 64, [1, 1, 1, 2], [40001, 3, 12345, 777], seed=9)


@pytest.mark.parametrize("dtype,d,lens", [("f32", 64, [150000]), ("bf16", 64, [700, 90001, 0, 40000]), ("f32", 256, [60001, 9])])
def test_attn_many_parts_of_a_problem(eng, dtype, d, lens):
    """Long enough that over 32 CTAs share a problem, which merge in two levels."""
    news = [min(n, 1) for n in lens]
    for _ in range(3):  # the arrival counters are left at 0
        check_attn(eng, dtype, 4, 1, d, 64, news, lens, seed=12)


@pytest.mark.parametrize("lens", [[640], [250] * 40, [700, 1, 0, 33] * 30, [500] * 200])
def test_attn_problems_cut_and_uncut(eng, lens):
    check_attn(eng, "bf16", 8, 2, 128, 32, [min(n, 1) for n in lens], lens, seed=13)


@pytest.mark.parametrize("dtype,d,hq", [("f32", 64, 8), ("bf16", 128, 16)])
def test_attn_one_long_prompt(eng, dtype, d, hq):
    check_attn(eng, dtype, hq, 2, d, 64, [700, 1], [2100, 5], seed=10)


@pytest.mark.parametrize("dtype,d,hkv", [("f32", 64, 4), ("bf16", 64, 4), ("f32", 128, 2), ("bf16", 256, 2)])
def test_attn_many_tiles_of_a_problem_on_one_cta(eng, dtype, d, hkv):
    """More problems than CTAs, of 44 tiles of 64 keys each: a CTA's tables of a problem's records wrap."""
    n = 75 if d < 256 else 80
    lens = [2816 - (7 * i) % 50 for i in range(n)]
    check_attn(eng, dtype, 8 * hkv, hkv, d, 64, [16] * n, lens, seed=14)


@pytest.mark.parametrize("dtype,d,total", [("f32", 64, 60001), ("bf16", 128, 100000), ("bf16", 256, 40011), ("f32", 256, 60000)])
@pytest.mark.parametrize("new", [5, 16])
def test_attn_many_parts_of_packed_rows(eng, dtype, d, total, new):
    """One session's drafts on a long context: over a hundred CTAs hold parts of one problem."""
    for _ in range(2):
        check_attn(eng, dtype, 8, 1, d, 64, [new], [total], seed=15)


@pytest.mark.parametrize("dtype,d", [("f32", 64), ("bf16", 128), ("bf16", 256), ("f32", 512)])
@pytest.mark.parametrize("chunk", [60, 700])
def test_attn_chunks_beside_single_tokens(eng, dtype, d, chunk):
    """A batch that decodes most of its sequences and takes a prompt's chunk in two: one call for all."""
    news = [1, 1, chunk, 0, 1, 1, 5, 1, chunk // 2] + [1] * 20
    lens = [900, 1, chunk + 1500, 40, 17, 3000, 64, 333, chunk // 2] + [100 + 37 * i for i in range(20)]
    check_attn(eng, dtype, 8, 2, d, 32, news, lens, seed=16)
    check_attn(eng, dtype, 8, 2, d, 32, news, lens, seed=16, window=100)


@pytest.mark.parametrize("dtype,d", [("f32", 64), ("bf16", 128), ("bf16", 256)])
def test_attn_scales_at_random_over_many_tiles(eng, dtype, d):
    lens, new = [6000, 3000], 40
    cache = Cache(lens, 32, 1, d, 22)
    g = torch.Generator(device="cuda").manual_seed(10)
    far = torch.rand(cache.scale.shape[:-1], device="cuda", generator=g) < 0.05
    up = torch.randint(-30, 31, far.shape, device="cuda", generator=g)
    cache.scale[..., 1] *= torch.exp2(torch.where(far, up, 0).float())
    check_attn(eng, dtype, 8, 1, d, 32, [new, new], lens, cache=cache)


def test_attn_many_sequences(eng):
    lens = [(i * 37) % 200 for i in range(300)]
    check_attn(eng, "bf16", 4, 2, 64, 16, [min(n, 1) for n in lens], lens, seed=11)


def test_attn_strided_rows(eng):
    check_attn(eng, "f32", 4, 2, 64, 16, [1, 3, 40], [20, 30, 90], pad=12)
    check_attn(eng, "bf16", 4, 2, 64, 16, [1, 3, 40], [20, 30, 90], pad=24)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("qmul", [1e-20, 30.0, 1e15])
def test_attn_magnitudes(eng, dtype, qmul):
    """q far outside f16's range, scores that make the softmax one-hot or flat."""
    cache = Cache([300, 40], 32, 2, 128, 3)
    if qmul > 1e10:
        cache.scale[..., 0] = torch.exp2(torch.log2(cache.scale[..., 0]) - 48)
    check_attn(eng, dtype, 4, 2, 128, 32, [1, 20], [300, 40], cache=cache, qmul=qmul)


def test_attn_scales_far_apart(eng):
    """V records whose scales differ by 2^40: large values dominate, small ones keep their part."""
    cache = Cache([256, 64], 16, 1, 64, 4)
    cache.scale[::2, :, :, 1] *= 2.0 ** -40
    check_attn(eng, "f32", 2, 1, 64, 16, [1, 4], [256, 64], cache=cache)
    cache.scale[..., 1] = 2.0 ** 60
    check_attn(eng, "f32", 2, 1, 64, 16, [1, 4], [256, 64], cache=cache)
    cache.scale[..., 1] = 2.0 ** -60
    check_attn(eng, "f32", 2, 1, 64, 16, [1, 4], [256, 64], cache=cache)


@pytest.mark.parametrize("d,hkv,news,lens", [(64, 4, [1000, 900], [31000, 20000]), (128, 4, [1000, 900], [31000, 20000]), (256, 2, [1000, 900], [31000, 20000]),
                                             (256, 8, [1] * 48, [8192 - 5 * i for i in range(48)]), (64, 4, [1] * 96, [80000 - 5 * i for i in range(96)])])
def test_attn_f32_sums_do_not_wear_off(eng, d, hkv, news, lens):
    """Keys of about equal weight and values of either sign: the tensor core cuts products off at 2^-24 of the
    sum so far, toward zero, so that a sum of n loses sqrt(n) 2^-24 of itself.  Sums are of 512 keys at
    most (16 with up to 16 rows per kv head) before they are added in f32: 1.4e-6, twice that for the sum's
    spread, and 1e-6 for the scores."""
    cache = Cache([64], 64, hkv, d, 24)  # (for its methods; the pool is made on the GPU)
    pages = [-(-n // 64) for n in lens]
    g = torch.Generator(device="cuda").manual_seed(11)
    total = sum(pages)
    cache.data = torch.empty(total, hkv, 4, 2, 16 * d, dtype=torch.uint8, device="cuda")
    for part in cache.data.split(8192):
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    cache.scale = torch.full((total, hkv, 4, 2), 2.0 ** -6, device="cuda")
    cache.table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    at = 0
    for b, n in enumerate(pages):
        cache.table[b, :n] = order[at:at + n]
        at += n
    q = torch.randn(sum(news), 2 * hkv * d, device="cuda", generator=g)
    out = torch.empty_like(q)
    start, kv_len, _ = rows_of(news, lens)
    eng.kv8_attn(cache.kv8(), 0, q, out, start, kv_len, sum(news), 2 * hkv, d ** -0.5)
    eng.sync()
    # every tenth row is enough
    keep = torch.arange(0, sum(news), 10, device="cuda")
    off = norm = 0.0
    row = 0
    for b, (n, m) in enumerate(zip(news, lens)):
        mine = keep[(keep >= row) & (keep < row + n)]
        if len(mine):
            k, v = cache.values(b, m)
            hide = torch.arange(m, device="cuda")[None] > (m - n + mine - row)[:, None]
            for h in range(2 * hkv):
                z = (q[mine, h * d:(h + 1) * d].double() @ k[:, h // 2].T * d ** -0.5).masked_fill_(hide, -math.inf)
                want = torch.softmax(z, -1) @ v[:, h // 2]
                off += float((out[mine, h * d:(h + 1) * d] - want).square().sum())
                norm += float(want.square().sum())
        row += n
    assert math.sqrt(off / norm) <= 4e-6, math.sqrt(off / norm)


@pytest.mark.parametrize("d,new,rows_form", [(64, 1, 39), (128, 2, 39), (256, 1, 39), (512, 1, 39), (64, 5, 32), (256, 5, 32)])
@pytest.mark.parametrize("depth", [20.3, 25.4, 28.7])
def test_attn_one_dominant_key_and_many_small_ones(eng, d, new, rows_form, depth):
    """Equal p of 2^-depth err alike: each by 2^-22 of itself, and by the last bit that f16 leaves beside
    the dominant one, 2^-39 (2^-32 with many rows per kv head); `total` of them add up."""
    total = 100000
    cache = Cache([total], 64, 1, d, 23)
    cache.data[:, :, :, 0] = 0  # K: scores of 0
    cache.data[:, :, :, 1] = 0x3E  # V: 1.75 scale
    cache.scale[..., 1] = 1.0
    page, slot, t = int(cache.table[0, 100]), 1, 5
    in_k, in_v = (x.reshape(16, d) for x in places(d))
    cache.data[page, 0, slot, 0, in_k[t]] = 0x38  # 1
    cache.data[page, 0, slot, 1, in_v[t]] = 0xB8  # -1
    cache.scale[page, 0, slot, 0] = 1.0
    q = torch.full((new, 8 * d), depth * math.log(2) / math.sqrt(d), device="cuda")
    start, kv_len, _ = rows_of([new], [total])
    out = torch.empty_like(q)
    eng.kv8_attn(cache.kv8(), 0, q, out, start, kv_len, new, 8, d ** -0.5)
    eng.sync()
    want, mass, dz = want_attn(cache, q, [new], [total], 8, d ** -0.5, 0)
    tol = tolerance("f32", want, mass, dz, d) + 1.75 * total * 2.0 ** -rows_form
    assert ((out.double() - want).abs() <= tol).all(), float(((out.double() - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("new", [1, 5, 140])
@pytest.mark.parametrize("kind", ["past_the_end", "before_the_window", "later_row", "no_weight", "no_weight_first", "every_other", "all_but_one"])
def test_attn_large_values_without_weight(eng, dtype, d, new, kind):
    """A record's scale may come from a value that a row does not see, or that has no weight in it: what
    the row sees beside it keeps its precision.  (A refused draft, a token that a window has left, an
    outlier that nothing attends to.)  The other tokens of such a record hold zeros, which is what a scale
    so far above them leaves of them."""
    code, dt = DT[dtype]
    total, window = 409 + new, 150 if kind == "before_the_window" else 0
    cache = Cache([total], 32, 1, d, 17)
    g = torch.Generator(device="cuda").manual_seed(4)
    base = torch.randn(d, device="cuda", generator=g)
    q = (base + 0.1 * torch.randn(new, 4, d, device="cuda", generator=g)).reshape(new, 4 * d).to(dt)
    start, kv_len, _ = rows_of([new], [total])
    dz = want_attn(cache, q, [new], [total], 4, d ** -0.5, window)[2]  # (before: what is added has no weight)
    in_k, in_v = (x.reshape(16, d) for x in places(d))

    def record(pos, exponent, large=None):
        page, slot = int(cache.table[0, pos // 32]), pos % 32 // 16
        cache.data[page, 0, slot, 1] = 0
        cache.scale[page, 0, slot, 1] = 2.0 ** exponent
        if large is not None:
            cache.data[page, 0, slot, 1, in_v[large % 16]] = 0x7E
        return page, slot

    if kind == "past_the_end":
        record(total - 1, 50, total | 15)
    elif kind == "before_the_window":
        first = total - new - window + 1  # the first key that some row sees
        record(first, 50, first - 1 if first % 16 else None)
    elif kind == "later_row":
        record(total - 1, 50, total - 1)
    elif kind in ("no_weight", "no_weight_first"):
        pos = 3 if kind == "no_weight_first" else 200
        page, slot = record(pos, 50, pos)
        cache.data[page, 0, slot, 0] = 0
        cache.scale[page, 0, slot, 0] = 0.25
        cache.data[page, 0, slot, 0, in_k[pos % 16]] = torch.where(base > 0, 0xFE, 0x7E).to(torch.uint8)
    elif kind == "every_other":
        for pos in range(0, total, 32):
            record(pos, 60)
    else:
        for pos in range(0, total, 16):
            if pos != 112:
                record(pos, 60)
        cache.scale[int(cache.table[0, 3]), 0, 1, 1] = 2.0 ** -50
    out = torch.empty_like(q)
    eng.kv8_attn(cache.kv8(), code, q, out, start, kv_len, new, 4, d ** -0.5, window=window)
    eng.sync()
    want, mass, _ = want_attn(cache, q, [new], [total], 4, d ** -0.5, window)
    tol = tolerance(dtype, want, mass, dz, d)
    bad = ~((out.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((out.double() - want).abs() / tol).max()), bad.nonzero()[:3].tolist())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("new", [1, 5, 140])
def test_attn_scales_at_random(eng, dtype, d, new):
    """V records with scales anywhere in 2^-40 .. 2^40 and, every third of them, zeros in half of their
    elements: each element of the output is as near as its own terms allow."""
    cache = Cache([500 + new, 90 + new], 32, 2, d, 21)
    g = torch.Generator(device="cuda").manual_seed(9)
    cache.scale[..., 1] = torch.exp2(torch.randint(-40, 41, cache.scale.shape[:-1], device="cuda", generator=g).float())
    cut = places(d)[1].reshape(16, d)[:, : d // 2].reshape(-1)
    hit = torch.rand(cache.scale.shape[:-1], device="cuda", generator=g) < 1 / 3
    v = cache.data[..., 1, :]
    v[..., cut] = torch.where(hit[..., None], 0, v[..., cut])
    cache.data[..., 1, :] = v
    check_attn(eng, dtype, 8, 2, d, 32, [new, new], [500 + new, 90 + new], cache=cache)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("new", [1, 5, 140])
def test_attn_nan_in_masked_places(eng, dtype, d, new):
    """Stale tokens past the end, tokens before a window and later rows' tokens do not count."""
    code, dt = DT[dtype]
    total, window = 200 + new, 150
    cache = Cache([total], 32, 2, d, 6)
    q = torch.randn(new, 4 * d, device="cuda").to(dt)
    start, kv_len, _ = rows_of([new], [total])

    def run():
        out = torch.empty_like(q)
        eng.kv8_attn(cache.kv8(), code, q, out, start, kv_len, new, 4, 0.1, window=window)
        eng.sync()
        return out

    clean = run()
    in_k, in_v = places(d)

    def poison(pos):
        page, slot, t = int(cache.table[0, pos // 32]), pos % 32 // 16, pos % 16
        for w, p in ((0, in_k), (1, in_v)):
            cache.data[page, :, slot, w, p.reshape(16, d)[t]] = 0x7F

    for pos in range(total, -(-total // 32) * 32):
        poison(pos)
    for pos in range(0, total - new - window + 1):
        poison(pos)
    assert torch.equal(run(), clean)
    if new > 1:  # the last new token's key and value are NaN: its own row alone sees them
        poison(total - 1)
        got = run()
        assert torch.equal(got[:-1], clean[:-1]) and got[-1].isnan().all()
        mid = new // 2
        poison(total - new + mid)
        got = run()
        assert torch.equal(got[:mid], clean[:mid]) and got[mid:].isnan().all()


@pytest.mark.parametrize("new", [2, 140])
def test_attn_nan_value_only(eng, new):
    """A value's NaN reaches the rows that see it, in its element at least, and no other row."""
    d, total = 64, 50 + new
    cache = Cache([total], 16, 1, d, 6)
    q = torch.randn(new, d, device="cuda")
    start, kv_len, _ = rows_of([new], [total])
    pos = total - 1
    clean = torch.empty_like(q)
    eng.kv8_attn(cache.kv8(), sx.DTYPE_F32, q, clean, start, kv_len, new, 1, 0.1)
    cache.data[int(cache.table[0, pos // 16]), 0, 0, 1, places(d)[1].reshape(16, d)[pos % 16, 5]] = 0xFF
    out = torch.empty_like(q)
    eng.kv8_attn(cache.kv8(), sx.DTYPE_F32, q, out, start, kv_len, new, 1, 0.1)
    eng.sync()
    assert torch.equal(out[:-1], clean[:-1]) and out[-1, 5].isnan()


def test_attn_rows_outside_sequences_stay(eng):
    cache = Cache([30, 0, 5], 16, 1, 64, 8)
    q = torch.randn(9, 64, device="cuda")
    out = torch.full_like(q, 3.0)
    eng.kv8_attn(cache.kv8(), sx.DTYPE_F32, q, out, ints([0, 2, 2, 7]), ints([30, 0, 5]), 9, 1, 0.1)
    eng.sync()
    assert (out[7:] == 3.0).all() and not (out[:7] == 3.0).any()


def test_attn_bad_page_masks_and_reports(eng):
    for d in (64, 512):
        for new in (1, 70):
            lens = [new + 90]
            cache = Cache(lens, 16, 2, d, 8)
            page = 1
            good = int(cache.table[0, page])
            cache.table[0, page] = cache.pages
            q = torch.randn(new, 4 * d, device="cuda")
            out = torch.empty_like(q)
            start, kv_len, _ = rows_of([new], lens)
            eng.kv8_attn(cache.kv8(), sx.DTYPE_F32, q, out, start, kv_len, new, 4, 0.1)
            with pytest.raises(sx.SxError) as e:
                eng.sync()
            assert e.value.status == sx.SX_ERR_DEVICE
            # the same as keys of weight zero: compare with the softmax over the other tokens
            cache.table[0, page] = good
            k, v = cache.values(0)
            seen = torch.ones(lens[0], dtype=torch.bool, device="cuda")
            seen[16 * page:16 * page + 16] = False
            for h in range(4):
                z = q[-1, h * d:(h + 1) * d].double() @ k[:, h // 2].T * 0.1
                p = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
                assert torch.allclose(out[-1, h * d:(h + 1) * d].double(), p @ v[:, h // 2], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("start,lens", [([0, 1, 0], [80, 80]), ([0, 1, 1000], [80, 80]), ([0, 1, 2], [80, 100000]), ([0, 1, 2], [80, 0])])
def test_attn_bad_rows_are_skipped_and_reported(eng, new, start, lens):
    cache = Cache([80 * new, 80 * new], 16, 1, 64, 8)
    start = [s if s > 500 else s * new for s in start]
    lens = [x if x > 500 else x * new for x in lens]
    t = 2 * new
    q = torch.randn(t, 64, device="cuda")
    out = torch.full_like(q, 3.0)
    eng.kv8_attn(cache.kv8(), sx.DTYPE_F32, q, out, ints(start), ints(lens), t, 1, 0.1)
    with pytest.raises(sx.SxError) as e:
        eng.sync()
    assert e.value.status == sx.SX_ERR_DEVICE
    assert not (out[:new] == 3.0).any() and (out[new:] == 3.0).all()


def test_attn_beyond_32_bit_offsets(eng):
    """A pool of over 4 GiB: the last pages' byte offsets and record counts pass 32 bits."""
    d, hkv, page = 256, 8, 64
    pages = (5 << 30) // (page * hkv * 2 * d)
    data = torch.zeros(pages, hkv, page // 16, 2, 16 * d, dtype=torch.uint8, device="cuda")
    scale = torch.ones(pages, hkv, page // 16, 2, device="cuda")
    small = Cache([600], page, hkv, d, 12, spare=0)
    n = small.pages
    data[-n:], scale[-n:] = small.data, small.scale
    for new in (1, 40):
        q = torch.randn(new, 16 * d, device="cuda")
        start, kv_len, _ = rows_of([new], [600])
        a, b = torch.empty_like(q), torch.empty_like(q)
        eng.kv8_attn(small.kv8(), sx.DTYPE_F32, q, a, start, kv_len, new, 16, 0.06)
        table = torch.where(small.table >= 0, small.table + (pages - n), small.table)
        big = sx.KV8(data, scale, table, page, hkv, d)
        eng.kv8_attn(big, sx.DTYPE_F32, q, b, start, kv_len, new, 16, 0.06)
        eng.sync()
        assert torch.equal(a, b)


def test_attn_repeats_bit_for_bit_on_any_stream_and_in_a_graph(eng):
    for dtype, new in (("f32", 1), ("bf16", 5), ("bf16", 200)):
        cache, q, out = check_attn(eng, dtype, 8, 2, 128, 32, [new, new], [5000, 300 + new])
        start, kv_len, _ = rows_of([new, new], [5000, 300 + new])
        code, scale, t = DT[dtype][0], 128 ** -0.5, 2 * new
        s = torch.cuda.Stream()
        for _ in range(5):
            other = torch.empty_like(q)
            s.wait_stream(torch.cuda.current_stream())
            eng.set_stream(s.cuda_stream)
            eng.kv8_attn(cache.kv8(), code, q, other, start, kv_len, t, 8, scale)
            eng.sync()
            eng.set_stream(sx.STREAM_LEGACY)
            assert torch.equal(out, other)
        g = torch.cuda.CUDAGraph()
        other = torch.empty_like(q)
        kv8 = cache.kv8()
        with torch.cuda.graph(g, stream=s):
            eng.set_stream(s.cuda_stream)
            eng.kv8_attn(kv8, code, q, other, start, kv_len, t, 8, scale)
        eng.set_stream(sx.STREAM_LEGACY)
        for _ in range(3):
            other.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, other)


@pytest.mark.parametrize("dtype,d", [("f32", 64), ("bf16", 64), ("f32", 128), ("bf16", 128), ("f32", 256), ("bf16", 256), ("f32", 512)])
def test_attn_prompts_repeat_bit_for_bit(eng, dtype, d):
    """Sequences of several row groups and many tiles, split over CTAs: warps that run ahead of one
    another must not change anything."""
    news, lens = [1, 130, 0, 257, 64], [90, 130, 0, 300, 3000]
    cache, q, out = check_attn(eng, dtype, 8, 1, d, 32, news, lens)
    start, kv_len, _ = rows_of(news, lens)
    for _ in range(20):
        other = torch.empty_like(q)
        eng.kv8_attn(cache.kv8(), DT[dtype][0], q, other, start, kv_len, sum(news), 8, d ** -0.5)
        assert torch.equal(out, other)
    eng.sync()


@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_attn_scale_zero_and_negative(eng, new, scale):
    d, total = 64, 100 + new
    cache = Cache([total], 16, 1, d, 6)
    q = torch.randn(new, 2 * d, device="cuda")
    out = torch.empty_like(q)
    start, kv_len, _ = rows_of([new], [total])
    eng.kv8_attn(cache.kv8(), sx.DTYPE_F32, q, out, start, kv_len, new, 2, scale)
    eng.sync()
    want, mass, dz = want_attn(cache, q, [new], [total], 2, scale, 0)
    assert ((out.double() - want).abs() <= tolerance("f32", want, mass, dz, d)).all()


def test_attn_refusals(eng):
    c = Cache([20], 16, 2, 64, 1)
    q = torch.zeros(1, 4 * 64, device="cuda")
    start, kv_len, _ = rows_of([1], [20])

    def call(kv8=None, dtype=sx.DTYPE_F32, q=q, out=q, hq=4, tokens=1, q_ld=0, start=start):
        eng.kv8_attn(kv8 or c.kv8(), dtype, q, out, start, kv_len, tokens, hq, 1.0, q_ld=q_ld)

    def kv8(**kw):
        k = c.kv8()
        for n, v in kw.items():
            setattr(k, n, v)
        return k

    for bad in (dict(dtype=7), dict(q=None), dict(out=None), dict(hq=3), dict(hq=0), dict(hq=256), dict(q_ld=128), dict(q_ld=258),
                dict(start=None), dict(q=q.data_ptr() + 4), dict(kv8=kv8(head_dim=96)), dict(kv8=kv8(page_tokens=24)),
                dict(kv8=kv8(page_tokens=0)), dict(kv8=kv8(num_kv=0)), dict(kv8=kv8(max_pages=1 << 28)), dict(kv8=kv8(num_seqs=5000)),
                dict(kv8=kv8(data=None)), dict(kv8=kv8(scale=c.scale.data_ptr() + 4)), dict(kv8=kv8(table=None)), dict(tokens=1 << 30)):
        with pytest.raises(sx.SxError) as e:
            call(**bad)
        assert e.value.status == sx.SX_ERR_INVALID, bad
    call(tokens=0)
    eng.sync()
    with pytest.raises(ValueError):
        sx.KV8(c.data.flatten()[1:], c.scale, c.table, 16, 2, 64)


# ---------------------------------------------------------------------------------------- append
def step_of(x):
    """Distance between e4m3 neighbours at |x|."""
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp(2.0 ** -6, 448.0))) - 3)


def check_append(eng, dtype, hq, hkv, d, page, news, lens, rot, qkn=True, v_norm=True, k_eq_v=False, seed=1, mul=1.0, cache=None, q=True):
    code, dt = DT[dtype]
    cache = cache or Cache(lens, page, hkv, d, seed)
    t = sum(news)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    width = (hq + 2 * hkv) * d
    qkv = (rnd(t, width) * mul).to(dt)
    qi, ki, vi = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
    gq, gk = 1 + 0.1 * rnd(d), 1 + 0.1 * rnd(d)
    freq = torch.tensor([1e4 ** (-2 * i / max(rot, 1)) for i in range(rot // 2)], device="cuda")
    start, kv_len, host_start = rows_of(news, lens)
    q_out = torch.full((t, hq * d), 5.0, dtype=dt, device="cuda")
    data0, scale0 = cache.data.clone(), cache.scale.clone()
    eng.kv8_append(cache.kv8(), code, qi if q else None, ki, None if k_eq_v else vi, q_out if q else None, start, kv_len, t, hq if q else 0,
                   freq if rot else None, rot, q_norm_w=gq if qkn else None, k_norm_w=gk if qkn else None, v_norm=v_norm, k_eq_v=k_eq_v,
                   eps=1e-6, q_ld=width, k_ld=width, v_ld=width)
    eng.sync()

    def normed(x, w, on):
        x = x.double().reshape(t, -1, d)
        if on:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
            x = x * w.double() if w is not None else x
        return x

    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(news, lens)]).cuda()

    def turned(x):
        if rot == 0:
            return x
        a = (pos.float()[:, None] * freq).double()[:, None]
        h = rot // 2
        x0, x1 = x[..., :h], x[..., h:rot]
        return torch.cat((x0 * a.cos() - x1 * a.sin(), x0 * a.sin() + x1 * a.cos(), x[..., rot:]), -1)

    if q:
        want = turned(normed(qi, gq, qkn)).reshape(t, -1)
        # the norm's sum, its root, three products and the rotation: under 2^-20 of the row's scale
        tol = want.abs() * (2.0 ** -8 if dtype == "bf16" else 0) + want.abs().amax(-1, keepdim=True) * 2.0 ** -19 + 1e-37
        assert ((q_out.double() - want).abs() <= tol).all()
    new_k, new_v = turned(normed(ki, gk, qkn)), normed(ki if k_eq_v else vi, None, v_norm)
    touched = torch.zeros(cache.pages, hkv, page // 16, 2, dtype=torch.bool, device="cuda")
    for b, (m, n) in enumerate(zip(news, lens)):
        if m == 0:
            continue
        for blk in range((n - m) // 16, -(-n // 16)):
            pid, slot = int(cache.table[b, blk * 16 // page]), blk % (page // 16)
            lo, hi = max(n - m, blk * 16), min(n, blk * 16 + 16)
            touched[pid, :, slot] = True
            for w, new in ((0, new_k), (1, new_v)):
                x = new[host_start[b] + lo - (n - m):host_start[b] + hi - (n - m)].transpose(0, 1)  # hkv, cnt, d
                at = places(d)[w]
                old = codes()[data0[pid, :, slot, w][:, at].long()].reshape(hkv, 16, d)
                was = scale0[pid, :, slot, w].double()
                fresh = lo == blk * 16
                if fresh:
                    old, was = torch.zeros_like(old), torch.full_like(was, 2.0 ** -60)
                amax = torch.nan_to_num(x, nan=0.0).abs().amax((-1, -2))
                fit = torch.exp2(torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448)).clamp(-60, 60))
                now = torch.maximum(was, fit)
                got_scale = cache.scale[pid, :, slot, w].double()
                # amax may sit on a power of two's boundary up to the f32 arithmetic's error
                edge = (amax / (448 * fit) > 1 - 2.0 ** -18) | (amax / (224 * fit) < 1 + 2.0 ** -18)
                assert torch.equal(torch.where(edge, now, got_scale), now), (got_scale, now)
                now = got_scale
                got = codes()[cache.data[pid, :, slot, w][:, at].long()].reshape(hkv, 16, d)
                y = old * (was / now)[:, None, None]
                keep = torch.ones(16, dtype=torch.bool, device="cuda")
                keep[lo - blk * 16:hi - blk * 16] = False
                # old codes: nearest at the new scale, untouched when it did not change
                assert ((got - y).abs() <= step_of(y) / 2)[:, keep].all()
                same = (was == now) & torch.tensor(not fresh).cuda()
                raw0, raw = data0[pid, :, slot, w][:, at].reshape(hkv, 16, d), cache.data[pid, :, slot, w][:, at].reshape(hkv, 16, d)
                assert torch.equal(raw0[same][:, keep], raw[same][:, keep])
                z = x / now[:, None, None]
                gz = got[:, ~keep]
                tol = step_of(z) / 2 + amax[:, None, None] / now[:, None, None] * 2.0 ** -18
                assert ((gz - z.clamp(-448, 448)).abs() <= tol).all()
    assert torch.equal(data0[~touched], cache.data[~touched]) and torch.equal(scale0[~touched], cache.scale[~touched])
    return cache, q_out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 32), (256, 64), (256, 256), (512, 512), (128, 0), (64, 2), (128, 126)])
def test_append_ragged(eng, dtype, d, rot):
    news, lens = [1, 1, 1, 5, 20, 0, 33], [1, 16, 17, 50, 20, 7, 100]
    check_append(eng, dtype, 4, 2, d, 32, news, lens, rot, seed=d + rot)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (16, 8), (6, 2)])
@pytest.mark.parametrize("page", [16, 48, 128])
def test_append_heads_and_pages(eng, dtype, hq, hkv, page):
    check_append(eng, dtype, hq, hkv, 64, page, [3, 150, 1], [77, 150, 4], 64, seed=page)


@pytest.mark.parametrize("kw", [dict(qkn=False), dict(v_norm=False), dict(k_eq_v=True), dict(qkn=False, v_norm=False, k_eq_v=True), dict(q=False)])
def test_append_options(eng, kw):
    check_append(eng, "f32", 4, 2, 128, 32, [1, 7, 40], [9, 60, 41], 64, **kw)


@pytest.mark.parametrize("mul", [1e-30, 1e-3, 300.0, 1e25])
def test_append_rescales_older_tokens(eng, mul):
    """New values far below and above what the records hold, and past the scales' range."""
    check_append(eng, "f32", 2, 2, 64, 32, [1, 2, 7, 17], [30, 45, 16, 49], 64, qkn=False, v_norm=False, mul=mul)


def test_append_in_steps_equals_append_at_once(eng):
    """Without rescaling into subnormals, tokens appended one by one store what one call stores."""
    d, hkv, n = 64, 2, 50
    k, v = torch.randn(n, hkv * d, device="cuda"), torch.randn(n, hkv * d, device="cuda")
    k, v = (torch.copysign(x.abs().clamp(0.25, 4.0), x) for x in (k, v))
    one, many = Cache([n], 16, hkv, d, 1), Cache([n], 16, hkv, d, 2)
    many.table = one.table.clone()
    eng.kv8_append(one.kv8(), 0, None, k, v, None, ints([0, n]), ints([n]), n, 0, None, 0)
    for i in range(n):
        eng.kv8_append(many.kv8(), 0, None, k[i:i + 1], v[i:i + 1], None, ints([0, 1]), ints([i + 1]), 1, 0, None, 0)
    eng.sync()
    for a, b in zip(one.values(0), many.values(0)):
        assert torch.equal(a, b)


def test_append_then_attend_matches_unquantised_closely(eng):
    """The two operators together on one sequence: e4m3's 2^-4 relative rounding of keys and values."""
    d, n = 128, 80
    x = torch.randn(n, 3 * d, device="cuda")
    c = Cache([n], 16, 1, d, 1)
    freq = torch.tensor([1e4 ** (-2 * i / d) for i in range(d // 2)], device="cuda")
    q = torch.empty(n, d, device="cuda")
    eng.kv8_append(c.kv8(), 0, x, x[:, d:], x[:, 2 * d:], q, ints([0, n]), ints([n]), n, 1, freq, d, q_ld=3 * d, k_ld=3 * d, v_ld=3 * d)
    out = torch.empty_like(q)
    eng.kv8_attn(c.kv8(), 0, q, out, ints([0, n]), ints([n]), n, 1, d ** -0.5)
    eng.sync()
    k, v = c.values(0)
    z = (q.double() @ k[:, 0].T * d ** -0.5).masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
    assert torch.allclose(torch.softmax(z, -1) @ v[:, 0], out.double(), rtol=1e-4, atol=1e-4)
    assert (v[:, 0] - x[:, 2 * d:].double()).abs().max() <= x.abs().max() * 2.0 ** -4


def test_append_nan_and_inf(eng):
    d = 64
    c = Cache([16], 16, 1, d, 1)
    k, v = torch.randn(16, d, device="cuda"), torch.randn(16, d, device="cuda")
    k[3, 5], v[4, 6], v[7, 8] = math.nan, math.nan, -math.inf
    eng.kv8_append(c.kv8(), 0, None, k, v, None, ints([0, 16]), ints([16]), 16, 0, None, 0)
    eng.sync()
    gk, gv = c.values(0)
    assert gk[3, 0, 5].isnan() and int(gk.isnan().sum()) == 1
    assert gv[4, 0, 6].isnan() and int(gv.isnan().sum()) == 1 and gv[7, 0, 8] == -448 * 2.0 ** 60


def test_append_bad_rows_are_skipped_and_reported(eng):
    for start, lens, table in (([0, 1, 0], [20, 20], None), ([0, 1, 9], [20, 20], None), ([0, 1, 2], [20, 5000], None),
                               ([0, 1, 2], [20, 0], None), ([0, 1, 2], [20, 20], 99)):
        c = Cache([20, 20], 16, 1, 64, 1)
        if table is not None:
            c.table[1, 1] = table
        c0 = c.data.clone()
        k = torch.randn(2, 64, device="cuda")
        eng.kv8_append(c.kv8(), 0, None, k, k, None, ints(start), ints(lens), 2, 0, None, 0)
        with pytest.raises(sx.SxError) as e:
            eng.sync()
        assert e.value.status == sx.SX_ERR_DEVICE
        changed = (c.data != c0).flatten(1).any(1).nonzero().flatten().tolist()
        assert changed == [int(c.table[0, 1])]


def test_append_in_a_graph_and_on_another_stream(eng):
    news, lens = [3, 18], [20, 18]
    a, b = Cache(lens, 16, 2, 64, 1), Cache(lens, 16, 2, 64, 1)
    x = torch.randn(21, 128, device="cuda")
    start, kv_len, _ = rows_of(news, lens)
    eng.kv8_append(a.kv8(), 0, None, x, x, None, start, kv_len, 21, 0, None, 0)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    kv8 = b.kv8()
    with torch.cuda.graph(g, stream=s):
        eng.set_stream(s.cuda_stream)
        eng.kv8_append(kv8, 0, None, x, x, None, start, kv_len, 21, 0, None, 0)
    eng.set_stream(sx.STREAM_LEGACY)
    g.replay()
    g.replay()  # the same rows at the same places again: nothing changes
    torch.cuda.synchronize()
    assert torch.equal(a.data, b.data) and torch.equal(a.scale, b.scale)


def test_append_refusals(eng):
    c = Cache([20], 16, 2, 64, 1)
    x = torch.zeros(1, 256, device="cuda")
    start, kv_len, _ = rows_of([1], [20])

    def call(kv8=None, dtype=0, q=x, k=x, v=x, qo=x, hq=4, rot=0, freq=None, flags=None, k_ld=0, eps=1e-6, tokens=1):
        eng.kv8_append(kv8 or c.kv8(), dtype, q, k, v, qo, start, kv_len, tokens, hq, freq, rot, k_ld=k_ld, eps=eps)

    k8 = c.kv8()
    k8.head_dim = 80
    for bad in (dict(kv8=k8), dict(dtype=2), dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(hq=5), dict(rot=3, freq=x),
                dict(rot=66, freq=x), dict(rot=64), dict(k_ld=64), dict(k_ld=130), dict(eps=-1.0), dict(k=x.data_ptr() + 8), dict(tokens=1 << 31)):
        with pytest.raises(sx.SxError) as e:
            call(**bad)
        assert e.value.status == sx.SX_ERR_INVALID, bad
    call(tokens=0)
    eng.sync()


@pytest.mark.parametrize("rot", [0, 64])
@pytest.mark.parametrize("lead", [1, 15, 16, 17, 32, 100])
def test_append_rows_before_the_first_sequence(eng, lead, rot):
    """A part of a batch: row_start does not begin at 0, and the rows before it belong to nobody."""
    news, lens, d, hq, hkv = [1, 20, 3], [150, 120, 64], 64, 4, 2
    n = sum(news)
    a, b = (Cache(lens, 16, hkv, d, 1, spare=0) for _ in range(2))
    qkv = torch.randn(lead + n, (hq + 2 * hkv) * d, device="cuda")
    freq = torch.tensor([1e4 ** (-2 * i / max(rot, 1)) for i in range(rot // 2)], device="cuda")
    start, kv_len, _ = rows_of(news, lens)
    qa, qb = torch.full((n, hq * d), 5.0, device="cuda"), torch.full((lead + n, hq * d), 5.0, device="cuda")

    def call(c, rows, q_out, start, tokens):
        eng.kv8_append(c.kv8(), 0, rows, rows[:, hq * d:], rows[:, (hq + hkv) * d:], q_out, start, kv_len, tokens, hq,
                       freq if rot else None, rot, q_ld=qkv.shape[1], k_ld=qkv.shape[1], v_ld=qkv.shape[1])

    call(a, qkv[lead:], qa, start, n)
    call(b, qkv, qb, start + lead, lead + n)
    eng.sync()
    assert torch.equal(a.data, b.data) and torch.equal(a.scale, b.scale)
    assert torch.equal(qa, qb[lead:]) and (qb[:lead] == 5.0).all()


@pytest.mark.parametrize("start,lens,tokens", [([0, 1000, 1010, 0, 16], [1000, 400, 3, 16], 1010), ([40, 0, 5], [60, 9], 40), ([1000, 1001], [2000], 8)])
def test_append_falling_rows_are_reported(eng, start, lens, tokens):
    """A record is as it was, or as an append of its sequence alone leaves it, where the sequence's rows fit."""
    d = 64
    a, b, was = (Cache(lens, 16, 1, d, 3) for _ in range(3))
    k = torch.randn(tokens, d, device="cuda")
    eng.kv8_append(a.kv8(), 0, None, k, k, None, ints(start), ints(lens), tokens, 0, None, 0)
    with pytest.raises(sx.SxError) as e:
        eng.sync()
    assert e.value.status == sx.SX_ERR_DEVICE
    for i, (r0, r1) in enumerate(zip(start, start[1:])):
        if r0 <= r1 <= tokens:
            c = sx.KV8(b.data, b.scale, b.table[i:i + 1], 16, 1, d)
            eng.kv8_append(c, 0, None, k, k, None, ints([r0, r1]), ints(lens[i:i + 1]), tokens, 0, None, 0)
    eng.sync()
    as_it_was = (a.data == was.data).all(-1) & (a.scale == was.scale)
    appended = (a.data == b.data).all(-1) & (a.scale == b.scale)
    assert (as_it_was | appended).all()


@pytest.mark.parametrize("wide", [0, 100000])
@pytest.mark.parametrize("new,lead", [(1, 16), (1, 100), (40, 33)])
def test_attn_of_rows_before_the_first_sequence(eng, new, lead, wide):
    lens, d = [150, 64], 64
    Cache.spare_columns = wide  # (put back by the fixture)
    c = Cache(lens, 16, 2, d, 1)
    q = torch.randn(lead + 2 * new, 4 * d, device="cuda")
    start, kv_len, _ = rows_of([new, new], lens)
    a, b = torch.empty(2 * new, 4 * d, device="cuda"), torch.full_like(q, 3.0)
    eng.kv8_attn(c.kv8(), 0, q[lead:], a, start, kv_len, 2 * new, 4, 0.1)
    eng.kv8_attn(c.kv8(), 0, q, b, start + lead, kv_len, lead + 2 * new, 4, 0.1)
    eng.sync()
    assert (a - b[lead:]).abs().max() <= 1e-4 and (b[:lead] == 3.0).all()


def parallel_calls(eng):
    """An attention of each form that is cut over CTAs, and long rows' probabilities: calls that work in
    the engine's memory, and their outputs."""
    d, n = 128, 6000
    c, calls = Cache([n], 16, 2, d, 5), []
    for new in (1, 100):
        q, (start, kv_len, _) = torch.randn(new, 8 * d, device="cuda"), rows_of([new], [n])
        out = torch.empty_like(q)
        calls.append((lambda q=q, out=out, start=start, kv_len=kv_len, new=new:
                      eng.kv8_attn(c.kv8(), 0, q, out, start, kv_len, new, 8, d ** -0.5), out))
    z = torch.randn(24, 262144, device="cuda")
    p = torch.empty_like(z)
    calls.append((lambda: eng.probs(z, p, 24, 262144), p))
    return calls


@pytest.mark.parametrize("which", [0, 1, 2])
def test_calls_follow_one_another_over_streams(eng, which):
    """A call after set_stream begins when the one before it, on the other stream, has ended."""
    call, out = parallel_calls(eng)[which]
    call()
    eng.sync()
    want = out.clone()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    try:
        first, second = torch.cuda.Event(), torch.cuda.Event()
        for s, done in zip(streams, (first, second)):
            eng.set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                if done is first:
                    torch.cuda._sleep(200_000_000)  # a tenth of a second
                call()
                done.record()
        second.synchronize()
        assert first.query()
        # a capture between them: the stream in capture cannot wait, the next one does
        eng.set_stream(streams[0].cuda_stream)
        with torch.cuda.stream(streams[0]):
            torch.cuda._sleep(200_000_000)
            call()
            first.record()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(streams[1]):
            g.capture_begin(capture_error_mode="thread_local")
            eng.set_stream(streams[1].cuda_stream)
            call()
            g.capture_end()
        eng.set_stream(streams[2].cuda_stream)
        with torch.cuda.stream(streams[2]):
            call()
            second.record()
        second.synchronize()
        assert first.query()
        eng.sync()
        with torch.cuda.stream(streams[1]):
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    finally:
        torch.cuda.synchronize()
        eng.sync()
        eng.set_stream(sx.STREAM_LEGACY)


def test_a_stream_may_go_after_a_sync(eng):
    """Nothing is asked of the stream that is left once sx_engine_sync has waited for it."""
    call, out = parallel_calls(eng)[0]
    made, lib = ctypes.c_void_p(), ctypes.CDLL("libcudart.so.12")  # (torch's own streams are never destroyed)
    assert lib.cudaStreamCreateWithFlags(ctypes.byref(made), 1) == 0
    eng.set_stream(made.value)
    call()
    eng.sync()
    assert lib.cudaStreamDestroy(made) == 0
    eng.set_stream(sx.STREAM_LEGACY)
    want = out.clone()
    call()
    eng.sync()
    assert torch.equal(out, want)
