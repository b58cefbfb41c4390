"""The operators of a feed-forward block in 8-bit whole numbers: cases, inputs, plain forms.

Four operators, each once as elementary torch operations in 32 bits and once as the call of the
library (``own``):

* ``quantize``  rows (RMS-normalised with a gain, or as they are) to int8 with one scale per row;
* ``gemm``      y[t][n] = x_scale[t] w_scale[n] sum_k x[t][k] w[n][k] of int8 operands;
* ``gate_up``   gelu_tanh(gate) * up of two such products;
* ``norm``      the seam of two blocks: the norm after one, the residual and its scale, the norm
                before the next: x' = (x + rms(r) w_post) s, y = rms(x') w_pre, in f32, bf16 or int8.

A row's codes are rint(u * (127 / max|u|)) in f32, u = x * w: the norm's own factor cancels out of
them and enters the scale alone.
"""
import math

import torch

own = False

EPS = 1e-6
SCALAR = 0.875  # of a layer
TINY = 2.0 ** -100  # rows whose largest value is below count as zeros
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token's residual row, normalised and quantised ahead of its projections: latency
        dict(name="quantize_token", op="quantize", t=1, n=3840, dtype="f32", norm=True, pad=0),
        # the activations of 8 packed prompts ahead of the down projection
        dict(name="quantize_prompts", op="quantize", t=2697, n=15360, dtype="bf16", norm=False, pad=0),
        # the seam between two blocks for a step of 8 sessions
        dict(name="norm_sessions", op="norm", t=8, n=3840, dtype="f32", y="f32", pad=0),
        # and for 64 prompts of 264 tokens on average
        dict(name="norm_prompts", op="norm", t=16896, n=3840, dtype="bf16", y="bf16", pad=0),
        # the down projection of one token: streaming the weights
        dict(name="gemm_token", op="gemm", t=1, n=3840, k=15360, dtype="f32", pad=0),
        # q|k|v of a token and four drafts of 8 sessions
        dict(name="gemm_drafts", op="gemm", t=40, n=8192, k=3840, dtype="bf16", pad=0),
        # a short prompt through a smaller model's layer, with odd sizes and a slice of a wider buffer
        dict(name="gemm_ragged", op="gemm", t=361, n=1537, k=6144, dtype="f32", pad=48),
        # the down projection of 8 prompts
        dict(name="gemm_prompts", op="gemm", t=2697, n=3840, k=15360, dtype="bf16", pad=0),
        # q|k|v of 64 prompts
        dict(name="gemm_long", op="gemm", t=16896, n=8192, k=3840, dtype="f32", pad=0),
        # gate and up of one token, of a step of 8 sessions, of 64 prompts
        dict(name="gate_up_token", op="gate_up", t=1, n=15360, k=3840, dtype="f32", pad=0),
        dict(name="gate_up_sessions", op="gate_up", t=8, n=6144, k=1536, dtype="bf16", pad=0),
        dict(name="gate_up_long", op="gate_up", t=16896, n=15360, k=3840, dtype="bf16", pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "gemm", "gemm", "gemm", "gate_up", "gate_up"])
    case = dict(op=op, dtype=rng.choice(["f32", "bf16"]), pad=rng.choice([0, 0, 16 * rng.randint(1, 8)]))
    if op in ("quantize", "norm"):
        n = 16 * _log(rng, 4, 960)
        case.update(t=_log(rng, 1, min(16896, 16896 * 3840 // n)), n=n)
        return dict(case, norm=rng.random() < 0.5) if op == "quantize" else dict(case, y=rng.choice(["f32", "bf16", "i8"]))
    while True:
        t, n, k = _log(rng, 1, 16896), _log(rng, 64, 32768), 16 * _log(rng, 16, 960)
        two = 2 if op == "gate_up" else 1
        if two * n * k <= 30720 * 3840 and t * n <= 16896 * 15360 and two * t * n * k <= 16896 * 30720 * 3840:
            return dict(case, t=t, n=n, k=k)


def work(case):
    t, n, es = case["t"], case["n"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "quantize":
        return {"bytes": t * n * (es + 1) + 4 * t + (4 * n if case["norm"] else 0), "flops": 4 * t * n}
    if case["op"] == "norm":
        ys = {"f32": 4, "bf16": 2, "i8": 1}[case["y"]]
        return {"bytes": t * n * (8 + es + ys) + 8 * n, "flops": 10 * t * n}
    m = 2 if case["op"] == "gate_up" else 1
    k = case["k"]
    return {"bytes": t * k + m * n * k + 4 * (t + m * n) + t * n * es, "flops": 2 * m * t * n * k}


# ----------------------------------------------------------------------------------- inputs
def _codes(g, rows, k, pad, spread):
    """int8 rows as a quantiser leaves them, in a buffer `pad` columns wider, and their scales."""
    u = torch.randn(rows, k, device="cuda", generator=g)
    if spread:  # activations: a few channels are far above the others
        u *= torch.where(torch.rand(k, device="cuda", generator=g) < 0.004, 6.0, 1.0)
    else:  # weights
        u *= 0.02
    top = u.abs().amax(-1, keepdim=True)
    buf = torch.full((rows, k + pad), 77, dtype=torch.int8, device="cuda")
    buf[:, :k] = (u * (127.0 / top)).round_().to(torch.int8)
    return buf[:, :k], (top / 127.0)[:, 0].contiguous()


def _wide(rows, n, pad, dtype):
    return torch.zeros(rows, n + pad, dtype=dtype, device="cuda")[:, :n]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    t, n, pad, dt = case["t"], case["n"], case["pad"], DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("quantize", "norm"):
        # rows of different size, as residual streams and activations have
        x = _wide(t, n, pad, torch.float32 if case["op"] == "norm" else dt)
        x.copy_(rand(t, n) * rand(t, 1).exp())
        if case["op"] == "quantize":
            return dict(s, x=x, w=1 + 0.1 * rand(n) if case["norm"] else None, q=_wide(t, n, pad, torch.int8),
                        scale=torch.zeros(t, device="cuda"))
        r = _wide(t, n, pad, dt)
        r.copy_(rand(t, n) * 3)
        y = _wide(t, n, pad, torch.int8 if case["y"] == "i8" else DTYPES[case["y"]])
        return dict(s, x=x, r=r, post=1 + 0.1 * rand(n), pre=1 + 0.1 * rand(n), x_out=_wide(t, n, pad, torch.float32), y=y,
                    scale=torch.zeros(t, device="cuda"))
    k = case["k"]
    s["x"], s["x_scale"] = _codes(g, t, k, pad, True)
    s["w"], s["w_scale"] = _codes(g, n, k, 0, False)
    if case["op"] == "gate_up":
        s["w_up"], s["w_up_scale"] = _codes(g, n, k, 0, False)
    return dict(s, y=_wide(t, n, pad, dt))


# -------------------------------------------------------------------------- the plain forms
def _rms(x):
    return 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)


def _to_codes(u):
    top = u.abs().amax(-1, keepdim=True)
    top = torch.where(top >= TINY, top, 0.0)
    step = torch.full_like(top, 127.0) / top  # (one rounding: a number over a tensor is a reciprocal and a product)
    return torch.round(u * torch.where(top > 0, step, 0.0)).to(torch.int8), top / 127.0


def _plain_quantize(s):
    x = s["x"].float()
    q, scale = _to_codes(x if s["w"] is None else x * s["w"])
    return {"q": q, "scale": (scale if s["w"] is None else scale * _rms(x))[:, 0]}


def _plain_norm(s):
    r = s["r"].float()
    x = (s["x"] + r * _rms(r) * s["post"]) * SCALAR
    if s["case"]["y"] != "i8":
        return {"x": x, "y": (x * _rms(x) * s["pre"]).to(s["y"].dtype)}
    q, scale = _to_codes(x * s["pre"])
    scale = scale * _rms(x)
    return {"x": x, "scale": scale[:, 0], "y": q * scale.bfloat16()}


def _product(x, x_scale, w, w_scale):
    return x.float() @ w.float().T * x_scale[:, None] * w_scale


def _plain_gemm(s):
    return _product(s["x"], s["x_scale"], s["w"], s["w_scale"]).to(s["y"].dtype)


def _plain_gate_up(s):
    g = _product(s["x"], s["x_scale"], s["w"], s["w_scale"])
    u = _product(s["x"], s["x_scale"], s["w_up"], s["w_up_scale"])
    h = 0.5 * g * (1.0 + torch.tanh(0.7978845608 * (g + 0.044715 * g * g * g)))
    return (h * u).to(s["y"].dtype)


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
        _held.update(sx=sx, engine=e, types={torch.float32: sx.DTYPE_F32, torch.bfloat16: sx.DTYPE_BF16, torch.int8: sx.DTYPE_I8})
    return _held["engine"], _held["types"]


def _own(s):
    e, types = _engine()
    op, t, n = s["case"]["op"], s["case"]["t"], s["case"]["n"]
    if op == "quantize":
        e.quantize_i8(types[s["x"].dtype], s["x"], s["q"], s["scale"], t, n, norm_w=s["w"], eps=EPS, x_ld=s["x"].stride(0), q_ld=s["q"].stride(0))
        return {"q": s["q"], "scale": s["scale"]}
    if op == "norm":
        eight = s["case"]["y"] == "i8"
        e.residual_norm(s["x"], types[s["r"].dtype], s["r"], s["x_out"], types[s["y"].dtype], s["y"], t, n, post_w=s["post"], pre_w=s["pre"],
                        scalar=SCALAR, eps=EPS, y_scale=s["scale"] if eight else None, x_ld=s["x"].stride(0), r_ld=s["r"].stride(0),
                        x_out_ld=s["x_out"].stride(0), y_ld=s["y"].stride(0))
        if eight:
            return {"x": s["x_out"], "scale": s["scale"], "y": s["y"] * s["scale"].bfloat16()[:, None]}
        return {"x": s["x_out"], "y": s["y"]}
    k, dt = s["case"]["k"], types[s["y"].dtype]
    if op == "gemm":
        e.gemm_i8(s["x"], s["x_scale"], s["w"], s["w_scale"], dt, s["y"], t, n, k, x_ld=s["x"].stride(0), y_ld=s["y"].stride(0))
    else:
        e.gate_up_i8(s["x"], s["x_scale"], s["w"], s["w_scale"], s["w_up"], s["w_up_scale"], dt, s["y"], t, n, k,
                     x_ld=s["x"].stride(0), y_ld=s["y"].stride(0))
    return s["y"]


_PLAIN = {"quantize": _plain_quantize, "norm": _plain_norm, "gemm": _plain_gemm, "gate_up": _plain_gate_up}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------------------- 64-bit definitions
def _sums(x, w):
    """sum_k x[t][k] w[n][k]: whole numbers below 2^53, so f64 products and sums are exact."""
    out = torch.empty(x.shape[0], w.shape[0], dtype=torch.float64, device="cuda")
    wt = w.double().T
    for i in range(0, x.shape[0], 2048):
        torch.matmul(x[i:i + 2048].double(), wt, out=out[i:i + 2048])
    return out


def _exact_norm(s):
    r, x = s["r"].double(), s["x"].double()
    h = r / (r.square().sum(-1, keepdim=True) / r.shape[-1] + EPS).sqrt()
    x = (x + h * s["post"].double()) * SCALAR
    y = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * s["pre"].double()
    if s["case"]["y"] != "i8":
        return {"x": x, "y": y}
    step = y.abs().amax(-1, keepdim=True) / 127
    return {"x": x, "scale": step[:, 0], "y": torch.round(y / step) * step}


def exact(case, seed):
    """run()'s outputs in 64 bits; codes are whole numbers and have none."""
    s = prepare(case, seed)
    if case["op"] == "quantize":
        y = s["x"].double()
        if case["norm"]:
            y = y / (y.square().sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * s["w"].double()
        return {"q": None, "scale": y.abs().amax(-1) / 127}
    if case["op"] == "norm":
        return _exact_norm(s)
    out = _sums(s["x"], s["w"]).mul_(s["x_scale"].double()[:, None]).mul_(s["w_scale"].double())
    if case["op"] == "gate_up":
        out = out * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (out + 0.044715 * out ** 3)))
        out *= _sums(s["x"], s["w_up"]).mul_(s["x_scale"].double()[:, None]).mul_(s["w_up_scale"].double())
    return out
