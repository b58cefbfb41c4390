"""The int8 feed-forward operators without a GPU: the argument blocks that the binding packs, and what the
library refuses.  Arguments are looked at before the engine, so a call that would be taken says that the
engine is missing."""
import ctypes as C
import re
import struct
from pathlib import Path

import pytest

import sx

HEADER = (Path(__file__).resolve().parents[1] / "include" / "sx.h").read_text()
KINDS = {"uint32_t": C.c_uint32, "float": C.c_float}
BLOCKS = ["sx_quantize_i8_args", "sx_residual_norm_args", "sx_gemm_i8_args", "sx_gate_up_i8_args"]


def declared(name):
    """The struct `name` of the header as a ctypes one."""
    body = re.search(r"typedef struct \{([^{}]*)\} " + name + ";", HEADER).group(1)
    fields = []
    for line in filter(None, (x.strip() for x in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"))):
        kind, names = re.match(r"(?:const )?(\w+)\s*(.*)", line, re.S).groups()
        for f in (x.strip() for x in names.split(",")):
            fields.append((f.lstrip("* "), C.c_void_p if f.startswith("*") else KINDS[kind]))
    return type(name, (C.Structure,), {"_fields_": fields})


class Recorder:
    def __getattr__(self, name):
        def call(handle, block):
            self.name, self.block = name, bytes(block)
            return 0

        return call


@pytest.fixture
def engine():
    eng = sx.Engine.__new__(sx.Engine)
    eng.h = None
    return eng


def fields(rec, block):
    a = declared(block)
    a = a.from_buffer_copy(rec.block.ljust(C.sizeof(a), b"\0"))
    return {n: getattr(a, n) for n, _ in a._fields_}


@pytest.fixture
def recorded(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(sx, "lib", lambda: rec)
    return rec


def test_every_field_of_a_quantisation(engine, recorded):
    engine.quantize_i8(1, 11, 13, 14, 5, 64, norm_w=12, eps=0.5, x_ld=80, q_ld=96)
    assert recorded.name == "sx_dispatch_quantize_i8"
    assert fields(recorded, BLOCKS[0]) == dict(x=11, norm_w=12, q=13, scale=14, dtype=1, x_ld=80, q_ld=96, rows=5, n=64, eps=0.5)
    engine.quantize_i8(1, 11, 13, 14, 5, 64)
    got = fields(recorded, BLOCKS[0])
    assert (got["norm_w"], got["x_ld"], got["q_ld"]) == (None, 64, 64)


def test_every_field_of_a_seam(engine, recorded):
    engine.residual_norm(11, 1, 12, 15, 2, 16, 5, 64, post_w=13, pre_w=14, scalar=0.25, eps=0.5, y_scale=17, x_ld=68, r_ld=72,
                         x_out_ld=76, y_ld=80)
    assert recorded.name == "sx_dispatch_residual_norm"
    assert fields(recorded, BLOCKS[1]) == dict(x=11, r=12, post_w=13, pre_w=14, x_out=15, y=16, y_scale=17, r_dtype=1, y_dtype=2,
                                               x_ld=68, r_ld=72, x_out_ld=76, y_ld=80, rows=5, n=64, scalar=0.25, eps=0.5)


def test_every_field_of_a_product(engine, recorded):
    engine.gemm_i8(11, 12, 13, 14, 1, 15, 3, 5, 64, x_ld=80, w_ld=96, y_ld=7)
    assert recorded.name == "sx_dispatch_gemm_i8"
    assert fields(recorded, BLOCKS[2]) == dict(x=11, x_scale=12, w=13, w_scale=14, y=15, dtype=1, x_ld=80, w_ld=96, y_ld=7, t=3, n=5, k=64)


def test_every_field_of_a_gated_product(engine, recorded):
    engine.gate_up_i8(11, 12, 13, 15, 14, 16, 1, 17, 3, 5, 64, x_ld=80, w_ld=96, y_ld=7)
    assert recorded.name == "sx_dispatch_gate_up_i8"
    assert fields(recorded, BLOCKS[3]) == dict(x=11, x_scale=12, wg=13, wu=14, wg_scale=15, wu_scale=16, y=17, dtype=1, x_ld=80, w_ld=96,
                                               y_ld=7, t=3, n=5, k=64)


def test_lengths_are_checked_when_the_library_loads(monkeypatch):
    L = sx.lib()
    for i, name in enumerate(BLOCKS):
        assert L.sx_i8_args_bytes(i) == C.sizeof(declared(name))
    assert L.sx_i8_args_bytes(4) == 0
    for i in range(4):
        with monkeypatch.context() as m:
            blocks = list(sx._I8_ARGS)
            blocks[i] = struct.Struct(blocks[i].format + "2I")
            m.setattr(sx, "_I8_ARGS", tuple(blocks))
            with pytest.raises(ImportError, match="int8"):
                sx._check_layouts(L, "libsx.so")


# ------------------------------------------------------------------------------------ refusals
A, B, D, E, F, G = (16 * i for i in range(1, 7))  # addresses that are never read
Q = dict(dtype=0, x=A, q=B, scale=D, rows=5, n=64)
N = dict(x=A, r_dtype=0, r=B, x_out=D, y_dtype=0, y=E, rows=5, n=64, post_w=F, pre_w=G)
P = dict(x=A, x_scale=B, w=D, w_scale=E, dtype=0, y=F, t=5, n=7, k=64)
U = dict(x=A, x_scale=B, wg=D, wg_scale=E, wu=D, wu_scale=E, dtype=0, y=F, t=5, n=7, k=64)


def refusal(engine, call, args):
    with pytest.raises(sx.SxError) as e:
        getattr(engine, call)(**args)
    assert e.value.status == sx.SX_ERR_INVALID
    assert e.value.message.startswith(call + ": "), e.value.message
    return e.value.message[len(call) + 2:]


@pytest.mark.parametrize("call,args", [
    ("quantize_i8", Q), ("quantize_i8", dict(Q, dtype=1, norm_w=E, x_ld=72, q_ld=80)), ("quantize_i8", dict(Q, n=131056)),
    ("quantize_i8", dict(Q, rows=0)), ("residual_norm", N), ("residual_norm", dict(N, post_w=None, y=None, pre_w=None)),
    ("residual_norm", dict(N, r_dtype=1, y_dtype=2, y_scale=A)), ("residual_norm", dict(N, x_out=A)),
    ("gemm_i8", P), ("gemm_i8", dict(P, dtype=1, y=F + 2, x_ld=80, w_ld=96, y_ld=9)), ("gemm_i8", dict(P, k=131056)),
    ("gemm_i8", dict(P, y=F + 4, y_ld=7)), ("gate_up_i8", U), ("gate_up_i8", dict(U, t=0)),
])
def test_taken(engine, call, args):
    assert refusal(engine, call, args) == "null engine"


@pytest.mark.parametrize("call,args,why", [
    ("quantize_i8", dict(Q, dtype=2), "dtype"), ("quantize_i8", dict(Q, dtype=9), "dtype"), ("quantize_i8", dict(Q, x=None), "null"),
    ("quantize_i8", dict(Q, q=None), "null"), ("quantize_i8", dict(Q, scale=None), "null"), ("quantize_i8", dict(Q, n=0), "multiple of 16"),
    ("quantize_i8", dict(Q, n=72), "multiple of 16"), ("quantize_i8", dict(Q, n=131072), "131072"),
    ("quantize_i8", dict(Q, x_ld=48), "shorter"), ("quantize_i8", dict(Q, q_ld=48), "shorter"), ("quantize_i8", dict(Q, x=A + 8), "aligned"),
    ("quantize_i8", dict(Q, x_ld=66), "aligned"), ("quantize_i8", dict(Q, dtype=1, x_ld=68), "aligned"), ("quantize_i8", dict(Q, q=B + 4), "aligned"),
    ("quantize_i8", dict(Q, q_ld=72), "aligned"), ("quantize_i8", dict(Q, norm_w=E + 4), "aligned"), ("quantize_i8", dict(Q, scale=D + 2), "aligned"),
    ("quantize_i8", dict(Q, norm_w=E, eps=-1.0), "eps"), ("quantize_i8", dict(Q, norm_w=E, eps=float("nan")), "eps"),
    ("quantize_i8", dict(Q, rows=1 << 31), "too many"),
    ("residual_norm", dict(N, r_dtype=2), "r_dtype"), ("residual_norm", dict(N, y_dtype=3), "y_dtype"), ("residual_norm", dict(N, x=None), "null"),
    ("residual_norm", dict(N, r=None), "null"), ("residual_norm", dict(N, x_out=None), "null"), ("residual_norm", dict(N, pre_w=None), "pre_w"),
    ("residual_norm", dict(N, n=0), "multiple of 16"), ("residual_norm", dict(N, n=40), "multiple of 16"),
    ("residual_norm", dict(N, n=131072), "131072"), ("residual_norm", dict(N, x_ld=60), "shorter"), ("residual_norm", dict(N, r_ld=60), "shorter"),
    ("residual_norm", dict(N, x_out_ld=60), "shorter"), ("residual_norm", dict(N, y_ld=60), "shorter"), ("residual_norm", dict(N, x_ld=66), "aligned"),
    ("residual_norm", dict(N, r_dtype=1, r_ld=68), "aligned"), ("residual_norm", dict(N, x_out=D + 4), "aligned"),
    ("residual_norm", dict(N, y=E + 4), "aligned"), ("residual_norm", dict(N, pre_w=G + 4), "aligned"), ("residual_norm", dict(N, post_w=F + 4), "aligned"),
    ("residual_norm", dict(N, y_dtype=2), "y_scale"), ("residual_norm", dict(N, y_scale=A), "y_scale"),
    ("residual_norm", dict(N, y_dtype=2, y_scale=A + 1), "aligned"), ("residual_norm", dict(N, y_dtype=2, y_scale=A, y_ld=72), "aligned"),
    ("residual_norm", dict(N, x_out=A, x_out_ld=68), "stride"), ("residual_norm", dict(N, eps=-1e-6), "eps"), ("residual_norm", dict(N, rows=1 << 31), "too many"),
    ("gemm_i8", dict(P, dtype=2), "dtype"), ("gemm_i8", dict(P, k=0), "multiple of 16"), ("gemm_i8", dict(P, k=24), "multiple of 16"),
    ("gemm_i8", dict(P, k=131072), "131072"), ("gemm_i8", dict(P, n=0), "n must"), ("gemm_i8", dict(P, x_ld=48), "shorter"),
    ("gemm_i8", dict(P, w_ld=48), "shorter"), ("gemm_i8", dict(P, y_ld=6), "shorter"), ("gemm_i8", dict(P, x=A + 1), "aligned"),
    ("gemm_i8", dict(P, w=D + 8), "aligned"), ("gemm_i8", dict(P, x_ld=72), "aligned"), ("gemm_i8", dict(P, w_ld=72), "aligned"),
    ("gemm_i8", dict(P, y=F + 2), "aligned"), ("gemm_i8", dict(P, dtype=1, y=F + 1), "aligned"), ("gemm_i8", dict(P, x_scale=B + 2), "aligned"),
    ("gemm_i8", dict(P, w_scale=E + 1), "aligned"), ("gemm_i8", dict(P, t=1 << 31), "below"), ("gemm_i8", dict(P, n=1 << 31, y_ld=1 << 31), "below"),
] + [("gemm_i8", {**P, f: None}, "null") for f in ("x", "x_scale", "w", "w_scale", "y")] + [
    ("gate_up_i8", {**U, f: None}, "null") for f in ("x", "x_scale", "wg", "wg_scale", "wu", "wu_scale", "y")] + [
    ("gate_up_i8", dict(U, wu=D + 8), "aligned"), ("gate_up_i8", dict(U, wu_scale=E + 2), "aligned"), ("gate_up_i8", dict(U, k=8), "multiple of 16"),
])
def test_refused(engine, call, args, why):
    message = refusal(engine, call, args)
    assert why in message and "engine" not in message, message


def test_no_arguments_at_all():
    for call in ("quantize_i8", "residual_norm", "gemm_i8", "gate_up_i8"):
        assert getattr(sx.lib(), "sx_dispatch_" + call)(None, None) == sx.SX_ERR_INVALID
        assert "null arguments" in sx.last_error()


@pytest.mark.parametrize("call,args", [
    ("quantize_i8", dict(Q, rows=0, x=None, q=None, scale=None)), ("quantize_i8", dict(Q, rows=0, x=None, q=None, scale=None, norm_w=E)),
    ("residual_norm", dict(N, rows=0, x=None, r=None, x_out=None, y=None)),
    ("residual_norm", dict(N, rows=0, x=None, r=None, x_out=None, y=None, y_scale=None, y_dtype=2, x_ld=72)),
    ("gemm_i8", dict(P, t=0, x=None, x_scale=None, y=None)), ("gate_up_i8", dict(U, t=0, x=None, x_scale=None, y=None)),
])
def test_no_rows_have_no_addresses(engine, call, args):
    """Tensors of no rows have no memory, and the call no work: nothing but the engine is missed."""
    assert refusal(engine, call, args) == "null engine"


@pytest.mark.parametrize("call,args", [("gemm_i8", dict(P, t=0, w=None)), ("gate_up_i8", dict(U, t=0, wu_scale=None))])
def test_weights_are_there_without_rows_too(engine, call, args):
    assert "null weights" in refusal(engine, call, args)


@pytest.mark.parametrize("call,args", [("gemm_i8", P), ("gate_up_i8", U)])
def test_the_largest_results(engine, call, args):
    """Tiles are counted in 32 bits: t * n below 2^42."""
    for t, n in ((1 << 21, 1 << 21), (1 << 30, 1 << 12)):
        assert "2^42" in refusal(engine, call, dict(args, t=t, n=n, y_ld=n))
        assert refusal(engine, call, dict(args, t=t - 1, n=n, y_ld=n)) == "null engine"
