"""The argument blocks that the binding packs by hand for the paged 8-bit cache, against the structs in the
header: lengths at load, and every field at its place."""
import ctypes as C
import re
import struct
from pathlib import Path

import pytest

import sx

torch = pytest.importorskip("torch")

HEADER = (Path(__file__).resolve().parents[1] / "include" / "sx.h").read_text()


def declared(name, known=()):
    """The struct `name` of the header as a ctypes one."""
    body = re.search(r"typedef struct \{([^{}]*)\} " + name + ";", HEADER).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for line in filter(None, (x.strip() for x in body.split(";"))):
        kind, names = re.match(r"(?:const )?(\w+)\s*(.*)", line, re.S).groups()
        for f in names.split(","):
            f = f.strip()
            base = dict(known).get(kind) or {"void": None, "uint32_t": C.c_uint32, "float": C.c_float}[kind]
            fields.append((f.lstrip("* "), C.c_void_p if f.startswith("*") else base))
    return type(name, (C.Structure,), {"_fields_": fields})


CACHE = declared("sx_kv8")


def test_lengths_are_checked_when_the_library_loads(monkeypatch):
    L = sx.lib()
    sx._check_layouts(L, "libsx.so")
    for name in ("_APPEND_ARGS", "_ATTN_ARGS"):
        with monkeypatch.context() as m:
            m.setattr(sx, name, struct.Struct(getattr(sx, name).format + "2I"))
            with pytest.raises(ImportError, match="args"):
                sx._check_layouts(L, "libsx.so")


class Recorder:
    """A library that keeps the block it is called with."""

    def __getattr__(self, name):
        def call(handle, block):
            self.name, self.block = name, bytes(block)
            return 0

        return call


@pytest.fixture
def recorded(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(sx, "lib", lambda: rec)
    eng = sx.Engine.__new__(sx.Engine)
    eng.h = None
    data, scale = torch.zeros(6, 2, 1, 2, 16 * 64, dtype=torch.uint8), torch.zeros(6, 2, 1, 2)
    table = torch.zeros(3, 5, dtype=torch.int32)
    return rec, eng, sx.KV8(data, scale, table, 16, 2, 64), (data, scale, table)


def check_cache(c, tensors):
    data, scale, table = tensors
    assert (c.data, c.scale, c.table) == (data.data_ptr(), scale.data_ptr(), table.data_ptr())
    assert (c.num_pages, c.page_tokens, c.max_pages, c.num_seqs, c.num_kv, c.head_dim) == (6, 16, 5, 3, 2, 64)


def test_every_field_of_an_append(recorded):
    rec, eng, cache, tensors = recorded
    eng.kv8_append(cache, 1, 11, 12, 13, 16, 17, 18, 20, 8, 19, 32, q_norm_w=14, k_norm_w=15, v_norm=True, k_eq_v=True,
                   eps=0.5, q_ld=1024, k_ld=256, v_ld=512)
    assert rec.name == "sx_dispatch_kv8_append_args"
    a = declared("sx_kv8_append_args", {"sx_kv8": CACHE}.items())
    a = a.from_buffer_copy(rec.block.ljust(C.sizeof(a), b"\0"))
    check_cache(a.cache, tensors)
    assert (a.q_in, a.k_in, a.v_in, a.q_norm_w, a.k_norm_w, a.q_out, a.row_start, a.kv_len, a.inv_freq) == tuple(range(11, 20))
    assert (a.dtype, a.q_ld, a.k_ld, a.v_ld, a.tokens, a.num_q, a.rotary_dim) == (1, 1024, 256, 512, 20, 8, 32)
    assert a.flags == sx.KV8_V_NORM | sx.KV8_K_EQ_V and a.eps == 0.5


def test_every_field_of_an_attention(recorded):
    rec, eng, cache, tensors = recorded
    eng.kv8_attn(cache, 1, 11, 12, 13, 14, 20, 8, 0.25, window=77, q_ld=1024, out_ld=2048)
    assert rec.name == "sx_dispatch_kv8_attn_args"
    a = declared("sx_kv8_attn_args", {"sx_kv8": CACHE}.items())
    a = a.from_buffer_copy(rec.block.ljust(C.sizeof(a), b"\0"))
    check_cache(a.cache, tensors)
    assert (a.q, a.out, a.row_start, a.kv_len) == (11, 12, 13, 14)
    assert (a.dtype, a.q_ld, a.out_ld, a.tokens, a.num_q, a.window, a.scale) == (1, 1024, 2048, 20, 8, 77, 0.25)
