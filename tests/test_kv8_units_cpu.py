"""Which block of which sequence a CTA of the paged 8-bit append takes: the kernel's own integers
(sx_kv8_units.h), compiled for the host, against a walk over the sequences."""
import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parents[1] / "ai-research_b200" / "csrc"

# What sx_kv8_append.cu does with a unit before it touches a page, the search by 32 lanes included: one
# row of {sequence, block, first row, rows, place in the block} for each CTA that has work; bad: the call
# is reported.
HOST = r"""
#include "sx_kv8_units.h"
using namespace sx;
extern "C" int units(const uint32_t *row_start, const uint32_t *kv_len, uint32_t seqs, uint32_t tokens, uint32_t max_len,
                     uint32_t *out, int *bad) {
  int n = 0;
  *bad = 0;
  for (uint32_t i = 0; i < seqs; ++i) *bad |= row_start[i] > row_start[i + 1] || row_start[i + 1] > tokens;
  for (uint32_t u = 0; u < kv8_unit_count(tokens, seqs); ++u) {
    uint32_t b = 0;
    for (uint32_t left = seqs; left > 1;) {
      const uint32_t step = (left + 31) / 32;
      uint32_t k = 0;
      for (uint32_t lane = 0; lane < 32; ++lane)
        k += step * lane < left && kv8_unit_base(row_start[b + step * lane], b + step * lane) <= u;
      const uint32_t skip = k ? step * (k - 1) : 0;
      b += skip;
      left = step < left - skip ? step : left - skip;
    }
    Kv8Rows r;
    if (!kv8_rows_fit(row_start[b], row_start[b + 1], kv_len[b], tokens, max_len, &r)) {
      *bad = 1;
      continue;
    }
    Kv8Unit x;
    if (!kv8_unit(r, u - kv8_unit_base(r.r0, b), &x)) continue;
    const uint32_t row[5] = {b, x.block, x.row0, x.cnt, x.t0};
    for (int k = 0; k < 5; ++k) out[5 * n + k] = row[k];
    ++n;
  }
  return n;
}
"""


@pytest.fixture(scope="module")
def units(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("units")
    (d / "u.cpp").write_text(HOST)
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(CSRC), str(d / "u.cpp"),
                    "-o", str(d / "u.so")], check=True)
    lib = ctypes.CDLL(str(d / "u.so"))

    def call(row_start, kv_len, tokens, max_len):
        rs, kl = np.array(row_start, np.uint32), np.array(kv_len, np.uint32)
        out, bad = np.zeros((tokens // 16 + 2 * len(kl) + 1, 5), np.uint32), ctypes.c_int()
        ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
        n = lib.units(ptr(rs), ptr(kl), len(kl), tokens, max_len, ptr(out), ctypes.byref(bad))
        return [tuple(int(x) for x in row) for row in out[:n]], bool(bad.value)

    return call


def want(row_start, kv_len, tokens, max_len):
    """Every block that holds new rows of a sequence that fits; whether one does not; whether row_start falls."""
    out, bad = [], False
    for b, n_len in enumerate(kv_len):
        r0, r1 = row_start[b], row_start[b + 1]
        if r1 < r0 or r1 > tokens or r1 - r0 > n_len or n_len > max_len:
            bad = True
            continue
        first = n_len - (r1 - r0)
        for blk in range(first // 16, -(-n_len // 16)) if r1 > r0 else ():
            lo, hi = max(first, 16 * blk), min(n_len, 16 * blk + 16)
            out.append((b, blk, r0 + lo - first, hi - lo, lo - 16 * blk))
    return out, bad, any(a > b for a, b in zip(row_start, row_start[1:]))


def check(units, row_start, kv_len, tokens, max_len=4096):
    got, bad = units(row_start, kv_len, tokens, max_len)
    blocks, wrong, falls = want(row_start, kv_len, tokens, max_len)
    assert len(set(got)) == len(got) and bad == wrong, (row_start, kv_len, tokens)
    if falls:  # reported, and nothing but blocks of sequences that fit
        assert set(got) <= set(blocks), (row_start, kv_len, tokens)
    else:
        assert sorted(got) == blocks, (row_start, kv_len, tokens)


@pytest.mark.parametrize("row_start,kv_len,tokens", [([16, 17], [49], 17), ([32, 33], [50], 33), ([32, 33], [101], 33),
                                                     ([100, 140, 141], [300, 1], 141), ([0, 1000, 1010, 0, 16], [1000, 400, 3, 16], 1010),
                                                     ([0, 1, 0], [20, 20], 2), ([40, 0, 5], [60, 9], 40), ([1000, 1001], [2000], 8),
                                                     ([0, 16, 16, 31], [16, 500, 15], 31)])
def test_units_of_part_batches_and_falling_rows(units, row_start, kv_len, tokens):
    check(units, row_start, kv_len, tokens)


def test_units_of_random_batches(units):
    rng = random.Random(8)
    for n in range(4000):
        seqs = rng.randint(1, 40 if n % 20 else 1500)
        start = [rng.choice([0, rng.randint(0, 100)])]
        for _ in range(seqs):
            start.append(start[-1] + rng.choice([0, 1, 1, rng.randint(0, 9), rng.randint(0, 300 if seqs < 50 else 5)]))
        lens = [b - a + rng.choice([0, rng.randint(0, 400)]) for a, b in zip(start, start[1:])]
        tokens = start[-1] + rng.choice([0, 0, rng.randint(0, 50)])
        spoil = rng.random()
        if spoil < 0.2:
            start[rng.randrange(seqs + 1)] = rng.randint(0, 2 * tokens + 2)
        elif spoil < 0.3:
            lens[rng.randrange(seqs)] = rng.choice([0, 5000, 0xFFFFFFFF])
        elif spoil < 0.35:
            tokens = rng.randint(0, tokens)
        check(units, start, lens, tokens)
