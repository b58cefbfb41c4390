"""Page bookkeeping of the paged KV cache (host only) against a dictionary restatement, and the
refusals that need no GPU."""
import random

import numpy as np
import pytest

import sx


def test_pages_random_walk_never_shares_or_loses_a_page():
    rng = random.Random(5)
    pages, tokens, seqs, width = 40, 32, 6, 12
    p = sx.Pages(pages, tokens, seqs, width)
    length, released = [0] * seqs, [0] * seqs
    for _ in range(3000):
        s, op = rng.randrange(seqs), rng.randrange(10)
        if op < 5:
            want = length[s] + rng.randint(0, 90)
            need = -(-max(want, length[s]) // tokens) - -(-length[s] // tokens)
            if want > width * tokens:
                with pytest.raises(sx.SxError) as e:
                    p.extend(s, want)
                assert e.value.status == sx.SX_ERR_INVALID
            elif need > p.free_count:
                before, free = p.table(), p.free_count
                with pytest.raises(sx.SxError) as e:
                    p.extend(s, want)
                assert e.value.status == sx.SX_ERR_OOM
                assert np.array_equal(before, p.table()) and free == p.free_count
            else:
                p.extend(s, want)
                length[s] = max(length[s], want)
        elif op < 8:
            # keep at least one page that was not released
            floor = released[s] * tokens + 1
            to = rng.choice([0, rng.randint(min(floor, length[s]), length[s])])
            p.truncate(s, to)
            length[s] = to
            if to == 0:
                released[s] = 0
        else:
            pos = rng.randint(0, length[s])
            # a release up to the very end would leave nothing to append to
            pos = min(pos, max(0, length[s] - 1))
            p.release_before(s, pos)
            released[s] = max(released[s], pos // tokens)
        t = p.table()
        held = []
        for i in range(seqs):
            assert p.length(i) == length[i]
            have = -(-length[i] // tokens)
            assert (t[i, :released[i]] == sx.NO_PAGE).all() and (t[i, have:] == sx.NO_PAGE).all()
            held += t[i, released[i]:have].tolist()
        assert sx.NO_PAGE not in held and len(set(held)) == len(held) and max(held, default=0) < pages
        assert len(held) + p.free_count == pages


def test_pages_truncate_past_a_released_page_is_refused():
    p = sx.Pages(8, 16, 1, 8)
    p.extend(0, 100)
    p.release_before(0, 64)
    with pytest.raises(sx.SxError):
        p.truncate(0, 64)
    p.truncate(0, 65)
    with pytest.raises(sx.SxError):
        p.truncate(0, 66)
    p.truncate(0, 0)
    assert p.free_count == 8


def test_pages_truncate_to_the_same_length_changes_nothing():
    """A step whose drafts all stand takes nothing back, also when a window has passed every full page."""
    p = sx.Pages(8, 16, 1, 8)
    p.extend(0, 64)
    p.release_before(0, 64)
    before = p.table()
    p.truncate(0, 64)
    assert np.array_equal(before, p.table()) and p.length(0) == 64 and p.free_count == 8
    p.extend(0, 65)
    assert p.table()[0].tolist()[:4] == [sx.NO_PAGE] * 4 and p.table()[0, 4] < 8
    p.truncate(0, 0)
    p.truncate(0, 0)
    assert p.free_count == 8


@pytest.mark.parametrize("args", [(0, 16, 1, 1), (4, 0, 1, 1), (4, 24, 1, 1), (4, 2048, 1, 1), (4, 16, 0, 1),
                                  (4, 16, 1, 0), (4, 1024, 1, 1 << 21)])
def test_pages_bad_geometry(args):
    with pytest.raises(sx.SxError):
        sx.Pages(*args)


def test_pages_unknown_sequence():
    p = sx.Pages(4, 16, 2, 2)
    for call in (lambda: p.extend(2, 1), lambda: p.truncate(2, 0), lambda: p.release_before(2, 0)):
        with pytest.raises(sx.SxError):
            call()
    assert p.length(2) == 0


def test_dispatches_refuse_a_null_engine():
    L = sx.lib()
    assert L.sx_dispatch_kv8_append(None, None, 0, *[None] * 3, 0, 0, 0, *[None] * 5, 1, 1, None, 0, 0, 0.0) == sx.SX_ERR_INVALID
    assert L.sx_dispatch_kv8_attn(None, None, 0, None, None, 0, 0, None, None, 1, 1, 0, 1.0) == sx.SX_ERR_INVALID
    assert L.sx_dispatch_probs(None, None, 0, None, 0, 1, 1, 1.0) == sx.SX_ERR_INVALID
    assert L.sx_dispatch_verify(None, None, 0, None, 0, *[None] * 6, 1, 1, 1) == sx.SX_ERR_INVALID
    assert "null" in sx.last_error()
