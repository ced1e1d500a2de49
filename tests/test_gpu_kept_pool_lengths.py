"""Forks and trims of sequences whose window layers' rings hold newer tokens: refused where the next
token would see a position that the ring no longer holds."""
import random

import pytest

from keptcase import BF16, BLOCK

pytestmark = pytest.mark.gpu

LEN = 150


def pool_of(gkv, fmt, window, kept, layers=2, blocks=40):
    return gkv.Pool(n_layers=layers, n_kv_heads=1, max_seqs=4, max_seq_len=256, window=window,
                    num_blocks=blocks if layers > 1 else 0, v_format=fmt, kept=kept)


def held(kept, window, n, written):
    """Whether the token behind n tokens finds all that it sees, `written` tokens after the
    first in the ring, simulated place by place."""
    place = {}
    if kept is None:  # slot = position % window
        for t in range(written):
            place[t % window] = t
        return all(place[t % window] == t for t in range(max(0, n - window + 1), n))
    ring, kb = window // 16 + 1, kept // 16

    def entry(j):
        return j if j < kb else kb + (j - kb) % ring

    for t in range(written):
        place[entry(t // 16)] = t // 16
    return all(place[entry(t // 16)] == t // 16 for t in range(n) if t < kept or t > n - window)


def refused(gkv, call, *args):
    with pytest.raises(gkv.GkvError) as e:
        call(*args)
    assert e.value.status == gkv.GKV_ERR_ARG


@pytest.mark.parametrize("fmt,window,kept", [(BF16, 32, 16), (BLOCK, 32, 0), (BLOCK, 16, 48), (BF16, 32, None),
                                             (BF16, 64, None)])
@pytest.mark.parametrize("layers", [2, 1])  # (one: a window layer alone)
@pytest.mark.parametrize("written", [LEN, 144, 145, 30])
def test_fork_and_trim_go_back_as_far_as_the_ring(gkv, cuda, fmt, window, kept, layers, written):
    pool = pool_of(gkv, fmt, window, kept, layers)
    a = pool.seq_alloc()
    assert pool.reserve(a, written) == 0
    for n in range(written + 1):
        free = pool.free_blocks()
        if held(kept, window, n, written):
            c = pool.fork(a, n)
            pool.trim(c, n)
            assert pool.free(c) == 0
        else:
            refused(gkv, pool.fork, a, n)
            refused(gkv, pool.trim, a, n)
        assert pool.free_blocks() == free
    b, c, d = (pool.seq_alloc() for _ in range(3))  # (no refused call took a sequence)
    if written == LEN:
        assert not held(kept, window, 100, written)
    pool.trim(a, 0)
    pool.close()


def test_no_window_no_refusal(gkv, cuda):
    pool = pool_of(gkv, BLOCK, 0, None)
    a = pool.seq_alloc()
    assert pool.reserve(a, 250) == 0
    c = pool.fork(a, 17)
    pool.trim(a, 33)
    assert len(pool.seq_blocks(c)) == 2 and len(pool.seq_blocks(a)) == 3
    pool.close()


def test_room_made_ahead(gkv, cuda):
    """The last reserve's length counts: one of the tokens that are there makes up for room made
    ahead of them, and gives no block back."""
    pool = pool_of(gkv, BLOCK, 32, 16)
    a = pool.seq_alloc()
    assert pool.reserve(a, 250) == 0
    refused(gkv, pool.fork, a, 100)
    assert pool.reserve(a, 100) == 0 and len(pool.seq_blocks(a)) == 16
    c = pool.fork(a, 100)
    assert len(pool.seq_blocks(c)) == 7
    pool.trim(a, 100)
    assert len(pool.seq_blocks(a)) == 7
    pool.close()


def test_what_a_trim_dropped_stays_overwritten(gkv, cuda):
    """A shorter length behind a trim, or in a fork, brings nothing back into the ring."""
    pool = pool_of(gkv, BF16, 32, 0)
    a = pool.seq_alloc()
    assert pool.reserve(a, 130) == 0
    pool.trim(a, 128)                          # block 8 has been begun: block 5 is gone
    c = pool.fork(a, 128)
    for x in (a, c):
        assert pool.reserve(x, 128) == 0
        refused(gkv, pool.trim, x, 120)
        refused(gkv, pool.fork, x, 120)
        assert pool.reserve(x, 129) == 0
    assert pool.free(c) == 0
    b = pool.seq_alloc()                       # (a new sequence starts with an empty ring)
    assert pool.reserve(b, 60) == 0
    pool.trim(b, 48)
    pool.trim(a, 0)                            # begun anew: what is appended now is there
    assert pool.reserve(a, 50) == 0
    pool.trim(a, 48)
    pool.trim(pool.fork(a, 48), 47)
    pool.close()


@pytest.mark.parametrize("window,kept", [(32, 16), (48, 0), (32, None)])
def test_appends_trims_and_forks_in_any_order(gkv, cuda, window, kept):
    """... against the rings simulated place by place."""
    unit, kb, ring = (1, 0, window) if kept is None else (16, kept // 16, window // 16 + 1)
    entry = lambda u: u if u < kb else kb + (u - kb) % ring  # noqa: E731
    rng = random.Random(window)
    pool = pool_of(gkv, BF16, window, kept, blocks=96)
    lens, places = {}, {}
    x = pool.seq_alloc()
    lens[x], places[x] = 0, {}
    n_ok = n_no = 0
    for _ in range(1500):
        x = rng.choice(list(lens))
        if rng.random() < 0.5:
            n = rng.choice([1, 1, 3, 20, 50])
            if lens[x] + n <= 250 and pool.reserve(x, lens[x] + n) == 0:
                for u in range(lens[x] // unit, (lens[x] + n - 1) // unit + 1):
                    places[x][entry(u)] = u
                lens[x] += n
            continue
        n = max(0, lens[x] - rng.choice([0, 1, 2, 9, 17, 30, 33, 200]))
        fits = all(places[x].get(entry(t // unit)) == t // unit
                   for t in range(n) if t < (kept or 0) or t > n - window)
        trim = rng.random() < 0.5 or len(lens) == 4
        if not fits:
            refused(gkv, pool.trim if trim else pool.fork, x, n)
            n_no += 1
        elif trim:
            pool.trim(x, n)
            lens[x] = n
        else:
            try:
                c = pool.fork(x, n)
            except gkv.GkvError as e:
                assert e.status == gkv.GKV_ERR_CAPACITY
                continue
            lens[c], places[c] = n, dict(places[x])
        n_ok += fits
        if len(lens) == 4:
            y = rng.choice(list(lens))
            assert pool.free(y) == 0
            del lens[y], places[y]
    assert n_ok > 200 and n_no > 50
    pool.close()
