"""The host's lists of which tiles hold a key, carried through squeezes and copies: by-key searches afterwards wait for nothing
and answer as a search of the whole gallery does."""
import numpy as np
import pytest
import torch

from test_gpu_pages import DEAD, Pair, ctx      # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu


def squeeze_twin(p, to=None):
    to = p if to is None else to
    live = np.flatnonzero(p.k >= 0)
    t, k = p.t[live].copy(), p.k[live].copy()
    to.k[:] = DEAD
    to.t[:live.size], to.k[:live.size] = t, k


@pytest.mark.parametrize("how", ["in place", "into another", "copied under their own keys", "within the gallery"])
def test_a_by_key_search_afterwards_only_enqueues(how):
    """The stream is kept busy; the search returns before it is idle."""
    from frhot.engine import Context, Gallery
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = Context(device=0, max_batch=1, stream=s.cuda_stream)
        n = 20000
        g, h = Gallery(c, 64, 2 * n), Gallery(c, 64, 2 * n)
        rows = torch.nn.functional.normalize(torch.randn(n, 64, device="cuda")).half()
        keys = np.arange(n // 100, dtype=np.int32)
        g.write_dev(rows.data_ptr(), np.arange(0, n, 100), np.full(n // 100, 100, np.int32), keys)
        g.tombstone(np.arange(0, n, 3))
        q, ask = rows[[301, 5002, 6001, 6100]].contiguous(), np.array([3, 50, 60, 61], np.int32)
        out = [None] + [(torch.empty(4, 5, device="cuda"), torch.empty(4, 5, dtype=torch.int64, device="cuda")) for _ in range(2)]

        def search(gal, o):
            gal.search_dev_keyed(q.data_ptr(), ask, 4, 5, o[0].data_ptr(), o[1].data_ptr())
        more = (torch.empty(64, 5, device="cuda"), torch.empty(64, 5, dtype=torch.int64, device="cuda"))
        for gal in (g, h):                      # (buffers are allocated by the first search, here by a larger one)
            gal.search_mode(Gallery.SEARCH_BY_KEY)
            if gal is h:
                h.write_dev(rows.data_ptr(), np.arange(0, n, 100), np.full(n // 100, 100, np.int32), keys)
            gal.search_dev_keyed(rows.data_ptr(), keys[:64], 64, 5, more[0].data_ptr(), more[1].data_ptr())
        h.free_keys(keys)
        s.synchronize()
        asked = h
        if how == "in place":
            g.compact()
            asked = g
        elif how == "into another":
            g.compact(h)
        elif how == "copied under their own keys":
            h.copy([0, 10000], [10000, 0], [10000, 10000], source=g)
        else:
            g.copy([0, 10000], [30000, 20000], [10000, 10000])
            asked = g
        torch.cuda._sleep(50_000_000)
        mark = torch.cuda.Event()
        mark.record(s)
        search(asked, out[1])
        busy = not mark.query()
        s.synchronize()
        assert busy
        asked.search_mode(Gallery.SEARCH_WHOLE)
        search(asked, out[2])
        s.synchronize()
        assert torch.equal(out[1][0], out[2][0]) and torch.equal(out[1][1], out[2][1])
        assert (out[1][1][:, 0] >= 0).all() and (out[1][0][[0, 1, 2], 0] - 1).abs().max() <= 1e-3
        g.close(), h.close(), c.close()


def agree(p, nq, seed):
    """By key and whole: the same answers, and the twin's best row.  (Rows that were never written are zero and may live: they
    are not asked for.)"""
    live = np.flatnonzero((p.k >= 0) & (p.t != 0).any(1))
    if live.size == 0:
        return
    at = np.random.default_rng(seed).choice(live, nq)
    q = p.t[at].astype(np.float64)
    q /= np.linalg.norm(q, axis=1, keepdims=True)
    answers = []
    for mode in (p.gal.SEARCH_BY_KEY, p.gal.SEARCH_WHOLE):
        p.gal.search_mode(mode)
        answers.append(p.gal.search(q.astype(np.float32), p.k[at], 5))
    (s, r), (ws, wr) = answers
    assert np.array_equal(s, ws) and np.array_equal(r, wr)
    for i in range(nq):
        mine = np.flatnonzero(p.k == p.k[at[i]])
        assert p.k[r[i, 0]] == p.k[at[i]] and abs(s[i, 0] - (p.t[mine].astype(np.float64) @ q[i]).max()) <= 2e-3


@pytest.mark.parametrize("seed", range(4))
def test_random_traffic(ctx, seed):              # noqa: F811
    """Copies under own and new keys, inside a gallery and between two, freed keys, dead rows, squeezes in place and into the
    other: after every step the rows of each key are found by key and in the whole gallery."""
    rng = np.random.default_rng(seed)
    cap = 6000
    a, b = Pair(ctx, 64, cap, 2500, seed=seed, nkeys=6), Pair(ctx, 64, cap, seed=seed + 50)
    a.k[:2500] = np.sort(a.k[:2500]) if seed % 2 else a.k[:2500]
    a.gal.write_f16(a.t[:2500], a.k[:2500], np.arange(2500))
    for step in range(14):
        src, dst = (a, b) if rng.random() < 0.6 else (b, a)
        what = ["copy", "copy", "own", "free", "kill", "squeeze", "into", "inside"][int(rng.integers(8))]
        if what in ("copy", "own"):
            first, counts = np.array([3, 700, 1300]), np.array([300, 1, 513])
            to = np.array([2600, 100, 3000]) + int(rng.integers(0, 500))
            keys = None if what == "own" else rng.integers(0, 9, 3).astype(np.int32)
            dst.gal.copy(first, to, counts, keys, source=src.gal)
            for i in range(3):
                f, t, n = first[i], to[i], counts[i]
                dst.t[t:t + n] = src.t[f:f + n]
                dst.k[t:t + n] = src.k[f:f + n] if keys is None else keys[i]
        elif what == "inside":
            rows = rng.permutation(2000)[:400]
            to = 4000 + rng.permutation(1900)[:400]
            src.gal.copy(rows, to)
            src.t[to], src.k[to] = src.t[rows], src.k[rows]
        elif what == "free":
            key = int(rng.integers(0, 6))
            assert src.gal.free_keys([key]) == int((src.k == key).sum())
            src.k[src.k == key] = DEAD
        elif what == "kill":
            rows = rng.permutation(3000)[:700]
            src.gal.tombstone(rows)
            src.k[rows] = DEAD
        elif what == "squeeze":
            assert src.gal.compact() == int((src.k >= 0).sum())
            squeeze_twin(src)
        else:
            assert src.gal.compact(dst.gal) == int((src.k >= 0).sum())
            squeeze_twin(src, dst)
        for p in (a, b):
            p.check()
            agree(p, 8, step)
    for p in (a, b):
        for key in range(9):
            assert p.gal.free_keys([key]) == int((p.k == key).sum()), key
        assert (p.gal.read_keys(0, cap) == DEAD).all()
        p.gal.close()


def test_lists_that_are_too_long_are_read_back(ctx):      # noqa: F811
    """Keys strewn over everything, and copies of single rows beyond what is mapped: the answers stay right."""
    n = 30000
    p, q = Pair(ctx, 64, n, seed=1), Pair(ctx, 64, 2 * n, seed=2)
    rng = np.random.default_rng(3)
    v = rng.standard_normal((n, 64)).astype(np.float32)
    p.t[:] = (v / np.linalg.norm(v, axis=1, keepdims=True)).astype(np.float16)
    p.k[:] = rng.integers(0, 20000, n)
    p.gal.write_f16(p.t, p.k, np.arange(n))
    order = rng.permutation(n)
    q.gal.copy(np.arange(n), order, source=p.gal)
    q.t[order], q.k[order] = p.t, p.k
    q.check_search()
    kill = rng.permutation(n)[:n // 2]
    q.gal.tombstone(kill)
    q.k[kill] = DEAD
    q.gal.compact()
    squeeze_twin(q)
    q.check()
    q.check_search()
    p.gal.compact(q.gal)
    squeeze_twin(p, q)
    q.check_search()
    for key in q.k[[0, 77, 29999]]:
        assert q.gal.free_keys([key]) == int((q.k == key).sum())
    p.gal.close()
    q.gal.close()
