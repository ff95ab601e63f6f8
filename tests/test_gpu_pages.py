"""Pages of a gallery on the GPU: copying, forking, reading, writing, freeing, squeezing and reprojecting rows, against a
numpy table that is changed by the same calls (rows move unchanged: everything is compared bit for bit)."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEAD = -1


@pytest.fixture(scope="module")
def ctx():
    from frhot.engine import Context
    c = Context(device=0, max_batch=2)
    yield c
    c.close()


def unit(rng, n, d):
    v = rng.standard_normal((n, d)).astype(np.float32)
    return (v / np.linalg.norm(v, axis=1, keepdims=True)).astype(np.float16)


class Pair:
    """A gallery and its numpy twin."""

    def __init__(self, ctx, dim, capacity, rows=0, seed=0, nkeys=3):
        from frhot.engine import Gallery
        rng = np.random.default_rng(seed)
        self.ctx, self.dim, self.cap = ctx, dim, capacity
        self.gal = Gallery(ctx, dim, capacity)
        self.t = np.zeros((capacity, dim), np.float16)
        self.k = np.full(capacity, DEAD, np.int32)
        if rows:
            self.t[:rows] = unit(rng, rows, dim)
            self.k[:rows] = rng.integers(0, nkeys, rows)
            self.gal.write_f16(self.t[:rows], self.k[:rows], np.arange(rows))

    def check(self, rows=None):
        rows = np.arange(self.cap) if rows is None else rows
        v, k = self.gal.read(rows)
        assert np.array_equal(k, self.k[rows])
        live = self.k[rows] != DEAD
        assert np.array_equal(v[live].view(np.uint16), self.t[rows][live].view(np.uint16))

    def check_search(self, nq=5, seed=1):
        """By key and whole: the rows the twin's table gives."""
        rng = np.random.default_rng(seed)
        live = np.flatnonzero(self.k >= 0)
        if live.size == 0:
            return
        at = rng.choice(live, nq)
        q = self.t[at].astype(np.float32)
        for mode in (self.gal.SEARCH_BY_KEY, self.gal.SEARCH_WHOLE):
            self.gal.search_mode(mode)
            s, r = self.gal.search(q, self.k[at], 5)
            for i in range(nq):
                mine = live[self.k[live] == self.k[at[i]]]
                sc = self.t[mine].astype(np.float64) @ (q[i].astype(np.float64) / np.linalg.norm(q[i].astype(np.float64)))
                assert r[i, 0] >= 0 and self.k[r[i, 0]] == self.k[at[i]]
                assert abs(s[i, 0] - sc.max()) <= 2e-3
                got = set(int(v) for v in r[i] if v >= 0)
                assert len(got) == min(5, mine.size) and got <= set(mine.tolist())
        self.gal.search_mode(self.gal.SEARCH_AUTO)

    def close(self):
        self.gal.close()


def runs(rng, lo, hi, n):
    """n disjoint runs inside [lo, hi)"""
    edge = np.sort(rng.choice(np.arange(lo, hi + 1), 2 * n, replace=False))
    return edge[::2].astype(np.int64), (edge[1::2] - edge[::2]).astype(np.int32)


def rows_of(first, counts):
    return np.concatenate([np.arange(f, f + c) for f, c in zip(first, counts)])


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("dim", [64, 128, 448, 512, 4096, 8192])
@pytest.mark.parametrize("n", [1, 63, 64, 65, 255, 256, 257, 700])
def test_one_run(ctx, dim, n):
    """Every alignment of a run's start against the pages' edges."""
    for src, dst in ((0, 701), (3, 1000), (255, 1023), (256, 1280), (100, 767)):
        p = Pair(ctx, dim, 2100, 1024, seed=n)
        n = min(n, 1024 - src, dst - src)
        p.gal.copy([src], [dst], [n], 9)
        p.t[dst:dst + n], p.k[dst:dst + n] = p.t[src:src + n].copy(), 9
        p.check()
        p.close()
        if dim >= 4096:
            break


@pytest.mark.parametrize("dim", [64, 512])
@pytest.mark.parametrize("keep", [False, True])
def test_many_runs(ctx, dim, keep):
    """Odd runs in an order of their own, within one gallery and from another; with new keys and with the rows' own."""
    rng = np.random.default_rng(dim + keep)
    for other in (False, True):
        a = Pair(ctx, dim, 6000, 2500, seed=2)
        b = Pair(ctx, dim, 6000, 1100, seed=3) if other else a
        a.k[40:90] = DEAD
        a.gal.tombstone(np.arange(40, 90))
        first, counts = runs(rng, 0, 2500, 60)
        to = 2600 + np.concatenate([[0], np.cumsum(counts[:-1] + rng.integers(0, 5, 59))])
        perm = rng.permutation(60)
        first, counts, to = first[perm], counts[perm], to[perm]
        keys = None if keep else rng.integers(5, 9, 60).astype(np.int32)
        b.gal.copy(first, to, counts, keys, source=a.gal)
        s, d = rows_of(first, counts), rows_of(to, counts)
        b.t[d] = a.t[s]
        b.k[d] = a.k[s] if keep else np.repeat(keys, counts)
        b.check()
        b.check_search()
        a.check()
        b.close()
        if other:
            a.close()


def test_single_rows(ctx):
    """counts None: every entry is one row; a row may be a source more than once."""
    p = Pair(ctx, 192, 1000, 400)
    src = np.array([5, 5, 399, 0, 17, 5])
    dst = np.array([999, 500, 401, 777, 640, 512])
    p.gal.copy(src, dst, keys=[4, 5, 6, 4, 5, 6])
    p.t[dst], p.k[dst] = p.t[src], [4, 5, 6, 4, 5, 6]
    p.check()
    p.check_search()
    p.close()


@pytest.mark.parametrize("dim", [64, 512, 4096])
def test_read_and_write(ctx, dim):
    rng = np.random.default_rng(dim)
    p = Pair(ctx, dim, 2000, 1500)
    first, counts = runs(rng, 0, 2000, 25)
    rng.shuffle(first_counts := list(zip(first, counts)))
    first, counts = map(np.array, zip(*first_counts))
    at = rows_of(first, counts)
    out = torch.full((at.size + 2, dim), 7.0, dtype=torch.float16, device="cuda")
    keys = torch.full((at.size + 2,), 7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    p.gal.read_dev(first, counts, out.data_ptr(), keys.data_ptr())
    ctx.sync()
    assert np.array_equal(keys[:-2].cpu().numpy(), p.k[at]) and (keys[-2:] == 7).all() and (out[-2:] == 7).all()
    live = p.k[at] >= 0
    assert np.array_equal(out[:-2].cpu().numpy()[live], p.t[at][live])
    out2 = torch.empty_like(out)
    p.gal.read_dev(first, counts, out2.data_ptr())                      # without the keys
    new = unit(rng, at.size, dim)
    nd = dev(new)
    run_keys = rng.integers(-1, 4, first.size).astype(np.int32)         # dead ones among them
    torch.cuda.synchronize()
    p.gal.write_dev(nd.data_ptr(), first, counts, run_keys)
    ctx.sync()
    p.t[at], p.k[at] = new, np.repeat(run_keys, counts)
    p.check()
    p.check_search()
    p.close()


def test_forked_collection_is_searched_and_dropped(ctx):
    p = Pair(ctx, 512, 4000, 1500, nkeys=2)
    mine = np.flatnonzero(p.k == 1)
    from frhot.engine import runs_of
    first, counts = runs_of(mine)
    to = 2000 + np.concatenate([[0], np.cumsum(counts[:-1])])
    p.gal.copy(first, to, counts, 8)
    d = rows_of(to, counts)
    p.t[d], p.k[d] = p.t[mine], 8
    p.check_search(12)
    assert p.gal.free_keys([1]) == mine.size
    p.k[mine] = DEAD
    p.check()
    p.check_search(12)
    assert p.gal.free_keys([1]) == 0
    assert p.gal.free_keys([8, 0, 8, 55]) == int((p.k >= 0).sum())
    p.k[:] = DEAD
    p.check()
    s, r = p.gal.search(p.t[:3].astype(np.float32), None, 5)
    assert (r == -1).all()
    p.close()


def test_free_in_a_gallery_without_lists(ctx):
    """Keys strewn over every tile (the per-key tile lists were given up): every tile is looked at."""
    from frhot.engine import Gallery
    n = 256 * 5000
    gal = Gallery(ctx, 64, n)
    gal.fill_synthetic(5, 0, n, nkeys=3000)
    keys = np.empty(n, np.int32)
    _, keys[:1000] = gal.read(np.arange(1000))
    want = int(keys[3])
    freed = gal.free_keys([want])
    assert freed > 0
    _, k = gal.read(np.arange(1000))
    gone = keys[:1000] == want
    assert (k[gone] == DEAD).all() and np.array_equal(k[~gone], keys[:1000][~gone])
    assert gal.free_keys([want]) == 0
    gal.close()


@pytest.mark.parametrize("dim", [64, 512, 4096])
@pytest.mark.parametrize("rows,dead", [(1, 0.0), (1, 1.0), (256, 0.5), (257, 0.02), (1000, 0.0), (1000, 1.0), (1003, 0.97), (5000, 0.3)])
@pytest.mark.parametrize("inplace", [False, True])
def test_compact(ctx, dim, rows, dead, inplace):
    rng = np.random.default_rng(rows + int(dead * 100))
    p = Pair(ctx, dim, 5300, rows, seed=4)
    gone = np.flatnonzero(rng.random(rows) < dead) if dead < 1 else np.arange(rows)
    if gone.size:
        p.gal.tombstone(gone)
        p.k[gone] = DEAD
    to = p if inplace else Pair(ctx, dim, 5300, 3000, seed=5)       # what the target held goes
    place = torch.full((rows + 1,), 77, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    live = p.gal.compact(None if inplace else to.gal, place.data_ptr())
    alive = np.flatnonzero(p.k[:rows] >= 0)
    assert live == alive.size == to.gal.rows
    want = np.full(rows, -1, np.int64)
    want[alive] = np.arange(alive.size)
    assert np.array_equal(place[:rows].cpu().numpy(), want) and place[rows] == 77
    t, k = p.t[alive].copy(), p.k[alive].copy()
    if not inplace:
        p.check()
    to.t[:live], to.k[:] = t, DEAD
    to.k[:live] = k
    to.check()
    to.check_search()
    # and it takes new rows behind the squeezed ones
    new = unit(rng, 2, dim)
    to.gal.write_f16(new, [6, 6], [live, live + 1])
    to.t[live:live + 2], to.k[live:live + 2] = new, 6
    to.check_search()
    to.close()
    if not inplace:
        p.close()


def test_compact_keeps_the_order_of_equal_scores(ctx):
    from frhot.engine import Gallery
    gal = Gallery(ctx, 64, 2000)
    gal.fill_synthetic(3, 0, 2000, dup_every=2)                     # every second row equals the one before it
    gone = np.arange(0, 2000, 7)
    gal.tombstone(gone)
    q = gal.read(np.arange(1, 2000, 211))[0].astype(np.float32)
    s0, r0 = gal.search(q, None, 10)
    live = gal.compact()
    s1, r1 = gal.search(q, None, 10)
    alive = np.setdiff1d(np.arange(2000), gone)
    assert live == alive.size and np.array_equal(s0, s1) and np.array_equal(alive[r1], r0)
    gal.close()


def test_compact_into_a_smaller_gallery(ctx):
    from frhot import FrhotError
    p = Pair(ctx, 128, 2000, 1800)
    to = Pair(ctx, 128, 900, 100)
    with pytest.raises(FrhotError) as e:
        p.gal.compact(to.gal)
    assert e.value.code == -4
    to.check()
    p.gal.tombstone(np.arange(0, 1000))
    p.k[:1000] = DEAD
    assert p.gal.compact(to.gal) == 800
    to.t[:800], to.k[:800] = p.t[1000:1800], p.k[1000:1800]
    to.check()
    to.close()
    p.close()


def test_large_gallery_past_32_bit_offsets(ctx):
    """Rows whose byte offsets pass 2^32: copied there, read back from there, squeezed."""
    from frhot.engine import Gallery
    cap, dim = 1_400_000, 4096                                      # 11.5 GB
    gal = Gallery(ctx, dim, cap)
    rng = np.random.default_rng(0)
    v = unit(rng, 300, dim)
    gal.write_f16(v, 1, np.arange(300))
    gal.copy([0], [cap - 300], [300], 2)
    gal.copy([cap - 300], [600_001], [300], 3)
    for at, key in ((cap - 300, 2), (600_001, 3)):
        got, k = gal.read(np.arange(at, at + 300))
        assert np.array_equal(got, v) and (k == key).all()
    out = torch.empty(300, dim, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    gal.read_dev([cap - 300], [300], out.data_ptr())
    ctx.sync()
    assert np.array_equal(out.cpu().numpy(), v)
    small = Gallery(ctx, dim, 1000)
    assert gal.compact(small) == 900
    got, k = small.read(np.arange(900))
    assert np.array_equal(got, np.concatenate([v, v, v])) and np.array_equal(k, np.repeat([1, 3, 2], 300))
    assert gal.free_keys([2]) == 300
    small.close()
    gal.close()


def test_refusals(ctx):
    from frhot import FrhotError
    from frhot.engine import Context, Gallery
    p, q = Pair(ctx, 128, 1000, 500), Pair(ctx, 64, 1000, 10)

    def refused(code, f, *a, **k):
        with pytest.raises(FrhotError) as e:
            f(*a, **k)
        assert e.value.code == code, e.value
    g = p.gal
    refused(-1, g.copy, [], [])
    refused(-1, g.copy, [0], [600], [0])
    refused(-1, g.copy, [0], [600], [-3])
    refused(-4, g.copy, [0], [901], [100])
    refused(-4, g.copy, [901], [0], [100])
    refused(-4, g.copy, [-1], [600], [10])
    refused(-4, g.copy, [2 ** 62], [600], [10])
    refused(-1, g.copy, [0], [600], [10], -1)
    refused(-1, g.copy, [0], [5], [10], 3)                              # read and written
    refused(-1, g.copy, [0, 600], [600, 700], [10, 10], 3)              # a copy of what the call itself writes
    refused(-1, g.copy, [0, 100], [600, 605], [10, 10], 3)              # a destination twice
    refused(-1, g.copy, [0, 100], [605, 600], [10, 10], 3)
    refused(-1, g.copy, [0], [600], [10], 3, source=q.gal)              # other dimension
    c2 = Context(device=0, max_batch=1)
    g2 = Gallery(c2, 128, 100)
    refused(-1, g.copy, [0], [600], [10], 3, source=g2)
    refused(-1, g.compact, g2)
    refused(-1, g.compact, q.gal)
    buf = torch.zeros(64, 128, dtype=torch.float16, device="cuda")
    refused(-1, g.read_dev, [0], [4], 0)
    refused(-1, g.read_dev, [0], [4], buf.data_ptr() + 2)
    refused(-4, g.read_dev, [999], [2], buf.data_ptr())
    refused(-1, g.write_dev, buf.data_ptr() + 8, [0], [4], 1)
    refused(-1, g.write_dev, buf.data_ptr(), [0], [4], -2)
    refused(-1, g.write_dev, buf.data_ptr(), [0, 2], [4, 4], 1)
    refused(-4, g.write_dev, buf.data_ptr(), [998], [4], 1)
    refused(-1, g.free_keys, [])
    refused(-1, g.free_keys, [3, -1])
    refused(-1, g.compact, None, buf.data_ptr() + 4)
    assert ctx._lib.frhot_gallery_copy(None, None, None, None, None, None, 1) == -1
    assert ctx._lib.frhot_gallery_compact(None, None, None, None) == -1
    with pytest.raises(ValueError):
        g.copy([0, 1], [5], [1, 1])
    with pytest.raises(ValueError):
        g.copy([0, 1], [5, 6], [1])
    p.check()
    # row lists under graph capture
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c3 = Context(device=0, max_batch=1, stream=s.cuda_stream)
        g3 = Gallery(c3, 128, 100)
        gr = torch.cuda.CUDAGraph()
        gr.capture_begin()
        refused(-3, g3.read_dev, [0], [4], buf.data_ptr())
        refused(-3, g3.copy, [0], [50], [4], 1)
        gr.capture_end()
        s.synchronize()
        g3.close()
        c3.close()
    g2.close()
    c2.close()
    p.close()
    q.close()


def test_threads_copy_while_others_search(ctx):
    import threading
    p = Pair(ctx, 256, 20000, 2000, nkeys=1)
    want = p.gal.search(p.t[:8].astype(np.float32), [0] * 8, 5)
    errors = []

    def copier(j):
        try:
            for i in range(10):
                p.gal.copy([0], [3000 + (j * 10 + i) * 600], [500], 10 + j)
        except Exception as e:      # pragma: no cover
            errors.append(e)

    def searcher():
        try:
            for _ in range(20):
                s, r = p.gal.search(p.t[:8].astype(np.float32), [0] * 8, 5)
                assert np.array_equal(s, want[0]) and np.array_equal(r, want[1])
        except Exception as e:      # pragma: no cover
            errors.append(e)

    ts = [threading.Thread(target=copier, args=(j,)) for j in range(2)] + [threading.Thread(target=searcher) for _ in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not errors
    for j in range(2):
        for i in range(10):
            at = 3000 + (j * 10 + i) * 600
            p.t[at:at + 500], p.k[at:at + 500] = p.t[:500], 10 + j
    p.check()
    p.close()


# --------------------------------------------------------------------------------------- with a head
@pytest.mark.parametrize("rows,dims,acts,res", [(1, [128, 64], ["none"], [0]), (700, [512, 192, 64], ["gelu", "none"], [0, 0]),
                                                (3001, [256, 256], ["silu"], [1]), (5000, [64, 1024], ["relu"], [0])])
def test_reproject(ctx, rows, dims, acts, res):
    from frhot.engine import Head
    from test_gpu_heads import head64, head_layers, linear_of
    p = Pair(ctx, dims[0], 5100, rows, seed=6)
    if rows > 10:
        p.gal.tombstone(np.arange(3, 9))
        p.k[3:9] = DEAD
    to = Pair(ctx, dims[-1], 5200, 5150, seed=7)
    layers = head_layers(dims, acts, res, seed=rows)
    lins = [linear_of(ctx, w, b, "f16") for w, b, _, _ in layers]
    head = Head(ctx, [(l, a, r) for l, (_, _, a, r) in zip(lins, layers)])
    p.gal.reproject(head, to.gal)
    ctx.sync()
    v, k = to.gal.read(np.arange(5200))
    want = np.full(5200, DEAD, np.int32)
    want[:rows] = p.k[:rows]
    assert np.array_equal(k, want) and to.gal.rows == rows
    live = np.flatnonzero(want >= 0)
    y, tol = head64(torch.from_numpy(p.t[live]), layers)
    assert ((torch.from_numpy(v[live]).double() - y).abs() <= tol).all()
    to.t[:], to.k[:] = v, want
    to.check_search()
    p.check()
    head.close()
    [l.close() for l in lins]
    to.close()
    p.close()


def test_reproject_longer_than_one_pass(ctx):
    """More rows than a head takes at once: the same bits as the rows taken out and sent through by themselves."""
    from frhot.engine import Gallery, Head
    from test_gpu_heads import head_layers, linear_of
    n = 40000
    gal, to = Gallery(ctx, 128, n), Gallery(ctx, 64, n)
    gal.fill_synthetic(4, 0, n, nkeys=5)
    layers = head_layers([128, 64], ["none"], [0])
    lin = linear_of(ctx, layers[0][0], layers[0][1], "f16")
    head = Head(ctx, [(lin, "none", False)])
    gal.reproject(head, to)
    x, out = torch.empty(n, 128, dtype=torch.float16, device="cuda"), torch.empty(n, 64, dtype=torch.float16, device="cuda")
    got, keys = torch.empty_like(out), torch.empty(n, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    gal.read_dev([0], [n], x.data_ptr())
    head.run_dev(x.data_ptr(), n, out.data_ptr())
    to.read_dev([0], [n], got.data_ptr(), keys.data_ptr())
    ctx.sync()
    assert torch.equal(got, out)
    assert np.array_equal(keys.cpu().numpy(), gal.read(np.arange(n))[1])
    head.close()
    lin.close()
    gal.close()
    to.close()


def test_reproject_refusals(ctx):
    from frhot import FrhotError
    from frhot.engine import Gallery, Head, Linear
    lin = Linear(ctx, np.zeros((64, 128), np.float16))
    head = Head(ctx, [(lin, "none", False)])
    a, b, small = Gallery(ctx, 128, 300), Gallery(ctx, 64, 300), Gallery(ctx, 64, 100)
    a.fill_synthetic(1, 0, 200)
    for src, dst, code in ((a, a, -1), (b, b, -1), (b, a, -1), (a, small, -4)):
        with pytest.raises(FrhotError) as e:
            src.reproject(head, dst)
        assert e.value.code == code
    assert ctx._lib.frhot_gallery_reproject(a.handle, None, b.handle) == -1
    b.fill_synthetic(1, 0, 250)
    empty = Gallery(ctx, 128, 10)
    empty.reproject(head, b)                                            # no rows: everything b held dies
    ctx.sync()
    assert b.rows == 0 and (b.read(np.arange(300))[1] == DEAD).all()
    head.close()
    lin.close()
    for g in (a, b, small, empty):
        g.close()


# ------------------------------------------------------------------------- as a service uses them
def test_service_with_a_head_copies_drops_and_squeezes(gpu_ctx):
    """Faces enrolled through a head into a 256-wide gallery, recognised from their crops, the collection forked, the
    original dropped, the gallery squeezed: every step answers for the same people."""
    from frhot import synth
    from frhot.engine import Head
    from frhot.gallery_service import GalleryService
    from test_gpu_heads import head_layers, linear_of
    crops = synth.crops(seed=9, n=8, lo=90, hi=180)
    emb = gpu_ctx.embed(crops, gamma=True)
    # a layer that spreads the synthetic network's similar faces: random directions around their mean
    g = torch.Generator().manual_seed(3)
    w = (torch.randn(256, 4096, generator=g) / 8).half()
    mean = torch.from_numpy(emb).double().mean(0)
    lin = linear_of(gpu_ctx, w, (-(w.double() @ mean)).float(), "f16")
    head = Head(gpu_ctx, [(lin, "none", False)])
    rows = head.apply(emb)
    x16 = torch.from_numpy(emb).half()
    y = x16.double() @ w.double().t() - (w.double() @ mean).float().double()
    y = y / y.norm(dim=1, keepdim=True)
    assert (torch.from_numpy(rows).double() - y).abs().max() <= 2e-3
    svc = GalleryService(gpu_ctx, capacity=2000, head=head)
    try:
        assert svc.dim == 256
        svc.create_collection("7_Employees")
        rng = np.random.default_rng(1)
        for i in range(300):                                    # strangers around them, some of whom leave again
            svc.insert_point("7_Employees", rng.standard_normal(256).astype(np.float32), f"s{i}", "x", 7)
        for i, e in enumerate(emb):
            assert svc.insert_point("7_Employees", e, f"p{i}", f"n{i}", 7)[0] == 201
        for i in range(0, 300, 2):
            svc.delete_point("7_Employees", f"s{i}")

        def who(col):
            return [content["data"][0][1]["id"] if content["data"] else None
                    for _s, content, _e in svc.recognise_points([(col, c, 7) for c in crops])]
        want = [f"p{i}" for i in range(8)]
        assert who("7_Employees") == want
        assert svc.copy_collection("7_Employees", "8_Employees")[1]["points"] == 158
        assert who("8_Employees") == want
        assert svc.delete_collection("7_Employees")[0] == 200
        assert svc.recognise_points([("7_Employees", crops[0], 7)])[0][0] == 404
        assert who("8_Employees") == want
        assert svc.compact() == (200, {"message": "Gallery compacted", "points": 158})
        assert svc.gallery.rows == 158 and who("8_Employees") == want
        for i in range(8):
            assert svc.search_point("8_Employees", emb[i], 7)[1]["data"][0][1]["id"] == f"p{i}"
        assert svc.insert_point("8_Employees", emb[0] * 2, "again", "n", 7)[0] == 201
        assert svc.gallery.rows == 159
    finally:
        gpu_ctx.set_head(None)
        svc.close()
        head.close()
        lin.close()


def test_squeezing_while_others_recognise(gpu_ctx):
    """Threads that search while collections are dropped and the gallery squeezed: every answer names the asked person."""
    import threading
    from frhot.gallery_service import GalleryService
    svc = GalleryService(gpu_ctx, capacity=6000, dim=512)
    rng = np.random.default_rng(2)
    vecs = rng.standard_normal((60, 512)).astype(np.float32)
    svc.create_collection("1_Employees")
    for k in range(4):
        svc.create_collection(f"{k + 2}_Customers")
        for i in range(150):
            svc.insert_point(f"{k + 2}_Customers", rng.standard_normal(512).astype(np.float32), f"c{i}", "n", 1)
        for i in range(15 * k, 15 * k + 15):
            svc.insert_point("1_Employees", vecs[i], f"p{i}", "n", 1)
    errors, stop = [], threading.Event()

    def ask(j):
        r = np.random.default_rng(j)
        try:
            while not stop.is_set():
                i = int(r.integers(60))
                status, content = svc.search_point("1_Employees", vecs[i], 1)
                assert status == 200 and content["data"][0][1]["id"] == f"p{i}", content
        except Exception as e:
            errors.append(e)
    ts = [threading.Thread(target=ask, args=(j,)) for j in range(3)]
    [t.start() for t in ts]
    for k in range(4):
        assert svc.delete_collection(f"{k + 2}_Customers")[0] == 200
        assert svc.compact()[0] == 200
    stop.set()
    [t.join() for t in ts]
    assert not errors, errors[0]
    assert svc.gallery.rows == 60
    svc.close()


def test_more_runs_than_a_launch_has_threads():
    """2^24 + 5 runs of one row: several launches."""
    from frhot.engine import Context, Gallery
    ctx = Context(device=0, max_batch=1)                    # (its page-locked run list of 600 MB goes with it)
    n = (1 << 24) + 5
    gal = Gallery(ctx, 64, 2 * n)
    gen = torch.Generator("cuda").manual_seed(3)
    src = torch.randint(-30000, 30000, (2 * n, 64), generator=gen, device="cuda", dtype=torch.int16)
    out = torch.empty(n, 64, dtype=torch.int16, device="cuda")
    keys = torch.empty(n, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    gal.write_dev(src.data_ptr(), [0, n], [n, n], [4, 9])
    gal.read_dev(2 * np.arange(n, dtype=np.int64), None, out.data_ptr(), keys.data_ptr())
    ctx.sync()
    assert torch.equal(out, src[::2])
    assert torch.equal(keys, torch.where(2 * torch.arange(n, device="cuda") < n, 4, 9).int())
    gal.close()
    ctx.close()
    del src, out, keys
    torch.cuda.empty_cache()


def test_refused_under_capture():
    """Calls that wait or change the host's tables leave a capture as they found it: it goes on and replays."""
    from frhot.engine import Context, Gallery, Head, Linear
    from frhot._lib import FrhotError
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = Context(device=0, max_batch=1, stream=s.cuda_stream)
        lin = Linear(c, np.eye(64, dtype=np.float32))
        head = Head(c, [(lin, "none", False)])
        g, h = Gallery(c, 64, 600), Gallery(c, 64, 600)
        buf = torch.randn(600, 64, device="cuda").half()
        out = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
        g.write_dev(buf.data_ptr(), [0, 300], [300, 300], [1, 2])
        h.copy([0], [0], [600], source=g)                   # (own keys: the key lists of h are rebuilt when next needed)
        s.synchronize()
        gr = torch.cuda.CUDAGraph()
        gr.capture_begin()
        for call in (lambda: g.free_keys([1]), lambda: h.free_keys([1]), lambda: g.compact(), lambda: g.compact(h),
                     lambda: g.reproject(head, h), lambda: g.copy([0], [300], [4], 1), lambda: g.read_dev([0], [4], out.data_ptr()),
                     lambda: g.write_dev(buf.data_ptr(), [0], [4], 1), lambda: head.apply(np.ones((1, 64), np.float32))):
            with pytest.raises(FrhotError) as e:
                call()
            assert e.value.code == -3
        head.run_dev(buf.data_ptr(), 4, out.data_ptr())
        gr.capture_end()
        for _ in range(3):
            out.zero_()
            gr.replay()
            s.synchronize()
            want = buf[:4].double()
            assert ((out.double() - want / want.norm(dim=1, keepdim=True)).abs() <= 2.0 ** -10).all()
        assert (g.rows, h.rows) == (600, 600)
        assert h.free_keys([1]) == 300 and g.free_keys([1, 2]) == 600 and g.compact() == 0
        g.close(), h.close(), head.close(), lin.close(), c.close()


def test_read_refuses_keys_off_their_alignment(ctx):
    from frhot._lib import FrhotError
    p = Pair(ctx, 64, 300, 20)
    buf = torch.empty(16, 64, dtype=torch.float16, device="cuda")
    k = torch.empty(16, dtype=torch.int32, device="cuda")
    with pytest.raises(FrhotError):
        p.gal.read_dev([0], [4], buf.data_ptr(), k.data_ptr() + 2)
    p.gal.close()


@pytest.mark.parametrize("dim", [64, 128, 192])
def test_many_rows_of_few_components_in_odd_runs(ctx, dim):
    """Long items: runs of one to 3000 rows, shuffled, between and inside pages; keys kept, then given."""
    rng = np.random.default_rng(dim)
    n, cap = 90001, 200000
    p, q = Pair(ctx, dim, n, n, seed=dim), Pair(ctx, dim, cap)
    edge = np.unique(np.concatenate([[0, 1, 255, 256, 257, 600, 3600, n], rng.integers(1, n, 150)]))
    first, counts = edge[:-1], np.diff(edge)
    order = rng.permutation(len(first))
    dst = np.zeros(len(first), np.int64)
    at = 77
    for i in order:
        dst[i] = at
        at += counts[i] + int(rng.integers(0, 300))
    keys = rng.integers(0, 5, len(first)).astype(np.int32)
    for k in (None, keys):
        q.gal.copy(first, dst, counts, k, source=p.gal)
        for i in range(len(first)):
            s, d, c = first[i], dst[i], counts[i]
            q.t[d:d + c] = p.t[s:s + c]
            q.k[d:d + c] = p.k[s:s + c] if k is None else k[i]
        q.check()
        q.check_search()
    p.gal.close()
    q.gal.close()


def test_lists_of_any_kind(ctx):
    """Row lists as lists, ranges, other integer types, strided, read-only: the same rows move."""
    p = Pair(ctx, 64, 600, 300, seed=4)
    first = np.array([0, 9, 100], np.int64)
    ro = first.copy()
    ro.setflags(write=False)
    at = 300
    for rows in (first, first.tolist(), first.astype(np.int32), first.astype(np.uint16), np.repeat(first, 2)[::2], ro, first.astype(">i8")):
        p.gal.copy(rows, [at, at + 10, at + 20], [5, 1, 7], 2)
        for s, d, c in zip(first, (at, at + 10, at + 20), (5, 1, 7)):
            p.t[d:d + c], p.k[d:d + c] = p.t[s:s + c], 2
        at += 30
    p.check()
    n = int((p.k == 2).sum())
    assert p.gal.free_keys(ro[:0].tolist() + [2]) == n and p.gal.free_keys(np.array([2], ">i4")) == 0
    p.k[p.k == 2] = DEAD
    p.check()
    p.gal.close()
