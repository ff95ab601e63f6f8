"""Host side of the gallery's pages and of descriptor heads: the service's copy / delete / squeeze over a numpy stand-in,
argument checks that need no device, the bfloat16 rounding of weights."""
import ctypes as C
import threading

import numpy as np
import pytest

from fakes import NumpyGallery


class PagedGallery(NumpyGallery):
    """NumpyGallery with the page calls of frhot.engine.Gallery."""

    @property
    def rows(self):
        return self.nrows

    def copy(self, src_rows, dst_rows, counts=None, keys=None, source=None):
        for i, (s, d) in enumerate(zip(src_rows, dst_rows)):
            n = 1 if counts is None else int(counts[i])
            assert (self.keys[d:d + n] == -1).all(), "a live row would be overwritten"
            self.g[d:d + n] = self.g[s:s + n].copy()
            self.keys[d:d + n] = self.keys[s:s + n] if keys is None else keys[i]
            self.nrows = max(self.nrows, d + n)

    def free_keys(self, keys):
        hit = np.isin(self.keys, keys)
        self.keys[hit] = -1
        return int(hit.sum())

    def compact(self, into=None, new_rows_dev=None):
        live = np.flatnonzero(self.keys >= 0)
        g, k = self.g[live].copy(), self.keys[live].copy()
        self.keys[:] = -1
        self.g[:len(live)], self.keys[:len(live)] = g, k
        self.nrows = len(live)
        return len(live)


def service(dim=32, capacity=3000, **kw):
    from frhot.gallery_service import GalleryService
    return GalleryService(None, capacity=capacity, dim=dim, gallery=PagedGallery(dim, capacity), **kw)


def enrol(svc, rng, col, n, stores=(1, 2), start=0):
    svc.create_collection(col)
    vecs = {}
    for i in range(start, start + n):
        v = rng.standard_normal(svc.dim).astype(np.float32)
        st = stores[i % len(stores)]
        assert svc.insert_point(col, v, f"p{i}", f"name{i}", st, uid=f"{col}-{i}")[0] == 201
        vecs[i] = (v, st)
    return vecs


def found(svc, col, vec, store):
    status, content = svc.search_point(col, vec, store)
    assert status == 200
    return content["data"][0][1]["id"] if content["data"] else None


def check_tables(svc):
    """Rows, keys and allocator agree: every point's row is live under its key, no row is handed out twice."""
    for r, p in svc._points.items():
        assert svc.gallery.keys[r] == svc._keys[(p["collection"], p["payload"]["store_id"])]
        assert r in svc._by_id[(p["collection"], p["payload"]["id"])]
    assert int((svc.gallery.keys >= 0).sum()) == len(svc._points)
    free = [r for v in svc._rows._free.values() for r in v]
    assert len(free) == len(set(free)) and not set(free) & set(svc._points)
    assert svc._rows.free_count() == svc.capacity - len(svc._points)


def test_copy_delete_and_compact_on_random_traffic():
    rng = np.random.default_rng(3)
    svc = service()
    a = enrol(svc, rng, "A_Employees", 300)
    b = enrol(svc, rng, "B_Employees", 200, stores=(1, 2, 3))
    for i in range(0, 300, 3):
        svc.delete_point("A_Employees", f"p{i}")
        del a[i]
    assert svc.copy_collection("A_Employees", "C_Employees") == (201, {"message": "Collection copied", "points": len(a)})
    check_tables(svc)
    for i in list(a)[:20]:
        v, st = a[i]
        assert found(svc, "C_Employees", v, st) == f"p{i}" == found(svc, "A_Employees", v, st)
        assert found(svc, "C_Employees", v, 3 - st) != f"p{i}"
    uids = [p["uid"] for p in svc._points.values()]
    assert len(set(uids)) == len(uids)
    # the copy lives by itself
    assert svc.delete_collection("A_Employees") == (200, {"message": "Collection deleted"})
    check_tables(svc)
    assert not svc.collection_exists("A_Employees") and svc.point_count("C_Employees") == len(a)
    v, st = a[1]
    assert svc.search_point("A_Employees", v, st)[0] == 404 and found(svc, "C_Employees", v, st) == "p1"
    before = svc.gallery.rows
    assert svc.compact() == (200, {"message": "Gallery compacted", "points": len(a) + len(b)})
    assert svc.gallery.rows == len(a) + len(b) < before
    check_tables(svc)
    for i in list(a)[::15]:
        assert found(svc, "C_Employees", *a[i]) == f"p{i}"
    for i in list(b)[::15]:
        assert found(svc, "B_Employees", *b[i]) == f"p{i}"
    # and goes on: new points, deletions, the same again
    enrol(svc, rng, "D_Customers", 400, stores=(9,))
    svc.delete_collection("B_Employees")
    svc.compact()
    check_tables(svc)
    assert svc.point_count("D_Customers") == 400 and svc.point_count("C_Employees") == len(a)


def test_eviction_continues_in_a_copy():
    """The ten-faces limit drops the oldest of the copied faces first (app.py:207-240)."""
    rng = np.random.default_rng(1)
    svc = service()
    svc.create_collection("A_Employees")
    vs = [rng.standard_normal(32).astype(np.float32) for _ in range(12)]
    for i in range(9):
        svc.insert_point("A_Employees", vs[i], "p", "n", 1, time_created=f"2025/01/0{i + 1} 00:00:00")
    svc.copy_collection("A_Employees", "B_Employees")
    for i in (9, 10):
        svc.insert_point("B_Employees", vs[i], "p", "n", 1, time_created=f"2025/02/0{i - 8} 00:00:00")
    times = sorted(p["payload"]["time_created"] for p in svc._points.values() if p["collection"] == "B_Employees")
    assert len(times) == 10 and times[0] == "2025/01/02 00:00:00"
    assert svc.point_count("A_Employees") == 9


def test_copy_refusals_leave_everything_as_it_was():
    rng = np.random.default_rng(2)
    svc = service(capacity=512)
    enrol(svc, rng, "A_Employees", 200, stores=(1,))
    enrol(svc, rng, "B_Employees", 10, stores=(1,))
    for bad in ((None, "X_Employees"), ("", "X_Employees"), ("A_Employees", ""), ("Z_Employees", "X_Employees"), ("A_Employees", "A_Employees")):
        assert svc.copy_collection(*bad)[0] == 404
    assert svc.copy_collection("A_Employees", "B_Employees")[0] == 409
    assert svc.copy_collection("A_Employees", "C_Employees")[0] == 201
    assert svc.copy_collection("A_Employees", "D_Employees")[0] == 404          # no room
    assert not svc.collection_exists("D_Employees")
    check_tables(svc)
    free = svc._rows.free_count()
    svc.delete_collection("C_Employees")

    def broken(*a, **k):
        raise RuntimeError("device")
    svc.gallery.copy, plain = broken, svc.gallery.copy
    assert svc.copy_collection("A_Employees", "D_Employees") == (404, {"message": "device"})
    svc.gallery.copy = plain
    assert svc._rows.free_count() == free + 200 and not svc.collection_exists("D_Employees")
    check_tables(svc)
    for bad in (None, "", "Z_Employees"):
        assert svc.delete_collection(bad)[0] == 404


def test_compact_of_an_empty_and_of_a_full_gallery():
    rng = np.random.default_rng(4)
    svc = service(capacity=300)
    assert svc.compact() == (200, {"message": "Gallery compacted", "points": 0})
    enrol(svc, rng, "A_Employees", 300, stores=(1,))
    assert svc._rows.free_count() == 0
    assert svc.compact()[1]["points"] == 300
    check_tables(svc)
    svc.delete_collection("A_Employees")
    assert svc.compact()[1]["points"] == 0 and svc._rows.free_count() == 300
    check_tables(svc)


def test_compact_drops_rows_that_the_table_does_not_know():
    """A row left alive by a failed write does not shift the others' numbers."""
    rng = np.random.default_rng(5)
    svc = service()
    vs = enrol(svc, rng, "A_Employees", 20, stores=(1,))
    svc.gallery.keys[30], svc.gallery.nrows = 0, 31
    svc.delete_point("A_Employees", "p3")
    assert svc.compact() == (200, {"message": "Gallery compacted", "points": 19})
    check_tables(svc)
    assert found(svc, "A_Employees", *vs[19]) == "p19"


def test_search_in_flight_while_rows_move():
    """A search that was on the device while the gallery was squeezed is answered from the new row numbers."""
    rng = np.random.default_rng(6)
    svc = service()
    vs = enrol(svc, rng, "A_Employees", 50, stores=(1,))
    started, go = threading.Event(), threading.Event()
    plain = svc.gallery.search

    def slow(q, qkeys=None, k=5):
        out = plain(q, qkeys, k)
        if not started.is_set():
            started.set()
            assert go.wait(10)
        return out
    svc.gallery.search = slow
    answer = {}
    t = threading.Thread(target=lambda: answer.update(res=svc.search_point("A_Employees", vs[40][0], 1)))
    t.start()
    assert started.wait(10)
    for i in range(0, 30):
        svc.delete_point("A_Employees", f"p{i}")
    assert svc.compact()[0] == 200
    go.set()
    t.join(10)
    assert answer["res"][0] == 200 and answer["res"][1]["data"][0][1]["id"] == "p40"


def test_service_with_a_head():
    """Descriptors of the head's input length are projected on their way in and to a search; rows of the gallery's own
    length go as they are; other lengths are refused."""
    rng = np.random.default_rng(7)
    w = rng.standard_normal((32, 128)).astype(np.float32)

    class Head:
        din, dout, calls = 128, 32, 0

        def apply(self, x):
            Head.calls += 1
            y = x.reshape(-1, 128) @ w.T
            return y / np.linalg.norm(y, axis=1, keepdims=True)
    svc = service(head=Head())
    assert svc.dim == 32
    svc.create_collection("A_Employees")
    v = rng.standard_normal(128).astype(np.float32)
    assert svc.insert_point("A_Employees", v, "p", "n", 1)[0] == 201
    assert found(svc, "A_Employees", v, 1) == "p" and Head.calls == 2
    assert found(svc, "A_Employees", Head().apply(v)[0], 1) == "p"
    for bad in (np.zeros(64, np.float32), None):
        assert svc.insert_point("A_Employees", bad, "q", "n", 1)[0] == 404
        assert svc.search_point("A_Employees", bad, 1)[0] == 404


def test_sharded_service_drops_collections_and_refuses_moves():
    from frhot.sharded_service import ShardedGalleryService
    import torch
    from oracle import search as osr

    class Backend:
        def __init__(self):
            self.gallery, self.cap, self.device, self.qdtype = PagedGallery(32, 600), 600, torch.device("cpu"), torch.float32

        def unit_queries(self, vecs):
            return torch.from_numpy(osr.unit_rows(vecs))

        def search_local(self, q, s, r, keys=None):
            a, b = self.gallery.search(q.numpy(), keys.numpy(), s.shape[1])
            s.copy_(torch.from_numpy(a))
            r.copy_(torch.from_numpy(b))

        def merge(self, s_all, r_all, out_s, out_r, block_bytes):
            out_s.copy_(s_all[0])
            out_r.copy_(r_all[0])
    svc = ShardedGalleryService(Backend(), 0, 1, 600, 32, batch=4)
    rng = np.random.default_rng(8)
    ops = [("create_collection", "A_Employees"), ("create_collection", "B_Employees")]
    ops += [("insert_point", dict(collection_name=c, vector_embedding=rng.standard_normal(32).astype(np.float32), id=f"{i}", name="n",
                                  store_id=1)) for c in ("A_Employees", "B_Employees") for i in range(20)]
    assert all(a[0] == 201 for a in svc.mutate(ops))
    assert svc.mutate([("delete_collection", "A_Employees"), ("delete_collection", "A_Employees")]) == [
        (200, {"message": "Collection deleted"}), (404, {"message": "Collection name not found or invalid!"})]
    assert svc.point_count("B_Employees") == 20 and int((svc.gallery.b.gallery.keys >= 0).sum()) == 20
    for f in (lambda: svc.copy_collection("B_Employees", "C_Employees"), svc.compact):
        with pytest.raises(NotImplementedError):
            f()


def test_row_allocator_reset():
    from frhot.gallery_service import TILE, _RowAllocator
    a = _RowAllocator(5 * TILE)
    keys = [4] * 200 + [7] * 300 + [4] * 100
    a.reset(keys)
    assert a.free_count() == 5 * TILE - 600
    assert a.alloc(a._owner[2]) == 600                   # the last tile's own key goes on behind the squeezed rows
    other = a.alloc(99)
    assert other == 3 * TILE
    a.release(0)
    assert a.alloc(a._owner[0]) == 0
    full = _RowAllocator(300)
    full.reset([1] * 300)
    with pytest.raises(MemoryError):
        full.alloc(1)


def test_bf16_bits_round_to_nearest_even():
    import torch
    from frhot.engine import bf16_bits
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(5000).astype(np.float32) * np.float32(10) ** rng.integers(-30, 30, 5000),
                        np.array([0, -0.0, np.inf, -np.inf, 3.4e38, -3.4e38, 1.00390625, 1.01171875, 1e-40], np.float32)]).astype(np.float32)
    want = torch.from_numpy(x).bfloat16().view(torch.int16).numpy().view(np.uint16)
    assert np.array_equal(bf16_bits(x), want)
    nan = np.array([0x7F800001, 0xFFFFFFFF, 0x7FC00000], np.uint32).view(np.float32)
    assert np.isnan(torch.from_numpy(bf16_bits(nan).view(np.int16)).view(torch.bfloat16).float().numpy()).all()


def test_runs_of():
    from frhot.engine import runs_of
    first, counts = runs_of([5, 6, 7, 2, 3, 9, 8, 100])
    assert first.tolist() == [5, 2, 9, 8, 100] and counts.tolist() == [3, 2, 1, 1, 1]
    first, counts = runs_of([])
    assert first.size == counts.size == 0


def test_null_handles_are_refused_without_a_device():
    from frhot import _lib
    lib = _lib.load()
    h, n = C.c_void_p(), C.c_int64(5)
    i64, i32, f32 = (t * 4 for t in (C.c_int64, C.c_int32, C.c_float))
    buf = f32()
    assert lib.frhot_linear_create(None, C.addressof(buf), None, 2, 2, 0, C.byref(h)) == -1
    assert lib.frhot_linear_dev(None, None, 0, 0, 0, None, 0, 0, None, 0, 0) == -1
    assert lib.frhot_unit_rows_dev(None, None, 0, 0, 0, 0, None, 0) == -1
    assert lib.frhot_head_create(None, None, None, None, 0, C.byref(h)) == -1
    assert lib.frhot_head_dev(None, None, 0, 0, None, 0) == -1
    assert lib.frhot_head_apply(None, buf, 1, buf) == -1
    assert lib.frhot_ctx_head(None, None) == -1
    assert lib.frhot_linear_destroy(None) == 0 and lib.frhot_head_destroy(None) == 0
    rows, counts = i64(), i32()
    for rc in (lib.frhot_gallery_copy(None, rows, None, rows, counts, None, 1), lib.frhot_gallery_read_dev(None, rows, counts, 1, None, None),
               lib.frhot_gallery_write_dev(None, None, rows, counts, counts, 1), lib.frhot_gallery_free_keys(None, counts, 1, C.byref(n)),
               lib.frhot_gallery_compact(None, None, None, C.byref(n)), lib.frhot_gallery_reproject(None, None, None)):
        assert rc == -1 and lib.frhot_last_error()
    assert n.value == 0
