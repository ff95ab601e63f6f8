"""Host side of descriptor heads in a service, over stand-ins."""
import threading

import numpy as np

from test_pages_cpu import PagedGallery, found, service       # noqa: F401


class FakeHead:
    """A linear map with a bias: what it gives depends on its input's length."""

    def __init__(self, din=128, dout=32, seed=7):
        rng = np.random.default_rng(seed)
        self.din, self.dout = din, dout
        self.w, self.b = rng.standard_normal((dout, din)).astype(np.float32), rng.standard_normal(dout).astype(np.float32)
        self.calls = []

    def apply(self, x):
        x = np.asarray(x, np.float32).reshape(-1, self.din)
        self.calls.append(len(x))
        y = x @ self.w.T + self.b
        return y / np.linalg.norm(y, axis=1, keepdims=True)


def test_a_service_binds_its_gallery_and_leaves_the_context_alone():
    from frhot.gallery_service import GalleryService
    bound = []

    class Ctx:
        def set_head(self, head):
            raise AssertionError("the context serves others too")

    class Bound(PagedGallery):
        def set_head(self, head):
            bound.append(head)
    head = FakeHead()
    GalleryService(Ctx(), capacity=600, gallery=Bound(32, 600), head=head)
    assert bound == [head]
    GalleryService(Ctx(), capacity=600, dim=32, gallery=Bound(32, 600))
    assert bound == [head]


def test_vectors_of_any_length_give_the_same_row():
    """Cosine does not care how long a vector is, and a bias behind it must not either."""
    rng = np.random.default_rng(1)
    head = FakeHead()
    svc = service(head=head)
    svc.create_collection("A_Employees")
    v = rng.standard_normal(128).astype(np.float32)
    v /= np.linalg.norm(v)
    other = head.apply(-v)[0]
    assert svc.insert_point("A_Employees", other, "other", "n", 1)[0] == 201
    scales = [1, 3, 1e6, 1e-6, 1e18]
    for i, s in enumerate(scales):
        assert svc.insert_point("A_Employees", v * np.float32(s), f"p{i}", "n", 1)[0] == 201
    want = head.apply(v)[0]
    rows = [r for r, p in svc._points.items() if p["payload"]["id"] != "other"]
    assert len(rows) == len(scales)
    for r in rows:
        assert np.abs(svc.gallery.g[r] - want).max() <= 1e-5           # (float32 sums of 128 terms)
    for s in scales:
        assert found(svc, "A_Employees", v * np.float32(s), 1).startswith("p")
    assert svc.insert_point("A_Employees", np.zeros(128, np.float32), "zero", "n", 1)[0] == 201       # the bias alone, as the head gives it


def test_nonfinite_vectors_are_refused():
    svc = service(head=FakeHead())
    svc.create_collection("A_Employees")
    v = np.ones(128, np.float32)
    assert svc.insert_point("A_Employees", v, "p", "n", 1)[0] == 201
    for bad in (np.nan, np.inf, -np.inf, 1e39):
        w = v.astype(np.float64)
        w[5] = bad
        assert svc.insert_point("A_Employees", w, "q", "n", 1) == (404, {"message": "Embedding not found or invalid!"})
        assert svc.insert_point("A_Employees", list(w), "q", "n", 1)[0] == 404
        assert svc.search_point("A_Employees", w, 1)[0] == 404
    assert svc.insert_point("A_Employees", ["x"] * 128, "q", "n", 1)[0] == 404 and svc.search_point("A_Employees", [None, "x"] * 64, 1)[0] == 404
    assert svc.point_count("A_Employees") == 1


def test_a_batch_of_searches_goes_through_the_head_at_once_and_without_the_lock():
    rng = np.random.default_rng(2)
    head = FakeHead()
    svc = service(head=head)
    svc.create_collection("A_Employees")
    vecs = rng.standard_normal((40, 128)).astype(np.float32)
    for i, v in enumerate(vecs):
        assert svc.insert_point("A_Employees", v, f"p{i}", "n", 1)[0] == 201
    head.calls.clear()
    started, go, done = threading.Event(), threading.Event(), threading.Event()
    plain = head.apply

    def slow(x):
        started.set()
        assert go.wait(10)
        return plain(x)
    head.apply = slow
    own = plain(vecs[33])[0]                        # a row of the gallery's own length among them
    reqs = [("A_Employees", v, 1) for v in vecs[:32]] + [("A_Employees", own, 1), ("B_Employees", vecs[0], 1), ("A_Employees", None, 1)]
    head.calls.clear()
    answer = {}
    t = threading.Thread(target=lambda: answer.update(out=svc.search_points(reqs)))
    t.start()
    assert started.wait(10)
    other = threading.Thread(target=lambda: (svc.delete_point("A_Employees", "p39"), done.set()))
    other.start()
    assert done.wait(10), "a deletion waits for the head"
    go.set()
    t.join(10)
    other.join(10)
    out = answer["out"]
    assert head.calls == [32]
    assert [c["data"][0][1]["id"] for _s, c in out[:33]] == [f"p{i}" for i in range(32)] + ["p33"]
    assert [s for s, _c in out[33:]] == [404, 404]


def test_a_failing_head_answers_404():
    svc = service(head=FakeHead())
    svc.create_collection("A_Employees")
    assert svc.insert_point("A_Employees", np.ones(128, np.float32), "p", "n", 1)[0] == 201

    def broken(x):
        raise RuntimeError("device lost")
    svc.head.apply = broken
    v = np.ones(128, np.float32)
    assert svc.search_points([("B_Employees", v, 1), ("A_Employees", v, 1), ("A_Employees", v, 99)]) == [
        (404, {"message": "Collection name not found or invalid!"}), (404, {"message": "device lost"}),
        (200, {"message": "Point not found", "data": []})]
    assert svc.insert_point("A_Employees", v, "q", "n", 1) == (404, {"message": "device lost"})


def test_null_gallery_is_refused():
    from frhot import _lib
    assert _lib.load().frhot_gallery_head(None, None) == -1
