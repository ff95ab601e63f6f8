"""Host side of descriptor heads in a service, over stand-ins."""
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
    assert svc.point_count("A_Employees") == 1


def test_null_gallery_is_refused():
    from frhot import _lib
    assert _lib.load().frhot_gallery_head(None, None) == -1
