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


def test_null_gallery_is_refused():
    from frhot import _lib
    assert _lib.load().frhot_gallery_head(None, None) == -1
