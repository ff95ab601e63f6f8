"""A service with a head on the device: vectors from the host and descriptors that never leave it give the same rows."""
import numpy as np
import pytest
import torch

from test_gpu_heads import linear_of
from test_gpu_head_binding import faces, serve, spreading_head      # noqa: F401  (faces: the fixture)

pytestmark = pytest.mark.gpu


def rows_by_id(svc, ids):
    at = [next(r for r, p in svc._points.items() if p["payload"]["id"] == i) for i in ids]
    return svc.gallery.read(np.asarray(at))[0].astype(np.float64)


def test_vectors_of_any_length(gpu_ctx, faces):                      # noqa: F811
    """A face's vector, times anything: the row of the face as recognise makes it."""
    crops, emb = faces
    head = spreading_head(gpu_ctx, emb, 256, 3)
    svc = serve(gpu_ctx, emb, np.random.default_rng(0), head=head)
    scales = [3.0, 2.0 ** -10, 1e6, 1e-20]
    for i, s in enumerate(scales):
        assert svc.insert_point("7_Employees", emb[i] * np.float32(s), f"q{i}", "n", 7)[0] == 201
    a, b = rows_by_id(svc, [f"p{i}" for i in range(4)]), rows_by_id(svc, [f"q{i}" for i in range(4)])
    assert np.isfinite(b).all()
    # a component of the descriptor moves by one fp16 step at most where float32's rounding of the division crosses a border: the
    # difference reaches a row through the layer's gain on differences from the mean, 1/8 a component
    assert ((a * b).sum(1) >= 1 - 1e-4).all()
    for i, s in enumerate(scales):
        hits = svc.search_point("7_Employees", emb[i] * np.float32(s), 7)[1]["data"]
        assert hits and hits[0][1]["id"] in (f"p{i}", f"q{i}")
    svc.close()
    head.close()


def test_apply_refuses_what_fp16_does_not_hold(gpu_ctx, faces):      # noqa: F811
    from frhot import FrhotError
    _, emb = faces
    head = spreading_head(gpu_ctx, emb, 256, 3)
    x = emb[:3].copy()
    x[1, 77] = 65519.0                                               # rounds to 65504
    assert np.isfinite(head.apply(x)).all()
    for big in (65520.0, -1e30):
        x[1, 77] = big
        with pytest.raises(FrhotError) as e:
            head.apply(x)
        assert e.value.code == -1 and "component 77 of row 1" in str(e.value)
    x[1, 77] = np.nan
    got = head.apply(x)
    assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2]]).all()
    head.close()


def test_host_vectors_are_rounded_once(gpu_ctx):
    """Rows of few large components, where rounding to fp16, bringing to unit length and rounding again is not rounding once:
    what the service stores and asks with are the head's own rows, bit for bit."""
    from frhot.engine import Gallery, Head
    from frhot.gallery_service import GalleryService
    rng = np.random.default_rng(0)
    w = np.zeros((64, 4096), np.float16)
    w[:4] = rng.standard_normal((4, 4096))

    def unit(v):
        v = v.astype(np.float32)
        return (v / np.sqrt((v.astype(np.float64) ** 2).sum(1, keepdims=True)).astype(np.float32)).astype(np.float16)
    at = np.flatnonzero((unit(w[:4].T) != unit(unit(w[:4].T))).any(1))
    assert at.size >= 20
    x = np.zeros((at.size, 4096), np.float32)
    x[np.arange(at.size), at] = 1
    head = Head(gpu_ctx, [(linear_of(gpu_ctx, torch.from_numpy(w), None, "f16"), "none", False)])
    xd, own = torch.from_numpy(x).half().cuda(), torch.empty(at.size, 64, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    head.run_dev(xd.data_ptr(), at.size, own.data_ptr())
    gpu_ctx.sync()
    want = own.cpu().numpy()
    assert np.array_equal(head.apply(x), want.astype(np.float32))
    assert np.array_equal(head.project(x), w[:, at].T.astype(np.float32))
    svc = GalleryService(gpu_ctx, capacity=600, head=head)
    svc.create_collection("7_Employees")
    for i in range(at.size):
        assert svc.insert_point("7_Employees", x[i], f"p{i}", "n", 7)[0] == 201
    rows = [next(r for r, p in svc._points.items() if p["payload"]["id"] == f"p{i}") for i in range(at.size)]
    assert np.array_equal(svc.gallery.read(rows)[0], want)
    other = Gallery(gpu_ctx, 64, 400)
    other.fill_synthetic(5, 0, 400)
    s, r = torch.empty(at.size, 5, device="cuda"), torch.empty(at.size, 5, dtype=torch.int64, device="cuda")
    other.search_dev(own.data_ptr(), None, at.size, 5, s.data_ptr(), r.data_ptr())
    gpu_ctx.sync()
    hs, hr = other.search(head.project(x), None, 5)
    assert np.array_equal(hs, s.cpu().numpy()) and np.array_equal(hr, r.cpu().numpy())
    other.close()
    svc.close()
    head.close()


def test_host_rows_of_many_sizes(gpu_ctx, faces):                    # noqa: F811
    """The staging grows and shrinks between calls; every call gives the rows of run_dev."""
    _, emb = faces
    head = spreading_head(gpu_ctx, emb, 256, 6)
    x = np.random.default_rng(1).standard_normal((2000, 4096)).astype(np.float32) / 64
    xd, own = torch.from_numpy(x).half().cuda(), torch.empty(2000, 256, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    for n in (1, 5, 2000, 3, 700, 1):
        own.zero_()
        torch.cuda.synchronize()
        head.run_dev(xd.data_ptr(), n, own.data_ptr())
        gpu_ctx.sync()
        assert np.array_equal(head.apply(x[:n]), own[:n].cpu().numpy().astype(np.float32))
    head.close()
