"""A service with a head on the device: vectors from the host and descriptors that never leave it give the same rows."""
import numpy as np
import pytest
import torch

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
