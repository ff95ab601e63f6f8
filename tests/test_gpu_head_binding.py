"""Heads and galleries of one context: each gallery's queries come from the head that it is bound to."""
import numpy as np
import pytest
import torch

from test_gpu_heads import linear_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def faces(gpu_ctx):
    from frhot import synth
    crops = synth.crops(seed=9, n=8, lo=90, hi=180)
    return crops, gpu_ctx.embed(crops, gamma=True)


def spreading_head(ctx, emb, width, seed):
    """Random directions around the faces' mean: the synthetic network's faces are alike."""
    from frhot.engine import Head
    w = (torch.randn(width, 4096, generator=torch.Generator().manual_seed(seed)) / 8).half()
    mean = torch.from_numpy(emb).double().mean(0)
    return Head(ctx, [(linear_of(ctx, w, (-(w.double() @ mean)).float(), "f16"), "none", False)])


def serve(ctx, emb, rng, **kw):
    from frhot.gallery_service import GalleryService
    svc = GalleryService(ctx, capacity=600, **kw)
    svc.create_collection("7_Employees")
    for i in range(100):
        svc.insert_point("7_Employees", rng.standard_normal(svc.dim).astype(np.float32), f"s{i}", "x", 7)
    for i, e in enumerate(emb):
        vec = e if svc.head is not None else e[:svc.dim]
        assert svc.insert_point("7_Employees", vec, f"p{i}", f"n{i}", 7)[0] == 201
    return svc


def test_services_of_one_context_do_not_share_a_head(gpu_ctx, faces):
    """Two services with heads of one width, one of another width and one without a head: each answers as it does alone,
    while the others live and after they have gone."""
    crops, emb = faces
    rng = np.random.default_rng(0)
    a, b, c = (spreading_head(gpu_ctx, emb, w, s) for w, s in ((256, 3), (256, 4), (128, 5)))

    def answer(svc):
        s, r, _ = gpu_ctx.recognise(svc.gallery, crops, None, 5, gamma=True)
        return s, r
    svcs, alone = [], []
    for kw in (dict(head=a), dict(dim=256), dict(head=b), dict(head=c), dict(dim=128)):
        svcs.append(serve(gpu_ctx, emb, rng, **kw))
        alone.append(answer(svcs[-1]))
        for svc, want in zip(svcs, alone):
            got = answer(svc)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), kw
    for i in (0, 2, 3):                     # through the heads: everyone is found as himself, and nearly one
        who = [content["data"][0][1]["id"] for _s, content, _e in svcs[i].recognise_points([("7_Employees", x, 7) for x in crops])]
        assert who == [f"p{j}" for j in range(8)]
        assert np.abs(alone[i][0][:, 0] - 1).max() <= 1e-3
    for i in (0, 3, 2):                     # (their heads go with them)
        svcs[i].close()
        svcs[i].head.close()
        for j in (1, 4):
            got = answer(svcs[j])
            assert np.array_equal(got[0], alone[j][0]) and np.array_equal(got[1], alone[j][1])
    for j in (1, 4):
        svcs[j].close()


def test_binding_and_attaching(gpu_ctx, faces):
    """A bound gallery does not look at the context's head, an unbound one does; refusals; a bound head stays."""
    from frhot import FrhotError
    from frhot.engine import Context, Gallery, Head, Linear
    from frhot.gallery_service import GalleryService
    crops, emb = faces
    a, b = spreading_head(gpu_ctx, emb, 256, 3), spreading_head(gpu_ctx, emb, 256, 4)
    gal = Gallery(gpu_ctx, 256, 300)
    gal.fill_synthetic(3, 0, 300)

    def answer():
        return gpu_ctx.recognise(gal, crops, None, 5)[0]
    lead = answer()
    gal.set_head(a)
    by_a = answer()
    assert not np.array_equal(lead, by_a)
    gpu_ctx.set_head(b)
    assert np.array_equal(answer(), by_a)
    gal.set_head(None)
    by_b = answer()
    assert not np.array_equal(by_b, by_a)
    gpu_ctx.set_head(None)
    assert np.array_equal(answer(), lead)

    def refused(code, f, *args, **kw):
        with pytest.raises(FrhotError) as e:
            f(*args, **kw)
        assert e.value.code == code, e.value
    gal.set_head(a)
    refused(-3, a.close)
    assert np.array_equal(answer(), by_a)
    other = Gallery(gpu_ctx, 128, 10)
    refused(-1, other.set_head, a)                                      # 256 outputs
    small = Head(gpu_ctx, [(Linear(gpu_ctx, np.zeros((128, 64), np.float16)), "none", False)])
    refused(-1, other.set_head, small)                                  # takes no descriptors
    refused(-1, GalleryService, gpu_ctx, capacity=10, head=small)
    c2 = Context(device=0, max_batch=1)
    far = Gallery(c2, 256, 10)
    refused(-1, far.set_head, a)
    gal.set_head(b)
    a.close()
    assert np.array_equal(answer(), by_b)
    gal.close()                                                         # unbinds
    b.close()
    for x in (other, far, small):
        x.close()
    c2.close()


def test_services_asked_at_the_same_time(gpu_ctx, faces):
    """Threads on two services with heads of one width, by crop and by vector, while one of them is squeezed."""
    import threading
    crops, emb = faces
    rng = np.random.default_rng(3)
    heads = [spreading_head(gpu_ctx, emb, 256, s) for s in (3, 4)]
    svcs = [serve(gpu_ctx, emb, rng, head=h) for h in heads]
    errors, stop = [], threading.Event()

    def ask(j):
        svc, r = svcs[j % 2], np.random.default_rng(j)
        try:
            while not stop.is_set():
                at = r.permutation(8)[:4]
                if j < 2:
                    got = [c["data"][0][1]["id"] for _s, c, _e in svc.recognise_points([("7_Employees", crops[i], 7) for i in at])]
                else:
                    got = [c["data"][0][1]["id"] for _s, c in svc.search_points([("7_Employees", emb[i] * 2, 7) for i in at])]
                assert got == [f"p{i}" for i in at], got
        except Exception as e:
            errors.append(e)
    ts = [threading.Thread(target=ask, args=(j,)) for j in range(4)]
    [t.start() for t in ts]
    try:
        for i in range(0, 100, 2):
            assert svcs[0].delete_point("7_Employees", f"s{i}")[0] == 200
            if i % 20 == 0:
                assert svcs[0].compact()[0] == 200
    finally:
        stop.set()
        [t.join(60) for t in ts]
    assert not errors, errors[0]
    for svc, h in zip(svcs, heads):
        svc.close()
        h.close()
