"""Every kernel that a layer's product runs as, on whole numbers whose products and sums fp32 holds exactly: the answers are
equal, not close.  NaN behind every row of x and behind the last one; what lies around the output stays."""
import pytest
import torch

from linear_plans import PLANS
from test_gpu_heads import DT, NAN, check_unit, ctx, linear_of      # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu


def whole(gen, shape, most, dtype):
    return torch.randint(-most, most + 1, shape, generator=gen, device="cuda", dtype=torch.int8).to(DT[dtype])


def exact(x, w, b):
    """x W^T + b by fp32 products of whole numbers: every partial sum stays below 2^24."""
    assert 9 * x.shape[1] + 1000 < 2 ** 24
    return x.float() @ w.float().t() + b


@pytest.mark.parametrize("i", range(len(PLANS)), ids=["-".join(map(str, p)) for p in PLANS])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_kernel(ctx, i, dtype):            # noqa: F811
    _shape, way, _splits, m, n, k = PLANS[i]
    gen = torch.Generator("cuda").manual_seed(i)
    ldx = k + 8 if way == "dma" else k + (1 if (k + 1) % 8 else 2)
    buf = torch.full((m + 1, ldx), NAN, dtype=DT[dtype], device="cuda")
    buf[:m, :k] = whole(gen, (m, k), 3, dtype)
    w, b = whole(gen, (n, k), 3, dtype), whole(gen, (n,), 100, "f32")
    lin = linear_of(ctx, w.cpu(), b.cpu(), dtype)
    out = torch.full((m + 1, n + 3), 7.0, device="cuda")
    torch.cuda.synchronize()
    lin.run_dev(buf.data_ptr(), m, out.data_ptr(), act="relu", ldx=ldx, ldo=n + 3, out_dtype="f32")
    ctx.sync()
    want = exact(buf[:m, :k], w, b).clamp_min_(0)
    assert torch.equal(out[:m, :n], want)
    assert (out[m] == 7).all() and (out[:, n:] == 7).all()
    lin.close()


@pytest.mark.parametrize("dims", [[512, 512], [512, 512, 512], [64, 500, 448]])
def test_a_gallery_through_large_tiles(ctx, dims):       # noqa: F811
    """Rows in a gallery's own order, more of them than one pass takes, and pairs behind an inner layer."""
    from frhot.engine import Gallery, Head
    import ctypes as C
    n = 70001
    plan = (C.c_int32 * 4)()
    gen = torch.Generator("cuda").manual_seed(len(dims))
    lins, v = [], None
    src, dst = Gallery(ctx, dims[0], n), Gallery(ctx, dims[-1], n)
    x = whole(gen, (n, dims[0]), 3, "f16")
    torch.cuda.synchronize()
    src.write_dev(x.data_ptr(), [0, 30000], [30000, n - 30000], [1, 2])
    for i in range(len(dims) - 1):
        w, b = whole(gen, (dims[i + 1], dims[i]), 3 if i == 0 else 1, "f16"), whole(gen, (dims[i + 1],), 100, "f32")
        lins.append(linear_of(ctx, w.cpu(), b.cpu(), "f16"))
        mag = (v if i else x).float().abs() @ w.float().abs().t()
        assert mag.max() < 2 ** 23
        v = (v if i else x.float()) @ w.float().t() + b
        if i == 0 and len(dims) > 2:
            v = v.clamp_min(0)
        assert ctx._lib.frhot_linear_debug_plan(dims[i + 1], dims[i], 16384, 1, i > 0, plan) == 0 and plan[0] >= 5
    head = Head(ctx, [(lin, "relu" if i == 0 and len(lins) > 1 else "none", False) for i, lin in enumerate(lins)])
    src.reproject(head, dst)
    out, keys = torch.empty(n, dims[-1], dtype=torch.float16, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    dst.read_dev([0], [n], out.data_ptr(), keys.data_ptr())
    ctx.sync()
    assert (keys == torch.where(torch.arange(n, device="cuda") < 30000, 1, 2)).all()
    check_unit(out.cpu(), v.cpu())
    head.close()
    [lin.close() for lin in lins]
    src.close()
    dst.close()
