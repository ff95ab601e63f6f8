"""The activations where their values leave fp32's normal range: relative accuracy up to there."""
import pytest
import torch

from test_gpu_heads import act64, ctx, linear_of        # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,lo,hi,step", [("silu", -97, -60, 1 / 16), ("gelu", -13.75, -11, 1 / 128), ("gelu_tanh", -12.5, -8, 1 / 128)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_the_far_left(ctx, act, lo, hi, step, out):      # noqa: F811
    v = torch.arange(lo, hi, step).half()
    assert (v.double() == torch.arange(lo, hi, step).double()).all()
    x, w = torch.zeros(v.numel(), 8, dtype=torch.float16), torch.zeros(32, 8, dtype=torch.float16)
    x[:, 0], w[:, 0] = v, 1
    lin = linear_of(ctx, w, None, "f16")
    xd = x.cuda()
    o = torch.empty(v.numel(), 32, dtype=torch.float32 if out == "f32" else torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    lin.run_dev(xd.data_ptr(), v.numel(), o.data_ptr(), act=act, out_dtype=out)
    ctx.sync()
    got, d = o.cpu().double(), v.double()
    assert (got == got[:, :1]).all()
    y = act64(d, act)
    # the exponential 3 units of 2^-24, twice; the fit 5, the reciprocals 2, products and the final rounding 6 (not all of them in one
    # activation); the tanh form's argument has three roundings of |2 u|.  gelu's normal distribution function goes below the normal range 13 times (4 bits) before its product.
    u2 = 1.6 * (d.abs() + 0.044715 * d.abs() ** 3)
    rel = {"silu": 16, "gelu": 16 + 16, "gelu_tanh": 16 + 3 * u2}[act] * 2.0 ** -24
    tol = rel * y.abs() + (torch.finfo(torch.bfloat16).eps / 2 * y.abs() if out == "bf16" else 0)
    normal = y.abs() >= 2.0 ** -126
    assert normal.sum() > 200 and (~normal).sum() > 5
    err = (got[:, 0] - y).abs()
    assert (err <= tol)[normal].all(), (v[normal & (err > tol)], got[:, 0][normal & (err > tol)])
    assert (got[:, 0].abs() <= 2.0 ** -126)[~normal].all() and (got[:, 0] <= 0).all()
    lin.close()
