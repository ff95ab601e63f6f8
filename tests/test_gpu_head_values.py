"""What a head's inner layers hand on: fp32 values of any range, not rounded between the layers.  The data are whole numbers
whose products and sums fp32 holds exactly, so the last layer's rows are known exactly and only their unit rows are rounded; or
powers of two times other data, which change no bit of a unit row."""
import numpy as np
import pytest
import torch

from test_gpu_heads import NAN, check_unit, ctx, linear_of      # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu


def whole(shape, most, seed):
    return torch.randint(-most, most + 1, shape, generator=torch.Generator().manual_seed(seed)).half()


def head_of(ctx, layers):
    from frhot.engine import Head
    lins = [linear_of(ctx, w, b, "f16") for w, b, _, _ in layers]
    return Head(ctx, [(lin, act, res) for lin, (_, _, act, res) in zip(lins, layers)])


def through(ctx, head, x):
    out = torch.empty(x.shape[0], head.dout, dtype=torch.float16, device="cuda")
    xd = x.cuda()
    torch.cuda.synchronize()
    head.run_dev(xd.data_ptr(), x.shape[0], out.data_ptr())
    ctx.sync()
    return out.cpu()


def exact_rows(x, layers):
    """The last layer's rows; whole numbers below 2^24 at every sum, checked on the magnitudes."""
    v = x.double()
    for w, b, act, res in layers:
        y, mag = v @ w.double().t(), v.abs() @ w.double().abs().t()
        if b is not None:
            y, mag = y + b.double(), mag + b.double().abs()
        if act == "relu":
            y = y.clamp_min(0)
        if res:
            y, mag = y + v, mag + v.abs()
        assert mag.max() < 2 ** 24
        v = y
    return v


@pytest.mark.parametrize("mid", [64, 130, 500, 2500])
@pytest.mark.parametrize("m", [1, 50, 2100])
def test_inner_layers_are_not_rounded(ctx, mid, m):      # noqa: F811
    """Inner values of several thousand with odd last bits, which fp16 does not hold."""
    layers = [(whole((mid, 64), 48, 1), whole((mid,), 2000, 2).float(), "relu", False), (whole((64, mid), 2, 3), None, "none", False)]
    x = whole((m, 64), 48, m)
    head = head_of(ctx, layers)
    check_unit(through(ctx, head, x), exact_rows(x, layers).float())
    head.close()


@pytest.mark.parametrize("m", [3, 700])
def test_inner_residuals_are_not_rounded(ctx, m):        # noqa: F811
    layers = [(whole((128, 128), 24, 1), whole((128,), 999, 2).float(), "none", True),
              (whole((128, 128), 1, 3), None, "relu", True), (whole((128, 128), 1, 4) * (whole((128, 128), 3, 5) == 0), None, "none", True),
              (whole((64, 128), 1, 6) * (whole((64, 128), 5, 7) == 0), None, "none", False)]
    x = whole((m, 128), 20, m)
    head = head_of(ctx, layers)
    check_unit(through(ctx, head, x), exact_rows(x, layers).float())
    head.close()


def test_inner_values_of_any_range(ctx):                 # noqa: F811
    """Inner rows from 2^-30 to 2^40 (fp16 ends at 2^16 and 2^-24): unit rows do not change by a bit."""
    g = torch.Generator().manual_seed(4)
    w1, w2 = torch.randn(320, 128, generator=g).half(), torch.randn(64, 320, generator=g).half()
    x = torch.randn(40, 128, generator=g).half()
    x = torch.where(x.abs() < 2.0 ** -4, torch.zeros_like(x), x)            # (so that no scaled value loses bits)
    w1 = torch.where(w1.abs() < 2.0 ** -4, torch.zeros_like(w1), w1)
    w3 = torch.where(w2.abs() < 2.0 ** -4, torch.zeros_like(w2), w2)
    plain = None
    for px, pw, extra in ((0, 0, 0), (12, 12, 0), (-8, -8, 0), (0, 13, 0), (11, 0, 0), (13, 13, 13), (-9, -9, -9)):
        layers = [(w1 * 2.0 ** pw, None, "relu", False), (w3 * 2.0 ** extra, None, "none", False)]
        head = head_of(ctx, layers)
        got = through(ctx, head, x * 2.0 ** px)
        head.close()
        assert torch.isfinite(got).all(), (px, pw)
        plain = got if plain is None else plain
        assert torch.equal(got, plain), (px, pw, extra)
    check_unit(plain, (torch.relu(x.double() @ w1.double().t()) @ w3.double().t()).float())


def test_inner_rows_of_different_ranges_and_nonfinite_ones(ctx):             # noqa: F811
    """Every row for itself: huge, tiny, zero, infinite and NaN rows beside ordinary ones."""
    g = torch.Generator().manual_seed(9)
    layers = [(torch.randn(192, 64, generator=g).half(), None, "relu", False), (torch.randn(64, 192, generator=g).half(), None, "none", False)]
    head = head_of(ctx, layers)
    x = torch.randn(60, 64, generator=g).half()
    x = torch.where(x.abs() < 2.0 ** -4, torch.zeros_like(x), x)
    plain = through(ctx, head, x)
    y = x.clone()
    y[3] *= 2.0 ** 13
    y[4] *= 2.0 ** -9
    y[7] = 0
    y[20, 5], y[33, 0], y[34, 1] = NAN, float("inf"), -float("inf")
    got = through(ctx, head, y)
    same = [i for i in range(60) if i not in (7, 20, 33, 34)]
    assert torch.equal(got[same], plain[same])
    assert (got[7] == 0).all() and torch.isnan(got[20]).all() and torch.isnan(got[[33, 34]]).all()
    head.close()


@pytest.mark.parametrize("scale", [1.0, 1e-30, 3e37, 1e-5])
def test_what_a_pair_of_fp16_numbers_loses(ctx, scale):  # noqa: F811
    """Inner values that use all of fp32's bits (a bias on nothing), passed on unchanged: half a step of the second number,
    2^-23 of the value, or 2^-39 of the row's largest, and the rounding of the two numbers' sum."""
    g = torch.Generator().manual_seed(5)
    b = torch.randn(1024, generator=g) * torch.rand(1024, generator=g) ** 8 * scale
    b[:4] = torch.tensor([scale, -scale, 0.0, scale * (1 + 2.0 ** -11 + 2.0 ** -23)])
    layers = [(torch.zeros(1024, 64, dtype=torch.float16), b, "none", False), (torch.eye(1024).half(), None, "none", False)]
    head = head_of(ctx, layers)
    got = torch.from_numpy(head.project(np.zeros((3, 64), np.float32))).double()
    want = b.double().expand(3, -1)
    tol = torch.maximum(2.0 ** -23 * want.abs(), 2.0 ** -39 * want.abs().max()) + 2.0 ** -24 * want.abs()
    assert ((got - want).abs() <= tol).all()
    head.close()
