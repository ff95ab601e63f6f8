"""Descriptor heads on the GPU: the matrix product with its epilogue, unit rows, heads of several layers, and the embed
path through an attached head, each against a 64-bit restatement of its formula.

Tolerances of a layer, per element: products of fp16 / bf16 values are exact in fp32, every one of the K + 1 additions is off
by at most 2^-23 of the sum of magnitudes (a truncating adder's step); the activations have slopes of at most 1.13; expf and
erfcf are within a few units of 2^-24 of their value and amplify their argument's rounding by the argument (exp) or its square
(erfc); the residual's addition is one more fp32 rounding and the result is rounded once to the output type."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
NAN = float("nan")


@pytest.fixture(scope="module")
def ctx():
    from frhot.engine import Context
    c = Context(device=0, max_batch=2)
    yield c
    c.close()


def act64(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    if act == "gelu_tanh":
        return v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return v


def layer64(x, w, b, act, r):
    """(value, bound on the fp32 value's error) on the CPU in 64 bits."""
    xd, wd = x.double(), w.double()
    v = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    if b is not None:
        v, mag = v + b.double(), mag + b.double().abs()
    tol = 1.13 * (x.shape[1] + 1) * 2.0 ** -23 * mag
    y = act64(v, act)
    if act != "none":
        tol = tol + (16 + 8 * v * v + v.abs() ** 3) * 2.0 ** -24 * y.abs()
    if r is not None:
        y = y + r.double()
        tol = tol + 2.0 ** -24 * y.abs()
    return y, tol


def rounding(y, dtype):
    """half a step of the output type at y (and half its smallest step below its normal range)"""
    info = torch.finfo(DT[dtype])
    return info.eps / 2 * y.abs() + info.tiny * info.eps / 2


def padded(t, ld, extra_rows=0, fill=NAN, off=0):
    """t inside rows of ld elements (`off` elements into a buffer), everything else `fill`; returns (buffer, view)."""
    buf = torch.full(((t.shape[0] + extra_rows) * ld + off,), fill, dtype=t.dtype, device="cuda")
    view = buf[off:].view(-1, ld)[:t.shape[0], :t.shape[1]]
    view.copy_(t)
    return buf, view


def make(m, n, k, dtype, seed, bias=True, residual=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(DT[dtype])
    w = (torch.randn(n, k, generator=g) / math.sqrt(k)).to(DT[dtype])
    b = torch.randn(n, generator=g) if bias else None
    r = torch.randn(m, n, generator=g).to(DT[residual]) if residual else None
    return x, w, b, r


def linear_of(ctx, w, b, dtype):
    from frhot.engine import Linear
    host = w.view(torch.uint16).numpy() if dtype == "bf16" else w.numpy()
    return Linear(ctx, host, None if b is None else b.numpy(), dtype=dtype)


def run_and_check(ctx, m, n, k, dtype="f16", act="none", bias=True, residual=None, out="f16", padx=0, pado=0, offx=0, offo=0, seed=0):
    x, w, b, r = make(m, n, k, dtype, seed + m * 7 + n * 3 + k, bias, residual)
    lin = linear_of(ctx, w, b, dtype)
    xb, _ = padded(x, k + padx, 3, off=offx)        # NaN behind the K-th column and the M-th row
    rb, rv = padded(r, n + pado, 3) if r is not None else (None, None)
    ob = torch.full(((m + 3) * (n + pado) + offo,), 7.0, dtype=DT[out], device="cuda")
    torch.cuda.synchronize()
    lin.run_dev(xb.data_ptr() + offx * xb.element_size(), m, ob.data_ptr() + offo * ob.element_size(), act=act,
                residual_dev=None if rb is None else rb.data_ptr(), ldx=k + padx, ldr=n + pado, ldo=n + pado, out_dtype=out,
                residual_dtype=residual or "f16")
    ctx.sync()
    o = ob[offo:].view(-1, n + pado).cpu()
    got = o[:m, :n].double()
    y, tol = layer64(x, w, b, act, r)
    tol = tol + rounding(y.abs() + tol, out)
    bad = ~((got - y).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), ((got - y).abs() / tol).max())
    assert (o[m:] == 7).all() and (o[:m, n:] == 7).all() and (ob[:offo] == 7).all(), "wrote outside [M, N]"
    lin.close()


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 127, 128, 129, 200, 256, 257, 513])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_rows(ctx, m, dtype):
    run_and_check(ctx, m, 160, 256, dtype, out=dtype)


@pytest.mark.parametrize("n,k", [(1, 1), (1, 4096), (8, 8), (31, 33), (32, 64), (33, 65), (131, 500), (64, 7), (127, 128), (512, 72),
                                 (513, 1000), (4096, 64), (40, 4096), (257, 4104), (100, 4097), (1000, 2048)])
@pytest.mark.parametrize("m", [1, 37, 130])
def test_widths(ctx, m, n, k):
    run_and_check(ctx, m, n, k, "f16", act="relu", out="f32")


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype,out,residual", [("f16", "f16", None), ("f16", "f32", "f16"), ("bf16", "bf16", "bf16"), ("f16", "bf16", "f32"),
                                                ("bf16", "f32", None), ("bf16", "f16", "f16")])
@pytest.mark.parametrize("m", [3, 70])
def test_epilogue(ctx, act, dtype, out, residual, m):
    run_and_check(ctx, m, 96, 192, dtype, act=act, out=out, residual=residual, bias=act != "none")


@pytest.mark.parametrize("padx,pado,offx,offo", [(8, 8, 0, 0), (1, 1, 0, 0), (3, 5, 1, 1), (0, 2, 8, 8), (64, 0, 4, 0), (7, 0, 0, 3), (16, 4, 8, 4)])
@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("m", [1, 19, 140])
def test_strides_and_alignment(ctx, m, padx, pado, offx, offo, dtype, out):
    run_and_check(ctx, m, 136, 200, dtype, act="silu", out=out, residual="f16", padx=padx, pado=pado, offx=offx, offo=offo)


@pytest.mark.parametrize("m,n,k", [(256, 4096, 4096), (1, 512, 4096), (2000, 512, 4096), (64, 1024, 25088), (700, 700, 700), (5000, 96, 320),
                                   (1025, 2049, 136)])
def test_large(ctx, m, n, k):
    run_and_check(ctx, m, n, k, "f16", act="gelu", out="f16", residual="f16")


def test_packed_rows_in_several_runs(ctx):
    """Rows that the 16-byte loads cannot take go through a bounded workspace run by run."""
    run_and_check(ctx, 9000, 40, 4097, "f16", out="f32", padx=2)


@pytest.mark.parametrize("m,n,k,padx,offx", [(9001, 137, 358, 0, 0), (20011, 19, 613, 1, 1), (3001, 700, 7, 0, 0), (2100, 300, 1, 2, 0),
                                             (4097, 512, 999, 0, 3), (12000, 1100, 65, 0, 1), (5000, 520, 2049, 3, 0), (70000, 33, 127, 0, 0),
                                             (33000, 600, 130, 6, 5), (394, 512, 4095, 0, 0), (20000, 600, 136, 1, 0), (300, 2100, 4097, 0, 7)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_many_rows_off_16_bytes(ctx, m, n, k, padx, offx, dtype):
    """Row addresses, row distances and widths that LDS-DMA cannot take, in every tile that takes them; NaN behind every row."""
    run_and_check(ctx, m, n, k, dtype, act="relu", out="f32", padx=padx, offx=offx)


@pytest.mark.parametrize("m,n,k", [(98304, 160, 384), (6533, 1504, 128), (13373, 224, 1024), (24000, 256, 448), (50001, 32, 64), (30112, 32, 2944),
                                   (21342, 96, 576), (644, 288, 320), (2595, 1568, 704), (40000, 30, 200)])
def test_tiles_of_short_and_narrow_layers(ctx, m, n, k):
    run_and_check(ctx, m, n, k, "f16", act="silu", out="f16")


def test_one_layer_called_at_many_sizes(ctx):
    """Row counts and alignments in turn on one layer: each call as if it were the only one."""
    n, k = 160, 520
    x, w, b, _ = make(5000, n, k, "f16", 77)
    lin = linear_of(ctx, w, b, "f16")
    y, tol = layer64(x, w, b, "relu", None)
    tol = tol + rounding(y.abs() + tol, "f32")
    bufs = {pad: padded(x, k + pad, 0)[0] for pad in (0, 3)}
    o = torch.empty(5000, n, device="cuda")
    for m, pad in ((1, 0), (5000, 0), (5000, 3), (5000, 0), (77, 3), (77, 0), (1, 3), (300, 0), (300, 3), (1, 0)):
        o.fill_(7.0)
        torch.cuda.synchronize()
        lin.run_dev(bufs[pad].data_ptr(), m, o.data_ptr(), act="relu", ldx=k + pad, out_dtype="f32")
        ctx.sync()
        got = o.cpu().double()
        assert ((got[:m] - y[:m]).abs() <= tol[:m]).all() and (got[m:] == 7).all(), (m, pad)
    lin.close()


def test_nonfinite_values_stay_in_their_rows(ctx):
    m, n, k = 40, 64, 128
    x, w, b, r = make(m, n, k, "f16", 3, residual="f16")
    x[5, 7], x[11, 0], x[20, 3] = NAN, float("inf"), -float("inf")
    r[30, 9] = NAN
    for act in ("none", "relu", "silu", "gelu", "gelu_tanh"):
        lin = linear_of(ctx, w, b, "f16")
        xd, rd = x.cuda(), r.cuda()
        o = torch.empty(m, n, dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        lin.run_dev(xd.data_ptr(), m, o.data_ptr(), act=act, residual_dev=rd.data_ptr())
        ctx.sync()
        o = o.cpu()
        y, tol = layer64(x, w, b, act, r)
        clean = [i for i in range(m) if i not in (5, 11, 20)]
        assert torch.isnan(o[5]).all()
        assert torch.equal(torch.isnan(o[clean]), torch.isnan(y[clean]))
        if act in ("none", "relu"):
            # +-inf rows: every output is +-inf (or relu's zero) plus the residual
            want = y[[11, 20]].half()
            assert torch.equal(torch.isinf(o[[11, 20]]), torch.isinf(want)) and torch.equal(o[[11, 20]].sign(), want.sign())
        ok = torch.isfinite(y)
        ok[[5, 11, 20]] = False
        err = (o.double() - y).abs()
        assert (err[ok] <= (tol + rounding(y.abs() + tol, "f16"))[ok]).all()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_activations_over_their_range(ctx, act):
    """act(x) itself (a layer that passes its input on), from the far negative tail to large values, to fp32: relative accuracy
    down to where the value leaves fp32's normal range, and zero or the smallest numbers beyond."""
    v = torch.cat([torch.linspace(-16, 16, 8193), torch.tensor([0.0, -0.0, 6e-8, -6e-8, 1e-3, -1e-3, 50, -50, 80, -80, 200, -200, 60000, -60000])]).half()
    x = torch.zeros(v.numel(), 8, dtype=torch.float16)
    x[:, 0] = v
    w = torch.zeros(32, 8, dtype=torch.float16)
    w[:, 0] = 1
    lin = linear_of(ctx, w, None, "f16")
    xd, o = x.cuda(), torch.empty(v.numel(), 32, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    lin.run_dev(xd.data_ptr(), v.numel(), o.data_ptr(), act=act, out_dtype="f32")
    ctx.sync()
    o = o.cpu().double()
    assert (o == o[:, :1]).all()
    y, d = act64(v.double(), act), v.double()
    y = torch.where(torch.isnan(y), torch.zeros_like(y), y)         # 0 * inf of the 64-bit formula's own overflow (tanh form, far left)
    # the fit and its evaluation: 5 units of 2^-24, exp 3, the reciprocals 2, products and the final rounding 4; the exponents' own
    # rounding: gelu carries v^2 exactly, the tanh form's argument has three roundings of |2 u|
    u2 = 1.6 * (d.abs() + 0.044715 * d.abs() ** 3)
    tol = (16 + (3 * u2 if act == "gelu_tanh" else 0)) * 2.0 ** -24 * y.abs() + d.abs() * 2.0 ** -125
    bad = ~((o[:, 0] - y).abs() <= tol)
    assert not bad.any(), (v[bad][:8], o[bad, 0][:8], y[bad][:8])


def test_overflow_rounds_to_infinity(ctx):
    x = torch.full((2, 64), 100.0, dtype=torch.float16)
    w = torch.full((32, 64), 100.0, dtype=torch.float16)
    lin = linear_of(ctx, w, None, "f16")
    o = torch.empty(2, 32, dtype=torch.float16, device="cuda")
    xd = x.cuda()
    torch.cuda.synchronize()
    lin.run_dev(xd.data_ptr(), 2, o.data_ptr())
    ctx.sync()
    assert torch.isinf(o).all()


def test_same_rows_same_bits_and_repeatable(ctx):
    """A pass is repeatable bit for bit."""
    for m, n, k in ((1, 512, 4096), (256, 4096, 4096), (77, 131, 500), (3000, 512, 1024)):
        x, w, b, r = make(m, n, k, "f16", 9, residual="f16")
        lin = linear_of(ctx, w, b, "f16")
        xd, rd = x.cuda(), r.cuda()
        outs = [torch.empty(m, n, dtype=torch.float32, device="cuda") for _ in range(4)]
        torch.cuda.synchronize()
        for o in outs:
            lin.run_dev(xd.data_ptr(), m, o.data_ptr(), act="gelu", residual_dev=rd.data_ptr(), out_dtype="f32")
        ctx.sync()
        for o in outs[1:]:
            assert torch.equal(o, outs[0])


def test_residual_in_place(ctx):
    m, n, k = 150, 256, 512
    x, w, b, r = make(m, n, k, "f16", 21, residual="f16")
    lin = linear_of(ctx, w, b, "f16")
    xd, rd, plain = x.cuda(), r.cuda(), torch.empty(m, n, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    lin.run_dev(xd.data_ptr(), m, plain.data_ptr(), act="silu", residual_dev=rd.data_ptr())
    lin.run_dev(xd.data_ptr(), m, rd.data_ptr(), act="silu", residual_dev=rd.data_ptr())
    ctx.sync()
    assert torch.equal(plain, rd)


def test_two_streams_take_turns(ctx):
    """A context on a torch stream and its own tensors: ordered by that stream alone."""
    from frhot.engine import Context
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c2 = Context(device=0, max_batch=1, stream=s.cuda_stream)
        x, w, b, _ = make(512, 512, 1024, "f16", 5)
        lin = linear_of(c2, w, b, "f16")
        xd = x.cuda()
        acc = torch.zeros(512, 512, device="cuda")
        o = torch.empty(512, 512, dtype=torch.float32, device="cuda")
        for i in range(6):
            xi = xd * (i + 1)
            lin.run_dev(xi.data_ptr(), 512, o.data_ptr(), out_dtype="f32")
            acc += o
        s.synchronize()
    want = sum(layer64((x * (i + 1)), w, b, "none", None)[0] for i in range(6))
    assert (acc.cpu().double() - want).abs().max() <= 6 * 1025 * 2.0 ** -22 * want.abs().max()
    lin.close()
    c2.close()


def test_graph_replays(ctx):
    """Captured once, replayed with new inputs between eager calls: every replay equals the eager answer."""
    from frhot.engine import Context
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c2 = Context(device=0, max_batch=1, stream=s.cuda_stream)
        x, w, b, r = make(64, 512, 4096, "f16", 5, residual="f16")
        lin = linear_of(c2, w, b, "f16")
        xd, rd = x.cuda(), r.cuda()
        o = torch.empty(64, 512, dtype=torch.float32, device="cuda")
        u = torch.empty(64, 512, dtype=torch.float16, device="cuda")
        eo, eu = torch.empty_like(o), torch.empty_like(u)

        def both(o, u):
            lin.run_dev(xd.data_ptr(), 64, o.data_ptr(), act="silu", residual_dev=rd.data_ptr(), out_dtype="f32")
            c2.unit_rows_dev(o.data_ptr(), 64, 512, u.data_ptr())

        both(eo, eu)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        g.capture_begin()
        both(o, u)
        g.capture_end()
        for i in range(5):
            xd.copy_((x * (0.5 + i)).cuda())
            both(eo, eu)
            o.zero_()
            u.zero_()
            g.replay()
            both(eo, eu)
            s.synchronize()
            assert torch.equal(o, eo) and torch.equal(u, eu)
    lin.close()
    c2.close()


def test_two_threads(ctx):
    """Calls of several threads on one context: serialised, each with its own answer."""
    import threading
    jobs = []
    for i, (m, n, k) in enumerate([(256, 1024, 2048), (77, 131, 500), (1, 512, 4096), (300, 64, 64)]):
        x, w, b, _ = make(m, n, k, "f16", 40 + i)
        lin, xd = linear_of(ctx, w, b, "f16"), x.cuda()
        o = [torch.empty(m, n, dtype=torch.float32, device="cuda") for _ in range(8)]
        jobs.append((lin, xd, m, o, layer64(x, w, b, "none", None)))
    torch.cuda.synchronize()

    def go(j):
        lin, xd, m, outs, _ = j
        for o in outs:
            lin.run_dev(xd.data_ptr(), m, o.data_ptr(), out_dtype="f32")

    ts = [threading.Thread(target=go, args=(j,)) for j in jobs]
    [t.start() for t in ts]
    [t.join() for t in ts]
    ctx.sync()
    for lin, _, m, outs, (y, tol) in jobs:
        for o in outs:
            assert ((o.cpu().double() - y).abs() <= tol + rounding(y.abs() + tol, "f32")).all()


def test_refusals(ctx):
    from frhot import FrhotError
    from frhot.engine import Head, Linear
    w = np.zeros((64, 128), np.float16)
    lin = Linear(ctx, w)
    x = torch.zeros(64, 256, dtype=torch.float16, device="cuda")
    o = torch.zeros(64, 256, dtype=torch.float16, device="cuda")

    def refused(code, f, *a, **k):
        with pytest.raises(FrhotError) as e:
            f(*a, **k)
        assert e.value.code == code, e.value
    run = lin.run_dev
    refused(-1, run, 0, 4, o.data_ptr())
    refused(-1, run, x.data_ptr(), 4, 0)
    refused(-1, run, x.data_ptr(), -1, o.data_ptr())
    refused(-1, run, x.data_ptr(), 2 ** 31, o.data_ptr())
    refused(-1, run, x.data_ptr(), 4, o.data_ptr(), ldx=127)
    refused(-1, run, x.data_ptr(), 4, o.data_ptr(), ldo=63)
    refused(-1, run, x.data_ptr(), 4, o.data_ptr(), residual_dev=x.data_ptr(), ldr=63)
    refused(-1, run, x.data_ptr() + 1, 4, o.data_ptr())
    refused(-1, run, x.data_ptr(), 4, o.data_ptr() + 2, out_dtype="f32")
    refused(-1, run, x.data_ptr(), 4, x.data_ptr() + 256)                       # out inside x
    refused(-1, run, x.data_ptr(), 4, o.data_ptr(), residual_dev=o.data_ptr() + 128)
    refused(-1, run, x.data_ptr(), 4, o.data_ptr(), residual_dev=o.data_ptr(), out_dtype="f32", residual_dtype="f16")
    for k in ("act", "out_dtype", "residual_dtype"):
        with pytest.raises(ValueError):
            run(x.data_ptr(), 4, o.data_ptr(), **{k: "f8"})
    assert ctx._lib.frhot_linear_dev(lin.handle, x.data_ptr(), 128, 4, 9, None, 0, 0, o.data_ptr(), 64, 0) == -1
    assert ctx._lib.frhot_linear_dev(lin.handle, x.data_ptr(), 128, 4, 0, None, 0, 0, o.data_ptr(), 64, 3) == -1
    assert ctx._lib.frhot_linear_dev(None, x.data_ptr(), 128, 4, 0, None, 0, 0, o.data_ptr(), 64, 0) == -1
    run(x.data_ptr(), 0, o.data_ptr())                                          # no rows: nothing happens
    run(0, 0, 0)
    for bad in ((0, 4), (4, 0), (65537, 4), (4, 65537)):
        h = C.c_void_p()
        assert ctx._lib.frhot_linear_create(ctx.handle, w.ctypes.data, None, bad[0], bad[1], 0, C.byref(h)) == -1
    with pytest.raises(FrhotError):
        Linear(ctx, w.view(np.uint16), dtype="f32")
    u = ctx.unit_rows_dev
    refused(-1, u, 0, 4, 64, o.data_ptr())
    refused(-1, u, x.data_ptr(), 4, 0, o.data_ptr())
    refused(-1, u, x.data_ptr(), 4, 64, o.data_ptr(), ldx=32)
    refused(-1, u, x.data_ptr(), 4, 64, x.data_ptr(), dtype="f16")
    u(x.data_ptr(), 0, 64, o.data_ptr())
    # heads
    refused(-1, Head, ctx, [])
    refused(-1, Head, ctx, [(lin, "none", True)])                               # 128 -> 64 cannot add its input
    refused(-1, Head, ctx, [(lin, "none", False), (lin, "none", False)])        # 64 does not feed 128
    refused(-1, Head, ctx, [(Linear(ctx, np.zeros((96, 128), np.float16)), "none", False)])
    refused(-1, Head, ctx, [(Linear(ctx, np.zeros((64, 128), np.float32), dtype="bf16"), "none", False)])
    head = Head(ctx, [(lin, "none", False)])
    refused(-1, ctx.set_head, head)                                             # 128 inputs: no descriptor
    refused(-3, lin.close)                                                      # the head holds it
    refused(-1, head.run_dev, x.data_ptr(), 4, x.data_ptr())
    head.run_dev(x.data_ptr(), 0, o.data_ptr())
    head.close()
    lin.close()


# ------------------------------------------------------------------------------------------ unit rows
def check_unit(got, x):
    xd = x.double()
    n = xd.norm(dim=1, keepdim=True)
    y = xd / torch.where(n < 1e-30, torch.ones_like(n), n)
    # the norm and the quotient are rounded to fp32 once each, the result to fp16 once
    tol = y.abs() * 2.0 ** -22 + rounding(y.abs() * (1 + 2.0 ** -22), "f16")
    assert ((got.double() - y).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 7, 16, 63, 64, 65, 100, 128, 255, 256, 320, 512, 1000, 1024, 2047, 4096, 4100, 8192, 10001])
def test_unit_rows(ctx, n, dtype):
    for m, padx, pado in ((1, 0, 0), (5, 3, 1), (67, 8, 8)):
        g = torch.Generator().manual_seed(n + m)
        x = (torch.randn(m, n, generator=g) * 3).to(DT[dtype])
        if m > 1:
            x[1] = 0                                                    # a zero row stays zero
        xb, _ = padded(x, n + padx, 2)
        ob = torch.full(((m + 2) * (n + pado),), 7.0, dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        ctx.unit_rows_dev(xb.data_ptr(), m, n, ob.data_ptr(), dtype=dtype, ldx=n + padx, ldo=n + pado)
        ctx.sync()
        o = ob.view(-1, n + pado).cpu()
        check_unit(o[:m, :n], x)
        assert (o[m:] == 7).all() and (o[:m, n:] == 7).all()


def test_unit_rows_extremes(ctx):
    """Squares that leave fp32's range on either side, infinities and NaN: each row on its own."""
    x = torch.randn(8, 96, generator=torch.Generator().manual_seed(1))
    x[0] *= 1e30
    x[1] *= 1e-25
    x[2] *= 1e-35
    x[3, 5] = NAN
    x[4, 5] = float("inf")
    xd, o = x.cuda(), torch.empty(8, 96, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    ctx.unit_rows_dev(xd.data_ptr(), 8, 96, o.data_ptr())
    ctx.sync()
    o = o.cpu()
    check_unit(o[[0, 1, 5, 6, 7]], x[[0, 1, 5, 6, 7]])
    assert (o[2] == 0).all()                    # shorter than 1e-30: divided by one, below fp16's range
    assert torch.isnan(o[3]).all()
    assert torch.isnan(o[4, 5]) and (o[4, torch.arange(96) != 5] == 0).all()


def test_unit_rows_equal_the_gallerys_own(ctx):
    """The rows a gallery stores for the same floats, bit for bit."""
    from frhot.engine import Gallery
    x = torch.randn(300, 512, generator=torch.Generator().manual_seed(8))
    gal = Gallery(ctx, 512, 300)
    gal.upsert(x.numpy(), 0, np.arange(300))
    stored, _ = gal.read(np.arange(300))
    xd, o = x.cuda(), torch.empty(300, 512, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    ctx.unit_rows_dev(xd.data_ptr(), 300, 512, o.data_ptr())
    ctx.sync()
    assert np.array_equal(o.cpu().numpy(), stored)
    gal.close()


# ------------------------------------------------------------------------------------------ heads
def head_layers(dims, acts, res, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i in range(len(dims) - 1):
        w = (torch.randn(dims[i + 1], dims[i], generator=g) * (2.0 if i == 0 else 1.0) / math.sqrt(dims[i])).half()
        out.append((w, torch.randn(dims[i + 1], generator=g) * 0.2, acts[i], res[i]))
    return out


def head64(x, layers):
    """(unit rows, tolerance): inner layers round to fp16, so each layer's inputs carry half a step, which reaches the
    output through the magnitudes of the weights."""
    v, err = x.double(), torch.zeros_like(x, dtype=torch.float64)
    for i, (w, b, act, res) in enumerate(layers):
        y, tol = layer64(v, w, b, act, v if res else None)
        tol = tol + 1.13 * err @ w.double().abs().t() + (err if res else 0)
        if i < len(layers) - 1:
            tol = tol + rounding(y.abs() + tol, "f16")
        v, err = y, tol
    n = v.norm(dim=1, keepdim=True)
    u = v / n
    return u, err / n + u.abs() * (err.norm(dim=1, keepdim=True) / n) + 2.0 ** -22 * u.abs() + rounding(u.abs(), "f16")


@pytest.mark.parametrize("dims,acts,res", [([4096, 512], ["none"], [0]), ([256, 320, 64], ["gelu", "none"], [0, 0]),
                                           ([512, 512], ["silu"], [1]), ([128, 128, 200, 200, 64], ["relu", "none", "silu", "none"], [1, 0, 1, 0])])
@pytest.mark.parametrize("m", [1, 50, 2100])
def test_heads(ctx, dims, acts, res, m):
    from frhot.engine import Head
    layers = head_layers(dims, acts, res)
    lins = [linear_of(ctx, w, b, "f16") for w, b, _, _ in layers]
    head = Head(ctx, [(l, a, r) for l, (_, _, a, r) in zip(lins, layers)])
    x = torch.randn(m, dims[0], generator=torch.Generator().manual_seed(m)).clamp_min(0)
    x = (x / x.norm(dim=1, keepdim=True)).half()
    xb, _ = padded(x, dims[0] + 8, 1)
    ob = torch.full((m + 1, dims[-1] + 8), 7.0, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    head.run_dev(xb.data_ptr(), m, ob.data_ptr(), ldx=dims[0] + 8, ldo=dims[-1] + 8)
    ctx.sync()
    o = ob.cpu()
    want, tol = head64(x, layers)
    assert ((o[:m, :dims[-1]].double() - want).abs() <= tol).all()
    assert (o[m:] == 7).all() and (o[:, dims[-1]:] == 7).all()
    head.close()
    [l.close() for l in lins]


def test_recognise_through_a_head(gpu_ctx):
    """Embed -> head -> search in one call: the same scores and rows as the pieces by hand; detached, the leading
    components are back."""
    from frhot import synth
    from frhot.engine import Context, Gallery, Head
    crops = synth.crops(seed=4, n=6, lo=90, hi=200)
    layers = head_layers([4096, 640, 256], ["silu", "none"], [0, 0], seed=2)
    lins = [linear_of(gpu_ctx, w, b, "f16") for w, b, _, _ in layers]
    head = Head(gpu_ctx, [(l, a, r) for l, (_, _, a, r) in zip(lins, layers)])
    emb = torch.from_numpy(gpu_ctx.embed(crops)).half()
    gal = Gallery(gpu_ctx, 256, 700)
    other = torch.randn(700, 256, generator=torch.Generator().manual_seed(3))
    gal.upsert(other.numpy(), 0, np.arange(700))
    before = gpu_ctx.recognise(gal, crops, None, 5)
    ed, q = emb.cuda(), torch.empty(6, 256, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    head.run_dev(ed.data_ptr(), 6, q.data_ptr())
    gpu_ctx.sync()
    want, tol = head64(emb, layers)
    assert ((q.cpu().double() - want).abs() <= tol).all()
    keys = np.zeros(6, np.int32)
    gal.write_dev(q.data_ptr(), np.arange(6) * 100, None, keys)            # enrol the six faces' head rows
    gpu_ctx.set_head(head)
    try:
        s, r, _ = gpu_ctx.recognise(gal, crops, None, 5)
        assert np.array_equal(r[:, 0], np.arange(6) * 100)
        assert np.abs(s[:, 0] - 1).max() <= 1e-3
        buf, off, hw, st = synth.pack_crops(crops)
        pix, q2 = torch.from_numpy(buf).cuda(), torch.empty_like(q)
        full = torch.empty(6, 4096, dtype=torch.float32, device="cuda")
        torch.cuda.synchronize()
        gpu_ctx.embed_dev(pix.data_ptr(), off, hw, st, Context.flags(), full.data_ptr(), q2.data_ptr(), 256)
        gpu_ctx.sync()
        assert torch.equal(q2, q), "embed_dev through the head = the head on the embedding"
        assert np.array_equal(full.cpu().numpy(), gpu_ctx.embed(crops)), "the descriptors themselves do not change"
        q3 = torch.empty(6, 512, dtype=torch.float16, device="cuda")
        gpu_ctx.embed_dev(pix.data_ptr(), off, hw, st, Context.flags(), None, q3.data_ptr(), 512)   # another width: leading components
        gpu_ctx.sync()
        lead = emb.double()[:, :512]
        assert (q3.cpu().double() - lead / lead.norm(dim=1, keepdim=True)).abs().max() <= 2.0 ** -10
    finally:
        gpu_ctx.set_head(None)
    gal.upsert(other[::100][:6].numpy(), 0, np.arange(6) * 100)
    after = gpu_ctx.recognise(gal, crops, None, 5)
    assert np.array_equal(before[0], after[0]) and np.array_equal(before[1], after[1])
    gpu_ctx.set_head(head)
    head.close()                                                            # detaches itself
    again = gpu_ctx.recognise(gal, crops, None, 5)
    assert np.array_equal(before[1], again[1])
    gal.close()
    [l.close() for l in lins]


def test_more_rows_than_a_launch_has_threads(ctx):
    """Calls whose rows times lanes pass 2^32 are several launches.  Small whole numbers: the products are exact."""
    gen = torch.Generator("cuda").manual_seed(8)
    m = (1 << 26) + 17
    x = torch.randint(-2, 3, (m, 8), generator=gen, device="cuda", dtype=torch.int8).to(torch.float16)
    w = torch.randint(-2, 3, (2, 8), generator=gen, device="cuda").float()
    lin = linear_of(ctx, w.cpu(), torch.tensor([1.0, -3.0]), "f16")
    o = torch.empty(m, 2, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    lin.run_dev(x.data_ptr(), m, o.data_ptr())
    ctx.sync()
    for lo in range(0, m, 1 << 24):
        part = x[lo:lo + (1 << 24)].float()
        want = torch.stack([(part * w[i]).sum(1) for i in range(2)], 1) + torch.tensor([1.0, -3.0], device="cuda")
        assert torch.equal(o[lo:lo + (1 << 24)].float(), want), lo
    lin.close()
    del o, w
    m = (1 << 30) + 3
    x = torch.randint(-2, 3, (m,), generator=gen, device="cuda", dtype=torch.int8).to(torch.float16)
    o = torch.full((m,), 7.0, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    ctx.unit_rows_dev(x.data_ptr(), m, 1, o.data_ptr(), dtype="f16")
    ctx.sync()
    for lo in range(0, m, 1 << 28):
        assert torch.equal(o[lo:lo + (1 << 28)], torch.sign(x[lo:lo + (1 << 28)])), lo
    del x, o
    torch.cuda.empty_cache()


@pytest.mark.parametrize("ld", [(1 << 30) + 8, (1 << 30) + 3])
def test_rows_gigabytes_apart(ctx, ld):
    """Row offsets past 2^32 bytes, on both sides, for rows that LDS-DMA takes and rows that it cannot."""
    m, n, k = 4, 40, 136
    x, w, b, r = make(m, n, k, "f16", 5, residual="f16")
    lin = linear_of(ctx, w, b, "f16")
    big = torch.zeros(3 * ld + 256, dtype=torch.float16, device="cuda")
    out = torch.zeros(3 * ld + 256, dtype=torch.float16, device="cuda")
    for i in range(m):
        big[i * ld:i * ld + k] = x[i].cuda()
        out[i * ld:i * ld + n] = r[i].cuda()            # (the residual, replaced by the result)
        out[i * ld + n] = 7.0
    torch.cuda.synchronize()
    lin.run_dev(big.data_ptr(), m, out.data_ptr(), act="gelu", residual_dev=out.data_ptr(), ldx=ld, ldr=ld, ldo=ld)
    ctx.sync()
    y, tol = layer64(x, w, b, "gelu", r)
    tol = tol + rounding(y.abs() + tol, "f16")
    got = torch.stack([out[i * ld:i * ld + n] for i in range(m)]).cpu().double()
    assert ((got - y).abs() <= tol).all()
    assert all(out[i * ld + n] == 7 for i in range(m))
    torch.cuda.synchronize()
    ctx.unit_rows_dev(big.data_ptr(), m, k, out.data_ptr(), dtype="f16", ldx=ld, ldo=ld)
    ctx.sync()
    check_unit(torch.stack([out[i * ld:i * ld + k] for i in range(m)]).cpu(), x)
    lin.close()
    del big, out
    torch.cuda.empty_cache()


def test_a_layer_twice_in_a_head_and_in_a_graph(ctx):
    """One layer used twice by a head; the head replayed from a graph where its products are split over K."""
    from frhot.engine import Context, Head
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c2 = Context(device=0, max_batch=1, stream=s.cuda_stream)
        _, w, b, _ = make(1, 640, 640, "f16", 12)
        _, w2, b2, _ = make(1, 64, 640, "f16", 13)
        l1, l2 = linear_of(c2, w, b, "f16"), linear_of(c2, w2, b2, "f16")
        head = Head(c2, [(l1, "silu", True), (l1, "none", True), (l2, "none", False)])
        layers = [(w, b, "silu", True), (w, b, "none", True), (w2, b2, "none", False)]
        m = 260
        x = torch.randn(m, 643, generator=torch.Generator().manual_seed(2)).half()      # (odd row distance)
        xd, o = x.cuda(), torch.zeros(m, 64, dtype=torch.float16, device="cuda")
        e = torch.zeros_like(o)
        head.run_dev(xd.data_ptr(), m, e.data_ptr(), ldx=643)
        s.synchronize()
        want, tol = head64(x[:, :640], layers)
        assert ((e.cpu().double() - want).abs() <= tol).all()
        g = torch.cuda.CUDAGraph()
        g.capture_begin()
        head.run_dev(xd.data_ptr(), m, o.data_ptr(), ldx=643)
        g.capture_end()
        for i in range(4):
            xd.copy_((x * (1 + i)).cuda())
            head.run_dev(xd.data_ptr(), m, e.data_ptr(), ldx=643)
            o.zero_()
            g.replay()
            s.synchronize()
            assert torch.equal(o, e)
        head.close()
        l1.close(), l2.close(), c2.close()
