"""Heads and layers while a graph is captured on their stream."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_creating_and_destroying_are_refused_under_capture():
    """The calls leave the capture as they found it: it goes on, replays, and the refused calls work afterwards."""
    from frhot import FrhotError
    from frhot.engine import Context, Gallery, Head, Linear
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = Context(device=0, max_batch=1, stream=s.cuda_stream)
        lin, spare = Linear(c, np.eye(64, dtype=np.float32)), Linear(c, np.eye(64, dtype=np.float32))
        head, spare_head = Head(c, [(lin, "none", False)]), Head(c, [(lin, "relu", False)])
        wide = Linear(c, np.eye(64, 4096, dtype=np.float32))
        taker = Head(c, [(wide, "none", False)])
        gal = Gallery(c, 64, 300)
        x, out = torch.randn(5, 64, device="cuda").half(), torch.zeros(5, 64, dtype=torch.float16, device="cuda")
        head.run_dev(x.data_ptr(), 5, out.data_ptr())
        s.synchronize()
        want = out.clone()
        g = torch.cuda.CUDAGraph()
        g.capture_begin()
        for call in (lambda: Linear(c, np.eye(64, dtype=np.float32)), lambda: spare.close(), lambda: Head(c, [(lin, "none", False)]),
                     lambda: spare_head.close(), lambda: c.set_head(taker), lambda: c.set_head(None), lambda: gal.set_head(taker),
                     lambda: head.apply(np.ones((1, 64), np.float32)), lambda: head.project(np.ones((1, 64), np.float32)),
                     lambda: gal.read_keys(0, 5)):
            with pytest.raises(FrhotError) as e:
                call()
            assert e.value.code == -3
        head.run_dev(x.data_ptr(), 5, out.data_ptr())
        g.capture_end()
        for i in range(3):
            out.zero_()
            g.replay()
            s.synchronize()
            assert torch.equal(out, want)
        spare_head.close(), spare.close()
        gal.set_head(taker), c.set_head(taker), c.set_head(None)
        gal.close(), taker.close(), wide.close(), head.close(), lin.close(), c.close()


def test_the_first_layer_of_a_context_is_refused_under_capture():
    """It would allocate the context's scratch."""
    from frhot import FrhotError
    from frhot.engine import Context, Linear
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = Context(device=0, max_batch=1, stream=s.cuda_stream)
        x, y = torch.ones(4, device="cuda"), torch.zeros(4, device="cuda")
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        g.capture_begin()
        with pytest.raises(FrhotError) as e:
            Linear(c, np.eye(64, dtype=np.float32))
        assert e.value.code == -3
        y.copy_(x)
        g.capture_end()
        g.replay()
        s.synchronize()
        assert (y == 1).all()
        Linear(c, np.eye(64, dtype=np.float32)).close()
        c.close()
