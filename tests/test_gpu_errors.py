"""A call that fails leaves nothing behind for the calls after it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_an_allocation_that_fails_is_not_reported_again():
    from frhot import FrhotError
    from frhot.engine import Context, Gallery, Head, Linear
    ctx = Context(device=0, max_batch=1)
    gal = Gallery(ctx, 64, 300)
    calls = (lambda: gal.fill_synthetic(1, 0, 300), lambda: gal.search(np.ones((1, 64), np.float32), None, 1),
             lambda: gal.copy([0], [100], [50], 3), lambda: gal.compact(), lambda: gal.free_keys([3]),
             lambda: Linear(ctx, np.eye(64, dtype=np.float32)).close(),
             lambda: Head(ctx, [(Linear(ctx, np.eye(64, dtype=np.float32)), "none", False)]).apply(np.ones((1, 64), np.float32)))
    for call in calls:
        with pytest.raises(FrhotError) as e:
            Gallery(ctx, 8192, 0x7fffff00)              # 32 TiB
        assert e.value.code == -2
        call()
    gal.close()
    ctx.close()
