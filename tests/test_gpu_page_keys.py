"""A gallery's keys read by themselves."""
import numpy as np
import pytest

from test_gpu_pages import DEAD, Pair, ctx      # noqa: F401  (ctx: the fixture)

pytestmark = pytest.mark.gpu


def test_read_keys(ctx):                         # noqa: F811
    from frhot import FrhotError
    p = Pair(ctx, 64, 1000, 700, seed=3)
    p.gal.tombstone(np.arange(5, 600, 7))
    p.k[5:600:7] = DEAD
    assert np.array_equal(p.gal.read_keys(), p.k[:700])
    for lo, n in ((0, 1000), (999, 1), (255, 2), (0, 1), (300, 257)):
        assert np.array_equal(p.gal.read_keys(lo, n), p.k[lo:lo + n])
    for lo, n in ((-1, 5), (990, 11), (1000, 1), (0, 1001)):
        with pytest.raises(FrhotError) as e:
            p.gal.read_keys(lo, n)
        assert e.value.code == -4
    assert ctx._lib.frhot_gallery_read_keys(p.gal.handle, 0, 5, None) == -1
    assert p.gal.read_keys(0, 0).size == 0
    p.gal.close()
