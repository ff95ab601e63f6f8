"""A service's copy and squeeze when the device's part of them fails, over the numpy stand-in."""
import numpy as np

from test_pages_cpu import check_tables, enrol, found, service


def test_a_copy_that_fails_on_the_device_leaves_no_live_rows():
    rng = np.random.default_rng(0)
    svc = service()
    vs = enrol(svc, rng, "A_Employees", 40)
    plain = svc.gallery.copy

    def late(*a, **k):
        plain(*a, **k)
        raise RuntimeError("reported after the rows were written")
    svc.gallery.copy = late
    assert svc.copy_collection("A_Employees", "B_Employees") == (404, {"message": "reported after the rows were written"})
    check_tables(svc)
    assert svc.search_point("B_Employees", vs[0][0], 1)[0] == 404       # the target was not created
    assert found(svc, "A_Employees", *vs[7]) == "p7"
    svc.gallery.copy = plain
    assert svc.copy_collection("A_Employees", "B_Employees")[0] == 201
    check_tables(svc)
