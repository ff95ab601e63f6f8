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


def test_a_squeeze_that_the_device_does_not_agree_with_moves_nothing():
    """A table row that is dead on the device (a tombstone that reported an error once its kernel had run): the squeeze is
    refused while nothing has moved; searches go on; with the point deleted it goes through."""
    rng = np.random.default_rng(1)
    svc = service()
    vs = enrol(svc, rng, "A_Employees", 30, stores=(1,))
    row = next(r for r, p in svc._points.items() if p["payload"]["id"] == "p4")
    svc.gallery.keys[row] = -1
    before = svc.gallery.keys.copy()
    status, content = svc.compact()
    assert status == 404 and "nothing was moved" in content["message"]
    assert np.array_equal(svc.gallery.keys, before)
    for i in (0, 3, 5, 29):
        assert found(svc, "A_Employees", *vs[i]) == f"p{i}"
    assert svc.insert_point("A_Employees", vs[0][0], "new", "n", 1)[0] == 201
    assert found(svc, "A_Employees", *vs[29]) == "p29"
    svc.delete_point("A_Employees", "p4")
    assert svc.compact() == (200, {"message": "Gallery compacted", "points": 30})
    check_tables(svc)
    assert found(svc, "A_Employees", *vs[29]) == "p29"
    # rows under a wrong key, and a table that is longer than the gallery
    svc.gallery.keys[3] = 77
    assert svc.compact()[0] == 404
    svc.gallery.keys[3] = 0
    rows, svc.gallery.nrows = svc.gallery.nrows, 20
    assert svc.compact()[0] == 404
    svc.gallery.nrows = rows
    assert svc.compact()[0] == 200


def test_a_squeeze_kills_only_what_is_alive():
    """Rows that are dead already do not go through host lists again."""
    rng = np.random.default_rng(2)
    svc = service()
    enrol(svc, rng, "A_Employees", 60, stores=(1,))
    for i in range(0, 50):
        svc.delete_point("A_Employees", f"p{i}")
    killed, plain = [], svc.gallery.tombstone

    def tombstone(rows):
        killed.extend(np.asarray(rows).tolist())
        plain(rows)
    svc.gallery.tombstone = tombstone
    svc.gallery.keys[61], svc.gallery.nrows = 0, 62
    assert svc.compact() == (200, {"message": "Gallery compacted", "points": 10})
    assert killed == [61]
    check_tables(svc)
