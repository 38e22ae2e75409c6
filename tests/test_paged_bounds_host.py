"""CPU tests: bounds whose pages overlap are refused where they are written."""

from test_paged_host import D, _refused, i64

ST = [2048, 1024, 64, 32, 16, 1]


def test_bounds_of_pages_that_overlap():
    """Workgroups of several pages would write one place."""
    good = [D, D, D, D, D, D, 3, 2, 64, 4, 2, 2, 16, 2, i64(*ST), i64(256, 128), None]
    _refused("sparkq_paged_key_bounds", good, [
        (15, i64(0, 128), -1, "overlap"), (15, i64(120, 1024), -1, "overlap")])
