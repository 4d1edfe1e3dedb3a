"""Whether two runs of rows share memory, against a set of the addresses that they have."""

import random

from flydsl_b200.row_ops import _share


def addresses(span):
    at, rows, step, width = span
    return {at + r * step + i for r in range(rows) for i in range(width)}


def test_shared_addresses_are_always_found():
    rng = random.Random(1)
    for _ in range(20000):
        spans = []
        for _ in range(2):
            width, rows = rng.randint(1, 6), rng.randint(0, 4)
            spans.append((rng.randint(0, 40), rows, rng.randint(6, 14) if rows > 1 else 0, width))
        assert _share(*spans) or not addresses(spans[0]) & addresses(spans[1]), spans


def test_columns_of_one_buffer_and_single_rows_between_are_apart():
    rng = random.Random(2)
    for _ in range(20000):
        step, rows = rng.randint(2, 14), rng.randint(2, 5)
        a = (rng.randint(0, 20), rows, step, rng.randint(1, step - 1))
        width = rng.randint(1, step)
        for b in ((a[0] + rng.randint(1 - step, step - 1), rows, step, width), (a[0] + rng.randint(-20, 80), 1, 0, width)):
            assert _share(a, b) == _share(b, a) == bool(addresses(a) & addresses(b)), (a, b)


def test_rows_of_two_distances_are_told_apart_by_their_ranges():
    assert _share((0, 4, 10, 2), (4, 4, 12, 2)) and not _share((0, 4, 10, 2), (32, 4, 12, 2)) and not _share((32, 4, 10, 2), (0, 3, 14, 4))
