"""Windows and trees over the paged cache, the same tests as
test_gpu_paged_sees.py and test_gpu_paged_sees_odd.py at sizes whose rows times
cells, or pairs of 16 rows and a sequence, are beyond what goes to the kernel of
few rows: all of these run the kernel of many rows."""
import numpy as np
import pytest

from tests import test_gpu_paged_sees as S
from tests import test_gpu_paged_sees_odd as O

pytestmark = pytest.mark.gpu

WINDOWS = [
    # lens, counts, T, Hq, Hkv, P, heads_first, sinks, cap, window, first
    ([345, 200], None, 150, 96, 8, 16, True, False, 0.0, 50, 4),
    ([190, 150, 140], None, 140, 96, 4, 64, False, False, 15.0, 12, 0),
    ([500, 333], [500, 20], 500, 16, 2, 48, False, True, 0.0, 100, 40),
    ([600], None, 600, 16, 4, 16, False, False, 0.0, 64, 10),
    ([2000, 1500], [100, 70], 100, 32, 8, 16, False, False, 0.0, 1900, 90),
    ([40, 30, 600, 1, 0], [200, 40, 200, 4, 0], 200, 32, 4, 16, False, False, 0.0, 17, 2),
]
TREES = [
    # lens, counts, T, Hq, Hkv, P, heads_first, sinks, cap
    ([500, 120, 170], [133, 1, 0], 133, 96, 8, 24, True, True, 0.0),
    ([164, 1000], [161, 164], 164, 96, 8, 32, False, False, 20.0),
    ([300, 277], [200, 165], 200, 64, 2, 16, False, True, 0.0),
]
SHARES = [(100, 24, 4, [100, 1, 7, 33], 2500), (100, 24, 4, [9, 0, 32, 20], 2500), (300, 24, 2, [5], 4000), (300, 24, 2, [300], 2000)]


@pytest.mark.parametrize("i", range(len(WINDOWS)))
def test_windows(gpu, monkeypatch, i):
    monkeypatch.setattr(S, "WINDOWS", WINDOWS)
    S.test_windows(gpu, i)


@pytest.mark.parametrize("window, first", [(0, 0), (40, 5), (3, 0), (1, 20)])
@pytest.mark.parametrize("i", range(len(TREES)))
def test_trees(gpu, monkeypatch, i, window, first):
    monkeypatch.setattr(S, "TREES", TREES)
    S.test_trees(gpu, i, window, first)


def test_what_a_row_does_not_see_does_not_reach_it(gpu):
    S.test_what_a_row_does_not_see_does_not_reach_it(gpu, 90, 192, 4)


@pytest.mark.parametrize("kind", ["window", "tree"])
@pytest.mark.parametrize("sinks", [None, 0.5])
def test_logits_that_overflow(gpu, kind, sinks):
    O.test_logits_that_overflow(gpu, 3000, 340, 8, 2, kind, sinks)


@pytest.mark.parametrize("kind", ["window", "tree", "both"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_odd_values_reach_the_rows_that_see_them(gpu, value, kind):
    O.test_odd_values_reach_the_rows_that_see_them(gpu, value, 60, 192, 4, kind)


@pytest.mark.parametrize("size, scale", [(1e-30, 0.2e30), (3e4, 0.2 / 3e4), (1e30, 0.2e-30), (1, -0.125), (1, 0.0), (1e-12, 1e-12)])
def test_scales_and_rows_of_any_size(gpu, size, scale):
    O.test_scales_and_rows_of_any_size(gpu, size, scale, 150, 96, 4)


def test_a_scale_that_is_no_number(gpu):
    O.test_a_scale_that_is_no_number(gpu, 340, 40, 4)


@pytest.mark.parametrize("apart", [5 * 2 ** 29, 5 * 2 ** 30])
def test_strided_operands_and_offsets_past_32_bits(gpu, apart):
    O.test_strided_operands_and_offsets_past_32_bits(gpu, 150, 96, 4, apart)


def test_negative_counts_are_reported(gpu):
    O.test_negative_counts_are_reported(gpu, 70, 66, 45, 24, 2)


@pytest.mark.parametrize("n, T, Hq, Hkv, window", [(70, 40, 32, 8, 30), (40, 70, 24, 2, 20)])
def test_many_sequences_of_many_rows(gpu, n, T, Hq, Hkv, window):
    O.test_many_sequences_of_many_rows(gpu, n, T, Hq, Hkv, window)


@pytest.mark.parametrize("i", range(len(SHARES)))
@pytest.mark.parametrize("window, first", [(0, 0), (700, 3)])
def test_row_groups_of_sequences_that_differ(gpu, monkeypatch, i, window, first):
    monkeypatch.setattr(O, "SHARES", SHARES)
    O.test_row_groups_of_sequences_that_differ(gpu, i, window, first)
