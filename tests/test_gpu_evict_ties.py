"""Slices in which nearly all weights are equal, of the longest tables taken."""
import pytest

from test_gpu_evict import check, kvr, make  # noqa: F401  (kvr: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[320000], [40000], [39999, 320000, 100]])
@pytest.mark.parametrize("keep,recent,first", [(1000, 100, 4), (200000, 0, 0)])
def test_long_slices_of_ties(kvr, lengths, keep, recent, first):  # noqa: F811
    check(kvr, make(lengths, 1, 8, 64, keep, seed=1, weights="equal"), keep, recent, first)
