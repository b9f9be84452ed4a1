"""fork_pages and compact_pages at the sizes up to which one workgroup does all
but the copies, and just past them: the same results from both ways."""
import numpy as np
import pytest

from tests.branch_util import Pages, caches_of
from tests.test_gpu_branch_compact import check as check_compact
from tests.test_gpu_branch_fork import check as check_fork

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sources,rows,width", [(16, 16, 64), (15, 16, 66), (16, 16, 65), (1, 1, 1024), (1, 1, 1025),
                                                (1024, 1024, 1), (1024, 1025, 1), (20, 82, 20), (82, 21, 20)])
def test_fork_around_2048_entries(sources, rows, width):
    rng = np.random.default_rng([sources, rows, width])
    p = Pages(rng, rng.integers(0, 4 * width + 1, sources), 1, 4, spare=rows, width=width)
    parents = rng.integers(-1, sources, rows)
    check_fork(p, parents, caches_of(rng, p, 2, 1, 8))


@pytest.mark.parametrize("rows,width,spare", [(128, 64, 300), (128, 128, 9), (129, 128, 9), (127, 129, 40),
                                              (1, 16384, 100), (1, 16385, 100), (16384, 1, 3000), (91, 180, 5000)])
def test_compact_around_16384_entries(rows, width, spare):
    rng = np.random.default_rng([rows, width])
    p = Pages(rng, rng.integers(0, width + 1, rows) if width > 1 else rng.integers(0, 2, rows), 1, 1, spare=spare,
              first=3, width=width)
    check_compact(p, caches_of(rng, p, 1, 1, 8))
