"""The choice among more than 32768 pages, whose keys no workgroup holds: ties over all of the table, pages that are not there, fewer pages than are asked for, what is not finite."""
import math

import pytest
import torch

import test_gpu_paged_sparse_limits as limits
from test_gpu_paged_sparse import a_choice, choose_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hkv,group,width", [(5, 2, 2, 32769), (9, 1, 1, 40000), (3, 2, 5, 65537)])
def test_select_of_long_tables(gpu, B, Hkv, group, width):
    """Any sequences over a pool of few pages."""
    limits.test_select_of_many_sequences(gpu, B, Hkv, group, width)


PAGES = 40000


def a_long_choice(gpu, kinds, seed):
    """Sequences of 40000 pages, of 33000 and of 3 over a pool of `kinds` pages."""
    q, bounds, _, lens = a_choice(gpu, [16 * PAGES, 16 * 33000 - 7, 40], 4, 2, 64, 16, seed=seed, width=PAGES)
    gen = torch.Generator().manual_seed(seed)
    return q, bounds[:kinds].contiguous(), torch.randint(0, kinds, (3, PAGES), generator=gen, dtype=torch.int32).to(gpu), lens


@pytest.mark.parametrize("kinds", [1, 2, 60])
def test_long_ties(gpu, kinds):
    """All scores equal, or of few values: those in front are chosen, over any number of the kernel's stretches."""
    print("ties", kinds, flush=True)
    q, bounds, table, lens = a_long_choice(gpu, kinds, kinds)
    for count, first, last in ((1, 0, 0), (20, 1, 1), (1024, 0, 0), (1025, 0, 1), (20000, 3, 9), (PAGES - 1, 0, 0), (PAGES, 1, 1)):
        got = choose_and_check(q, bounds, table, lens, 16, count, first, last)
        if kinds == 1 and (first, last) == (0, 0):
            assert got[0, 0].tolist() == list(range(count))


def test_long_tables_with_pages_that_are_not_there(gpu):
    """Every other entry outside the pool; more asked for than there are; none at all."""
    q, bounds, table, lens = a_long_choice(gpu, 60, 5)
    table[0, ::2], table[1, 5::3], table[2, :] = -1, bounds.shape[0], -(2**31)
    for count, first, last in ((1, 0, 0), (500, 2, 3), (PAGES // 2, 0, 1), (PAGES // 2 + 1, 0, 0), (PAGES, 5, 5), (PAGES + 3000, 0, 0)):
        got = choose_and_check(q, bounds, table, lens, 16, count, first, last)
        assert (got[2] == -1).all()


def test_long_tables_of_what_is_not_finite(gpu):
    """Pages whose bounds are not finite come before all others, and tie; a query that is not finite ties all pages."""
    q, bounds, table, lens = a_long_choice(gpu, 200, 6)
    bounds[7, :, 0, 3], bounds[11, 0, 1, 9], bounds[12, 1, 0, 0] = math.nan, math.inf, -math.inf
    for count in (30, 300, 2000):
        choose_and_check(q, bounds, table, lens, 16, count, 1, 1)
    q[1, 1, 5] = math.nan
    got = choose_and_check(q, bounds, table, lens, 16, 300, 0, 0)
    assert got[1, 0].tolist() == list(range(300))
