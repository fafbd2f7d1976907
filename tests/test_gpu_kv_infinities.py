"""Heads of a page that hold infinities and no finite number but 0: what they read as does not depend on how the page is changed afterwards."""
import pytest
import torch

from test_gpu_kv_cache import Pair

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def rows(p, n, at, finite):
    """n rows of numbers, those in `at` without a finite one other than 0 in head 0's keys and head 1's values."""
    k, v = p.rows(n), p.rows(n)
    k[at, 0], v[at, 1] = (0.0 if finite else NAN), (0.0 if finite else NAN)
    k[at, 0, 3::5], v[at, 1, ::7] = INF, -INF
    return [(k, v)] * p.layers


@pytest.mark.parametrize("finite", [True, False])
@pytest.mark.parametrize("n_pages", [400, 4])            # kept into new pages; in place
@pytest.mark.parametrize("codes", [0, 1])
def test_kept_beside_numbers(codes, n_pages, finite):
    p = Pair(4, 2, 64, 16, codes, "f32", n_pages=n_pages)
    p.step([0], [64], rows=rows(p, 64, slice(16, 32), finite))
    p.check_numbers([0])
    index = list(range(20, 40)) + [50, 63]               # half of the second page's tokens meet the third's
    p.kv.keep(0, 0, index)
    for r in p.ref:
        r.keep(0, 0, index)
    p.check_numbers([0])
    assert p.kv.status() == 32


@pytest.mark.parametrize("codes", [0, 1])
def test_appended_to(codes):
    p = Pair(4, 2, 64, 32, codes, "f32")
    p.step([0], [7], rows=rows(p, 7, slice(0, 7), True))
    p.check_numbers([0])
    p.step([0], [20])
    p.check_numbers([0])
    p.step([0], [3], rows=rows(p, 3, slice(0, 3), True))     # the scale is there: the largest code
    p.check_numbers([0])


@pytest.mark.parametrize("counts", [[1], [900]])        # the kernel for few rows, and the one for prompts
def test_values_that_read_as_nothing_weigh_nothing(counts):
    p = Pair(4, 2, 64, 16, 0, "f32")
    k, v = p.rows(16), torch.full((16, 2, 64), INF)
    p.step([0], [16], rows=[(k, v)] * 2)
    p.step([0], counts)
    p.check_attend([0], counts)
