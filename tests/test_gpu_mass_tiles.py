"""Weights added up by tiles where CTAs go from two tiles of positions at a time to single ones and back,
over odd numbers of tiles of rows."""
import numpy as np
import pytest

import span_ref as R
from test_gpu_shared import check_mass, queries, cache, run_mass, SCALE

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nkv,group,pos0,ntok", [
    (256, 1, 150, 129),              # 3 tiles of positions a head, 2 of rows: 5 units a CTA
    (192, 1, 0, 300),                # 3 of both, later positions have fewer
    (200, 1, 0, 140),                # 2 and 2
    (120, 2, 512, 128)])             # 5 tiles of positions, 2 of rows
def test_units_of_one_and_two_tiles(hv, nkv, group, pos0, ntok):
    g = np.random.default_rng(nkv)
    check_mass(hv, g, nkv, group, pos0, ntok, pos0 + ntok + 3, False, "same")


def test_repeats_of_many_units_are_equal(hv):
    g = np.random.default_rng(9)
    nkv, pos0, ntok = 200, 300, 130
    k, v = cache(g, nkv, pos0 + ntok)
    q = queries(g, ntok, nkv)
    first = run_mass(hv, q, k, v, pos0, None, False)
    for _ in range(5):
        again = run_mass(hv, q, k, v, pos0, None, False)
        for a, b in zip(first, again):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
