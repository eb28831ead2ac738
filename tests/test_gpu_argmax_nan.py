"""The greedy choice over logits that are not numbers."""
import numpy as np
import pytest

from gpu_util import Dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", ["one", "two", "all", "behind", "infinities", "lowest"])
def test_argmax_of_logits_that_are_not_numbers(hv, case):
    """np.argmax's order: the first NaN, whatever else there is; a token in any case, whose row the
    next step reads."""
    n = 5003
    x = np.random.default_rng(3).standard_normal(n).astype(np.float32)
    if case == "one":
        x[1234] = np.nan
    if case == "two":
        x[[40, 4999]] = np.nan
    if case == "all":
        x[:] = np.nan
    if case == "behind":
        x[17], x[-1] = np.inf, np.nan
    if case == "infinities":
        x[:] = -np.inf
        x[[7, 9]] = np.inf
    if case == "lowest":
        x[:] = -np.inf
    pv, pi = Dev(nbytes=128 * 4), Dev(nbytes=128 * 4)
    tok, step, pos, gen = (Dev(np.zeros(4, np.int32)) for _ in range(4))
    hv.argmax_partial(Dev(x), pv, pi, n, 128)
    hv.argmax_final(pv, pi, tok, gen, step, pos, 128)
    assert tok.get(np.int32)[0] == gen.get(np.int32)[0] == np.argmax(x)
