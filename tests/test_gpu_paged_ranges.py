"""8-bit pages whose rows differ in size by many powers of two: every token's result keeps the bits of the rows that it sees."""
import math

import pytest
import torch

from tests.paged_cases import Case

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def api():
    from vqtree_b200 import api as _api
    return _api


def _grow(c, s, at, factor):
    """Value row ``at`` of sequence s times a factor (its scale, that is)."""
    c.scales[2][c.table[s, at // c.P], :, at % c.P] *= factor
    c.dense[s][2][at] *= factor


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
# few tokens; a chunk converted on the way; one through the workspace
@pytest.mark.parametrize("qs,lens,G", [((1, 3), (300, 500), 4), ((40, 140), (300, 800), 2), ((300, 700), (300, 900), 4)])
@pytest.mark.parametrize("size,factor", [(1e-3, 1e7), (1e-4, 1e8)])
def test_a_large_value_row_costs_the_tokens_before_it_nothing(api, dtype, D, qs, lens, G, size, factor):
    c = Case(31, qs, lens, 1, G, D, 32, 128, 128, dtype, True, True, scale_v=size)
    _grow(c, 1, lens[1] - 1, factor)                          # the last token's own row: some 1e4
    ref, mag = c.expected()
    got = c.attend(api).double().cpu()
    api.check_status()
    clean = slice(0, c.T - 1)
    # a half output's own smallest step; what tolerance() allows for small weights goes by the rows these tokens see
    tol = c.tolerance(ref[clean], mag[clean]) + (2.0 ** -25 if dtype == F16 else 0.0)
    err = (got - ref).abs()[clean]
    assert (err <= tol).all(), float((err / tol).max())
    seen = slice(c.T - 1, c.T)
    assert ((got - ref).abs()[seen] <= c.tolerance(ref[seen], mag[seen])).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q,G", [(1, 1), (3, 4), (7, 4)])
def test_small_weights_of_large_value_rows_keep_their_bits(api, D, q, G):
    """bf16 caches, few tokens: one key's weight is 2^-22 of the others' and its value row 2^26 times as large: half of the sum's terms."""
    n, at, gap = 24, 15, 22
    c = Case(33, (q,), (n,), 1, G, D, 32, 128, 128, BF16, True, False, far=False, scale_v=2.0 ** -17)
    c.q1[:] = 0
    c.q1[:, :, 0] = 4
    page, row = c.table[0, at // c.P], at % c.P
    c.pools[0].zero_()                                        # scores of 0, but for this key's: -gap in units of log 2
    c.scales[0].fill_(1.0)
    c.dense[0][0].zero_()
    step = torch.tensor(gap * math.log(2.0) * D ** 0.5 / 4 / 127, dtype=torch.float32)
    c.pools[0][page, :, row, 0], c.scales[0][page, :, row] = -127, step
    c.dense[0][0][at, :, 0] = -127 * step.double()
    _grow(c, 0, at, 2.0 ** 26)
    ref, mag = c.expected()
    got = c.attend(api)[:c.T].double().cpu()
    api.check_status()
    tol = c.tolerance(ref, mag)
    assert ((got - ref).abs() <= tol).all(), float(((got - ref).abs() / tol).max())
