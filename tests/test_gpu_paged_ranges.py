"""8-bit pages whose rows differ in size by many powers of two: every token's result keeps the bits of the rows that it sees."""
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
