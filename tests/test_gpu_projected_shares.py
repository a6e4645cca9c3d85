"""projected_logprobs_bwd of rows that are not finite and have no gradient."""
import math

import pytest
import torch

from bmtk_amd import readout
from test_gpu_projected import case, run
from test_gpu_projected_edges import FEW_AND_MANY
from test_gpu_readout import DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", FEW_AND_MANY)
def test_a_row_that_is_not_finite_and_has_no_d_logp(rows, vocab, dim, dtype):
    """Its gradient, 0 times NaN, is NaN, and all of d_weight, of any number of rows and words; without a token it has no part."""
    c = case(rows, vocab, dim, dtype, ignored=0.0)
    want = run(c)
    for value in (math.nan, math.inf):
        x, d_logp = c["x"].clone(), c["d_logp"].clone()
        x[2, 0], d_logp[2] = value, 0.0
        got = run(dict(c, x=x, d_logp=d_logp))
        assert got["dx"][2].isnan().all() and got["d_weight"].isnan().all()
        others = torch.arange(rows, device="cuda") != 2
        assert torch.equal(got["dx"][others], want["dx"][others])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,dim", FEW_AND_MANY)
def test_a_row_of_nothing_but_minus_infinity_has_no_part(rows, vocab, dim, dtype):
    c = case(rows, vocab, dim, dtype, ignored=0.0)
    c["weight"][:, 0] = c["weight"][:, 0].abs() + 0.125
    c["d_logp"][2] = 0.25
    c["d_logp"][3] = 8.0   # (the largest, with and without row 2)
    tokens = c["tokens"].clone()
    tokens[2] = -100
    want = run(dict(c, tokens=tokens))
    x = c["x"].clone()
    x[2], x[2, 0] = 0.0, -math.inf
    r = readout.projected_logprobs(x, c["weight"], c["tokens"])
    got = run(dict(c, x=x))
    if dtype == torch.float32 and rows > 64 and vocab > 128:   # (parts of the weights have either sign)
        assert r.lse[2].isnan() and r.logp[2].isnan() and got["dx"][2].isnan().all() and got["d_weight"].isnan().all()
    else:
        assert r.lse[2] == -math.inf and r.logp[2] == -math.inf
        assert not got["dx"][2].any() and torch.equal(got["d_weight"], want["d_weight"])
