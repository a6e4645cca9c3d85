"""projected_logprobs where rows and weights lie in memory in different ways: one of them read as it is, the other laid out anew."""
import math

import pytest
import torch

from test_gpu_projected import case, check
from test_gpu_readout import DTYPES

pytestmark = pytest.mark.gpu


def among(t, before, after, filler):
    """The same numbers as rows of a wider tensor that holds something else beside them."""
    wide = torch.full((t.shape[0], before + t.shape[1] + after), filler, dtype=t.dtype, device="cuda")[:, before:before + t.shape[1]]
    wide.copy_(t)
    return wide


# beginning at whole 16 bytes, rows of whole 16 bytes; beginning anywhere; rows that begin anywhere
PLACES = {"whole": (8, 16), "odd": (1, 7), "ragged": (0, 3)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", [(150, 500, 72), (150, 500, 1000), (150, 500, 1001), (70, 300, 8), (300, 100, 520), (20, 700, 88)])
@pytest.mark.parametrize("x_at", list(PLACES))
@pytest.mark.parametrize("w_at", list(PLACES))
def test_rows_and_weights_each_in_its_own_place(rows, vocab, dim, dtype, x_at, w_at):
    c = case(rows, vocab, dim, dtype)
    for filler in (math.nan, math.inf):
        check(dict(c, x=among(c["x"], *PLACES[x_at], filler), weight=among(c["weight"], *PLACES[w_at], filler)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("which", ["x", "weight"])
def test_one_operand_with_rows_far_apart(dtype, which):
    """2^21 numbers from row to row, which are laid out anew; the other operand, beside NaN, is not."""
    c = case(100, 200, 72, dtype)
    far = torch.empty(c[which].shape[0], 1 << 21, dtype=dtype, device="cuda")[:, :72]
    far.copy_(c[which])
    other = "weight" if which == "x" else "x"
    check(dict(c, **{which: far, other: among(c[other], 8, 16, math.nan)}))
