"""projected_logprobs_bwd of so many logits that they are made in pieces of the vocabulary, of which the last is far smaller than the others."""
import pytest
import torch

from test_gpu_projected import case, reference, run
from test_gpu_readout import close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,dim,dtype", [(32768, 253953, 40, torch.bfloat16), (32768, 253953, 40, torch.float16), (9216, 340993, 24, torch.float32), (9216, 340994 + 60, 24, torch.float32)])
def test_a_last_piece_of_a_few_words(rows, vocab, dim, dtype):
    """Fewer steps of k than the sums are cut into.  Some rows have a token, most of them in the last piece, and only those are compared: all others have no gradient and no part."""
    c = case(rows, vocab, dim, dtype, ignored=1.0)
    some = torch.arange(48, device="cuda") * (rows // 48) + 5
    tokens = torch.full((rows,), -100, device="cuda")
    tokens[some] = torch.where(torch.arange(48, device="cuda") % 4 == 0, torch.arange(48, device="cuda") * 1000, vocab - 1)
    got = run(dict(c, tokens=tokens))
    want = reference(dict(c, x=c["x"][some], tokens=tokens[some], d_logp=c["d_logp"][some]))
    for name in ("lse", "logp", "dx"):
        close(got[name][some], *want[name], name)
    # (sums of all rows, of which 48 are not 0)
    close(got["d_weight"], *want["d_weight"], "d_weight")
    others = torch.ones(rows, dtype=torch.bool, device="cuda")
    others[some] = False
    assert not got["dx"][others].any() and not got["logp"][others].any()
