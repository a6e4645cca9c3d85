"""projected_logprobs against plain implementations in 64 bits.

Tolerances are bounds, made from the sums themselves: U = 2^-24 is half a step of fp32, a value rounded to type T is off by at most eps(T) / 2 of itself (and
half of the smallest subnormal), and a sum of k terms is off by at most k U times the sum of the terms' magnitudes."""
import math

import pytest
import torch

from bmtk_amd import readout
from test_gpu_readout import DTYPES, U, close, gen

pytestmark = pytest.mark.gpu


def case(rows, vocab, dim, dtype, ignored=0.2, scale=2.5, seed=0):
    g = gen(seed)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    tokens = torch.where(torch.rand(rows, generator=g) < ignored, -100, tokens)
    return dict(x=torch.randn(rows, dim, generator=g).to(dtype).cuda(), weight=(scale / math.sqrt(dim) * torch.randn(vocab, dim, generator=g)).to(dtype).cuda(), tokens=tokens.cuda(),
                d_logp=(torch.randn(rows, generator=g) * (100.0 if dtype == torch.float16 else 1.0)).cuda())


def reference(c):
    """Values in 64 bits and bounds, on the device."""
    x, w, tokens, d_logp = c["x"].double(), c["weight"].double(), c["tokens"], c["d_logp"].double()
    dtype, dim, vocab = c["x"].dtype, c["x"].shape[1], c["weight"].shape[0]
    wt = w.t().contiguous()
    logits, mag = x @ wt, x.abs() @ wt.abs()
    # products and additions of a row's channels; of fp32 operands in three parts, six products each, and what is left out, below 2^-24 of a term
    e_l = (dim + 8) * U * mag * (6 if dtype == torch.float32 else 1)
    lp = torch.log_softmax(logits, 1)
    lse = torch.logsumexp(logits, 1)
    # a sum of positive terms, each off by its exponent (the logit's error and that of up to 40 away from the largest) and a few roundings, in additions of vocab / 256 tiles and 256
    e_lse = e_l.amax(1) + (2 * 40 + 8 + 256 + vocab / 256) * U + 4 * U * lse.abs()
    given = tokens != -100
    at = torch.where(given, tokens, 0).unsqueeze(1)
    e_logp = e_lse + e_l.gather(1, at).squeeze(1) + 4 * U * logits.gather(1, at).squeeze(1).abs()
    out = dict(lse=(lse, e_lse), logp=(torch.where(given, lp.gather(1, at).squeeze(1), 0.0), torch.where(given, e_logp, 0.0)))
    p = torch.exp(lp)
    g = p.scatter_add(1, at, torch.full_like(at, -1.0, dtype=torch.float64)) * given.unsqueeze(1)
    # p - delta: p's own error, then half a step of the 16 bits that it, or it times up to 2, is rounded to (fp32: of 24); of fp16, in units of 2^-14, half of the smallest step, 2^-25
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U
    e_p = (p * torch.expm1(e_l + e_lse.unsqueeze(1)) + 8 * U * p) * given.unsqueeze(1)
    e_g = e_p + half * (g.abs() + e_p) + (2.0 ** -39 if dtype == torch.float16 else 0.0)
    gm = g.abs() + e_g
    k = 6 if dtype == torch.float32 else 1
    dx = -(d_logp * given).unsqueeze(1) * (g @ w)
    e_dx = d_logp.abs().unsqueeze(1) * (e_g @ w.abs() + k * (vocab + 16) * U * (gm @ w.abs()))
    # x times d_logp, rounded as the type is (of fp16 with a power of two taken out: its subnormals, of the largest)
    xw = x * (d_logp * given).unsqueeze(1)
    e_xw = (half + 2 * U) * xw.abs() + (2.0 ** -24 * d_logp.abs().max() * 2 if dtype == torch.float16 else 0.0) * given.unsqueeze(1)
    gt = g.t().contiguous()
    e_gt, gmt = e_g.t().contiguous(), gm.t().contiguous()
    dw = -(gt @ xw)
    e_dw = e_gt @ (xw.abs() + e_xw) + gmt @ e_xw + k * (x.shape[0] + 16) * U * (gmt @ xw.abs())
    out.update(dx=(dx, e_dx * given.unsqueeze(1)), d_weight=(dw, e_dw))
    return out


def run(c):
    r = readout.projected_logprobs(c["x"], c["weight"], c["tokens"])
    dx, dw = readout.projected_logprobs_bwd(c["x"], c["weight"], c["tokens"], r, c["d_logp"])
    return dict(logp=r.logp, lse=r.lse, dx=dx, d_weight=dw)


def check(c):
    got, want = run(c), reference(c)
    for name in want:
        close(got[name], *want[name], name)
    again = run(c)
    assert all(torch.equal(got[k], again[k]) for k in got)
    return got


SIZES = [(1, 1, 1), (1, 2, 8), (3, 300, 64), (16, 129, 100), (17, 1000, 72), (33, 31, 5), (64, 513, 130), (65, 257, 64), (70, 1000, 128), (200, 37, 16), (257, 259, 200), (300, 2000, 777),
         (129, 5000, 33), (1000, 10, 64), (1025, 1027, 96)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", SIZES)
def test_against_64_bits(rows, vocab, dim, dtype):
    check(case(rows, vocab, dim, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", [(4096, 12000, 256), (3000, 20011, 264), (5000, 300, 1000), (80, 70001, 72)])
def test_large_tiles(rows, vocab, dim, dtype):
    check(case(rows, vocab, dim, dtype, seed=3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_several_pieces_of_the_vocabulary(dtype):
    """G of all of it would be over 512 MB."""
    rows, vocab = (6000, 50001) if dtype == torch.bfloat16 else (2500, 40001)
    check(case(rows, vocab, 40, dtype, seed=4))
