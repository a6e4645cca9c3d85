"""projected_logprobs where it can go wrong: rows without a token that hold anything, tokens outside the vocabulary, logits far from zero, views, single numbers, and gradients by
differences."""
import math

import pytest
import torch

from bmtk_amd import readout
from test_gpu_projected import case, check, reference, run
from test_gpu_readout import DTYPES, U, close, gen

pytestmark = pytest.mark.gpu

# few rows of every class, and tiles; vocabularies of one, four and eight wavefronts a tile of few rows; small vocabularies, rows of one, four and eight wavefronts
FEW_AND_MANY = [(7, 1000, 96), (20, 40000, 40), (50, 66000, 24), (130, 700, 72), (300, 129, 200), (90, 7, 300), (9, 8, 1100), (2100, 100, 271), (66000, 40, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", FEW_AND_MANY)
def test_rows_without_a_token_hold_anything(rows, vocab, dim, dtype):
    c = case(rows, vocab, dim, dtype, ignored=0.4)
    ignored = c["tokens"] == -100
    want = run(c)
    for filler in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max):
        x, d_logp = c["x"].clone(), c["d_logp"].clone()
        x[ignored] = filler
        d_logp[ignored] = filler
        got = run(dict(c, x=x, d_logp=d_logp))
        assert torch.equal(got["d_weight"], want["d_weight"]) and torch.equal(got["dx"], want["dx"]) and torch.equal(got["logp"], want["logp"])
        assert torch.equal(got["lse"][~ignored], want["lse"][~ignored])
        assert not got["dx"][ignored].any() and not got["logp"][ignored].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", FEW_AND_MANY)
def test_no_row_has_a_token(rows, vocab, dim, dtype):
    c = case(rows, vocab, dim, dtype)
    got = run(dict(c, tokens=torch.full_like(c["tokens"], -100)))
    assert not got["logp"].any() and not got["dx"].any() and not got["d_weight"].any()
    close(got["lse"], *reference(c)["lse"], "lse")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", FEW_AND_MANY)
def test_rows_that_are_not_finite_leave_the_others_as_they_are(rows, vocab, dim, dtype):
    """Also tokens outside the vocabulary."""
    c = case(rows, vocab, dim, dtype, ignored=0.0)
    want = run(c)
    x, tokens = c["x"].clone(), c["tokens"].clone()
    x[1, 3], x[2, 0], x[3] = math.nan, math.inf, -math.inf
    tokens[4], tokens[5] = vocab, -1
    got = run(dict(c, x=x, tokens=tokens))
    assert got["logp"][1:6].isnan().all() and got["lse"][1:4].isnan().all() and torch.equal(got["lse"][4:6], want["lse"][4:6])
    assert got["dx"][1:6].isnan().all() and got["d_weight"].isnan().all()
    others = torch.ones(rows, dtype=torch.bool)
    others[1:6] = False
    for name in ("logp", "lse", "dx"):
        assert torch.equal(got[name][others], want[name][others]), name


@pytest.mark.parametrize("dtype,scale", [(torch.float32, 1e4), (torch.bfloat16, 1e4), (torch.float16, 2e2), (torch.float32, 0.0), (torch.bfloat16, 1e-3)])
@pytest.mark.parametrize("rows,vocab,dim", [(9, 3000, 40), (200, 3000, 40)])
def test_logits_far_from_zero_and_all_alike(rows, vocab, dim, dtype, scale):
    check(case(rows, vocab, dim, dtype, scale=scale))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", [(40, 2, 9), (40, 16, 70), (33, 17, 1030), (300, 128, 1100), (100, 32, 264), (9000, 100, 270), (8200, 65, 64), (8191, 64, 1025), (130, 128, 33),
                                            (65, 128, 2050)])
def test_small_vocabularies(rows, vocab, dim, dtype):
    check(case(rows, vocab, dim, dtype))


@pytest.mark.parametrize("vocab", [33, 130])
def test_very_many_rows(vocab):
    """One row's d_logp is far larger than all others', and the last one's."""
    c = case(65600, vocab, 300, torch.bfloat16)
    check(c)
    c["tokens"][65599] = 1
    c["d_logp"][65599] = 1e6
    check(c)


@pytest.mark.parametrize("rows,vocab,dim", [(1, 1, 1), (1, 1, 64), (70, 1, 5), (1, 300, 1), (65, 2, 3), (400, 3, 1)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_single_numbers(rows, vocab, dim, dtype):
    check(case(rows, vocab, dim, dtype, ignored=0.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(5, 64), (24, 72), (60, 33), (150, 64), (150, 61)])
def test_views_of_anything(rows, dim, dtype):
    """Rows further apart than their channels, beginning anywhere, beside NaN; one row for all (no distance), one vector of weights for all."""
    c = case(rows, 500, dim, dtype)
    for before, width in ((0, dim + 8), (8, dim + 24), (1, dim + 3)):
        wide_x, wide_w = (torch.full((n, width + before), math.nan, dtype=dtype, device="cuda")[:, before:before + dim] for n in (rows, 500))
        wide_x.copy_(c["x"])
        wide_w.copy_(c["weight"])
        check(dict(c, x=wide_x, weight=wide_w))
    check(dict(c, x=c["x"][:1].expand(rows, dim)))
    check(dict(c, weight=c["weight"][:1].expand(500, dim)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [5, 150])
def test_rows_far_apart(rows, dtype):
    """The last step of each of some sequences: rows 2^22 numbers apart."""
    c = case(rows, 300, 64, dtype)
    far = torch.empty(rows, 1 << 22, dtype=dtype, device="cuda")[:, -64:]
    far.copy_(c["x"])
    check(dict(c, x=far))


@pytest.mark.parametrize("rows", [3, 70])
def test_weights_of_more_than_32_bits_of_offsets(rows):
    """The last rows of 2.5 billion weights, the others 0: sums over the vocabulary known in closed form."""
    vocab, dim, used = 1_200_003, 2080, 5
    g = gen(rows)
    weight = torch.zeros(vocab, dim, dtype=torch.bfloat16, device="cuda")
    last = (2.0 / math.sqrt(dim) * torch.randn(used, dim, generator=g)).bfloat16().cuda()
    weight[-used:] = last
    x = torch.randn(rows, dim, generator=g).bfloat16().cuda()
    tokens = vocab - 1 - torch.arange(rows, device="cuda") % used
    r = readout.projected_logprobs(x, weight, tokens)
    logits = x.double() @ last.double().t()
    mag = x.double().abs() @ last.double().abs().t()
    lse = torch.log(torch.exp(logits).sum(1) + (vocab - used))
    at = (tokens - (vocab - used)).unsqueeze(1)
    # as in the other checks: dim + 8 roundings of a logit's terms; a sum of positive terms in additions of 256 and vocab / 256 tiles
    e_l = (dim + 8) * U * mag
    e_lse = e_l.amax(1) + (2 * 40 + 8 + 256 + vocab / 256) * U + 4 * U * lse.abs()
    want = logits.gather(1, at).squeeze(1) - lse
    close(r.lse, lse, e_lse, "lse")
    close(r.logp, want, e_lse + e_l.gather(1, at).squeeze(1) + 4 * U * logits.gather(1, at).squeeze(1).abs(), "logp")
    dx, dw = readout.projected_logprobs_bwd(x, weight, tokens, r, torch.ones(rows, device="cuda"))
    p = torch.exp(logits - lse.unsqueeze(1))
    d = torch.zeros_like(p).scatter(1, at, 1.0) - p
    # d_logp of 1 for all: p - delta is rounded to 16 bits once, and the result once (close's own)
    e_d = 2.0 ** -8 * d.abs() + p * (e_l + e_lse.unsqueeze(1)) * 2
    close(dx, d @ last.double(), e_d @ last.double().abs() + (vocab + 16) * U * (d.abs() @ last.double().abs()), "dx")
    close(dw[-used:], d.t().contiguous() @ x.double(), (e_d + (rows + 16) * U * d.abs()).t().contiguous() @ x.double().abs(), "d_weight")
    rest = torch.exp(-lse)
    # (all other rows have the same gradient: minus the sum of x e^-lse)
    close(dw[0], -(rest @ x.double()), (2.0 ** -8 + 2 * e_lse.max() + (rows + 16) * U) * (rest @ x.double().abs()), "d_weight of weights of 0")
    assert all(torch.equal(dw[k], dw[0]) for k in (1, 127, 70_000, vocab // 2, vocab - used - 1))


def test_shapes_of_more_and_fewer_dimensions():
    c = case(24, 50, 16, torch.bfloat16)
    want = run(c)
    shape = lambda t: t.view(2, 3, 4, *t.shape[1:])  # noqa: E731
    got = run(dict(c, x=shape(c["x"]), tokens=shape(c["tokens"]), d_logp=shape(c["d_logp"])))
    for name in ("logp", "lse", "dx"):
        assert torch.equal(got[name], shape(want[name])), name
    assert torch.equal(got["d_weight"], want["d_weight"])
    turned = c["tokens"].view(4, 6).t()
    got = run(dict(c, x=c["x"].view(4, 6, 16).transpose(0, 1), tokens=turned, d_logp=c["d_logp"].view(4, 6).t().contiguous()))
    assert torch.equal(got["logp"], want["logp"].view(4, 6).t()) and torch.equal(got["dx"], want["dx"].view(4, 6, 16).transpose(0, 1))
    row = readout.projected_logprobs(c["x"][3], c["weight"], c["tokens"][3])
    assert row.logp.shape == () and torch.equal(row.logp, readout.projected_logprobs(c["x"][3:4], c["weight"], c["tokens"][3:4]).logp[0])
    r = readout.projected_logprobs(c["x"][:0], c["weight"], c["tokens"][:0])
    assert all(v.shape == (0,) for v in r)
    dx, dw = readout.projected_logprobs_bwd(c["x"][:0], c["weight"], c["tokens"][:0], r, c["d_logp"][:0])
    assert dx.shape == (0, 16) and not dw.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", FEW_AND_MANY)
def test_the_same_bits_again(rows, vocab, dim, dtype):
    c = case(rows, vocab, dim, dtype)
    first = run(c)
    for _ in range(3):
        assert all(torch.equal(first[k], v) for k, v in run(c).items())


@pytest.mark.parametrize("rows", [12, 90])
def test_by_differences(rows):
    """The gradient against differences of the definition's own sum in 64 bits, along random directions."""
    c = case(rows, 70, 24, torch.float32, seed=3)
    got = run(c)
    x, w = c["x"].double(), c["weight"].double()
    given, at = c["tokens"] != -100, c["tokens"].clamp(min=0).unsqueeze(1)

    def loss(x, w):
        logp = torch.log_softmax(x @ w.t().contiguous(), 1).gather(1, at).squeeze(1)
        return (torch.where(given, logp, 0.0) * c["d_logp"].double()).sum()
    step = 1e-5
    for name, which in (("dx", 0), ("d_weight", 1)):
        v = torch.randn(got[name].shape, generator=gen(9), dtype=torch.float64).cuda()
        there, back = ((x + s * v, w) if which == 0 else (x, w + s * v) for s in (step, -step))
        terms = got[name].double() * v
        # differences of second order: 1e-10 times a third derivative, and 1e-16 / 1e-5 of the loss; fp32 gradients: six products of 70 + 16 terms each, of magnitudes whose sum is
        # some ten times the result's
        assert (terms.sum() - (loss(*there) - loss(*back)) / (2 * step)).abs() <= 6 * 86 * 10 * U * terms.abs().sum() + 1e-6 * (1 + terms.abs().sum()), name
