"""projected_logprobs_bwd of rows whose d_logp, or whose x, are far apart in size, or that are not finite and have no gradient."""
import math

import pytest
import torch

from bmtk_amd import readout
from test_gpu_projected import case, run
from test_gpu_projected_edges import FEW_AND_MANY
from test_gpu_readout import DTYPES, U, close, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("rows,vocab,dim", [(9, 200, 64), (40, 200, 64), (300, 40, 64), (300, 120, 72), (700, 1000, 72), (40000, 20, 64), (33000, 200, 64)])
@pytest.mark.parametrize("large,size", [(1.0, 1.0), (2.0 ** 9, 2.0 ** -9), (2.0 ** -7, 1.0)])
def test_fp16_rows_of_far_smaller_gradients(rows, vocab, dim, aligned, large, size):
    """One row's d_logp is 2^14, and its label one of the two words that it takes for likely; the others' are 2^-10 to 2^-26 of that, and their labels among the other words, of whose
    gradient they have all but channel 0.  large: that row's x; size: of the other rows' x, which have less or more of d_logp by as much."""
    g = gen(rows)
    weight = torch.randn(vocab, dim, generator=g) / 8
    weight[:2], weight[:, 0] = 0.0, 0.0
    weight[:2, 0] = 28.0 / large   # (of up to 3,584: e^28, so that all other words have 2^-40 of the row's probability)
    x = torch.randn(rows, dim, generator=g) * size
    x[:, 0] = 0.0
    at = rows // 2
    x[at] = 0.0
    x[at, 0] = large
    tokens = torch.randint(2, vocab, (rows,), generator=g)
    tokens[at] = 1
    d_logp = 2.0 ** (4.0 - 16.0 * torch.rand(rows, generator=g)) / size
    d_logp[at] = 2.0 ** 14 / max(large, 1.0)
    x, weight, tokens, d_logp = x.half().cuda(), weight.half().cuda(), tokens.cuda(), d_logp.cuda()
    if not aligned:
        x, weight = (torch.cat([torch.zeros(len(t), 1, dtype=t.dtype, device="cuda"), t], 1)[:, 1:] for t in (x, weight))
    got = run(dict(x=x, weight=weight, tokens=tokens, d_logp=d_logp))["d_weight"]
    xd, wd, dd = x.double(), weight.double(), d_logp.double().unsqueeze(1)
    logits, mag = xd @ wd.t().contiguous(), xd.abs() @ wd.abs().t().contiguous()
    p = torch.softmax(logits, 1)
    gr = p.scatter_add(1, tokens.unsqueeze(1), torch.full_like(tokens.unsqueeze(1), -1.0, dtype=torch.float64))
    # p: its logit's and its sum's errors; G: half a step of 16 bits, of a smallest step of 2^-24 in units of 2^-14; x times d_logp: half a step of 24 bits for each of three roundings, and half of
    # the smallest step where the largest product of the call is 2^14 or more of them, twice that for d_logp's mantissa
    e_p = p * torch.expm1(2 * (dim + 8) * U * mag.amax(1, keepdim=True) + (vocab + 80) * U) + 8 * U * p
    e_g = e_p + 2.0 ** -11 * (gr.abs() + e_p) + 2.0 ** -39
    xw = (xd * dd).abs()
    e_xw = 3 * U * xw + 2.0 ** -38 * xw.max()
    gm = gr.abs() + e_g
    error = e_g.t().contiguous() @ (xw + e_xw) + gm.t().contiguous() @ e_xw + (rows + 16) * U * (gm.t().contiguous() @ xw)
    close(got, -(gr.t().contiguous() @ (xd * dd)), error, "d_weight")


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


@pytest.mark.parametrize("rows,vocab,dim", [(300, 40, 64), (200, 500, 72)])
def test_fp16_captured_and_replayed_on_rows_of_other_sizes(rows, vocab, dim):
    """Two graphs, replayed in turn, whose rows and d_logp are larger or smaller each time; eager work and synchronizations in between."""
    cases = [case(rows, vocab, dim, torch.float16, seed=s) for s in range(3)]
    for k, c in enumerate(cases):
        c["x"], c["weight"] = c["x"] * (1.0, 2.0 ** 6, 2.0 ** -9)[k], c["weight"] / (1.0, 2.0 ** 6, 2.0 ** -5)[k]
        c["d_logp"] = c["d_logp"] * 2.0 ** -(20.0 * torch.rand(rows, generator=gen(k))).cuda() / (1.0, 2.0 ** 6, 2.0 ** -9)[k]
    want = [run(c) for c in cases]
    graphs = []
    for k in (0, 1):
        held = {name: t.clone() for name, t in cases[k].items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(held)
        graphs.append((graph, held, out))
    for turn in range(5):
        for k, (graph, held, _) in enumerate(graphs):
            for name, t in cases[(turn + k) % 3].items():
                held[name].copy_(t)
            graph.replay()
        run(cases[2])
        torch.cuda.synchronize()
        for k, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(out[name], t) for name, t in want[(turn + k) % 3].items()), (turn, k)
