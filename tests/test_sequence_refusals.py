"""What short_conv, selective_scan and projected_logprobs refuse, before any launch: by the C ABI's checks and by the Python functions' own."""
import os
import re

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from bmtk_amd import _lib, readout, training
from test_readout_refusals import P, ROOT, refused


def test_constants_are_the_headers():
    txt = open(os.path.join(ROOT, "include", "bmtk_amd.h")).read()
    value = lambda name: int(re.search(r"#define {} (\d+)".format(name), txt).group(1))  # noqa: E731
    assert value("BMTK_CONV_MAX_WIDTH") == _lib.CONV_MAX_WIDTH and value("BMTK_SELECTIVE_MAX_STATES") == _lib.SELECTIVE_MAX_STATES


def conv(backward, steps=5, batch=2, dim=8, width=4, dtype=0, weights=0, x=P, weight=P, y=P, last=P, dy=P, ws=P):
    sizes = steps, batch, dim, width, dtype, weights, 1, x, batch * dim, dim, weight, None, None, None
    if backward:
        return _lib.load().bmtk_short_conv_bwd(*sizes, dy, batch * dim, dim, None, y, last, None, None, ws, None)
    return _lib.load().bmtk_short_conv_fwd(*sizes, y, last, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("change,word", [
    (dict(x=None), "null"), (dict(weight=None), "null"), (dict(y=None), "null"), (dict(last=None), "null"), (dict(steps=0), "positive"), (dict(batch=0), "positive"),
    (dict(dim=-1), "positive"), (dict(width=1), "width"), (dict(width=9), "width"), (dict(dtype=3), "type"), (dict(dtype=1, weights=2), "weights"), (dict(dtype=0, weights=1), "weights"),
    (dict(steps=(1 << 31) - 4096), "too many"), (dict(batch=1 << 31, dim=1), "too many"), (dict(batch=1 << 16, dim=1 << 15), "too many")])
def test_short_conv(backward, change, word):
    refused(conv(backward, **change), "short_conv_" + ("bwd" if backward else "fwd"), word)


def test_short_conv_bwd():
    refused(conv(True, dy=None), "null")
    refused(conv(True, ws=None), "workspace")
    refused(conv(True, steps=1, batch=1, dim=1 << 27, width=2), "too many weights")
    size = _lib.load().bmtk_short_conv_workspace_bytes
    assert size(5, 2, 8, 4, 0) >= 2 * 8 * 5 * 4
    for wrong in ((0, 2, 8, 4, 0), (5, 0, 8, 4, 0), (5, 2, 0, 4, 0), (5, 2, 8, 1, 0), (5, 2, 8, 9, 0), (5, 2, 8, 4, 3), (5, 1 << 31, 8, 4, 0), (1 << 31, 2, 8, 4, 0)):
        assert size(*wrong) == 0


def selective(backward, steps=20, batch=2, dim=8, groups=1, states=4, dtype=0, gates=0, x=P, dt=P, write=P, read=P, rate=P, y=P, last=P, marks=P, dy=P, ws=P):
    row, shared = (batch * dim, dim), (batch * groups * states, groups * states)
    sizes = (steps, batch, dim, groups, states, dtype, gates, 1, x, *row, dt, *row, write, *shared, read, *shared, rate, None, None)
    if backward:
        return _lib.load().bmtk_selective_scan_bwd(*sizes, marks, None, dy, *row, None, y, last, P, P, P, None, None, None, ws, None)
    return _lib.load().bmtk_selective_scan_fwd(*sizes, None, None, y, last, None, ws, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("change,word", [
    (dict(x=None), "null"), (dict(dt=None), "null"), (dict(write=None), "null"), (dict(read=None), "null"), (dict(rate=None), "null"), (dict(y=None), "null"), (dict(last=None), "null"),
    (dict(steps=0), "positive"), (dict(batch=-1), "positive"), (dict(dim=0), "positive"), (dict(groups=0), "positive"), (dict(states=0), "positive"), (dict(groups=3), "evenly"),
    (dict(states=65), "64"), (dict(dtype=-1), "type"), (dict(dtype=1, gates=2), "dt"), (dict(dtype=0, gates=1), "dt"), (dict(ws=None), "workspace"),
    (dict(steps=(1 << 31) - 4096), "too many"), (dict(batch=1 << 16, dim=1 << 15), "too many"),
    # products of sizes that pass 64 bits
    (dict(steps=(1 << 31) - 8192, batch=(1 << 31) - 1, dim=1, states=64), "too many"),
    # a launch's threads: states of a step, states of a channel, lanes without a channel
    (dict(steps=1 << 20, batch=1 << 8, dim=4, states=16), "too many"), (dict(steps=20, batch=1 << 13, dim=1 << 13, states=64), "too many"),
    (dict(steps=20, batch=1 << 25, dim=4, groups=4, states=4), "too many"), (dict(steps=20, batch=1, dim=1 << 26, states=4), "too many")])
def test_selective_scan(backward, change, word):
    refused(selective(backward, **change), "selective_scan_" + ("bwd" if backward else "fwd"), word)


def test_selective_scan_bwd():
    refused(selective(True, marks=None), "null")
    refused(selective(True, dy=None), "null")
    size = _lib.load().bmtk_selective_scan_workspace_bytes
    assert size(20, 2, 8, 1, 4, 1) > size(20, 2, 8, 1, 4, 0) > 0 == size(8, 2, 8, 1, 4, 0) < size(8, 2, 8, 1, 4, 1)   # (up to eight steps need none)
    for wrong in ((0, 2, 8, 1, 4), (20, 0, 8, 1, 4), (20, 2, 8, 3, 4), (20, 2, 8, 1, 65), ((1 << 31) - 8192, (1 << 31) - 1, 1, 1, 64)):
        assert size(*wrong, 0) == size(*wrong, 1) == 0


def projected(backward, rows=100, vocab=500, dim=8, dtype=0, x=P, x_stride=8, weight=P, w_stride=8, tokens=P, logp=P, lse=P, peak=P, total=P, ws=P):
    given = rows, vocab, dim, dtype, x, x_stride, weight, w_stride, tokens, -100
    if backward:
        return _lib.load().bmtk_projected_logprobs_bwd(*given, peak, total, P, logp, lse, ws, None)
    return _lib.load().bmtk_projected_logprobs_fwd(*given, logp, lse, peak, total, ws, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("change,word", [
    (dict(x=None), "null"), (dict(weight=None), "null"), (dict(tokens=None), "null"), (dict(logp=None), "null"), (dict(lse=None), "null"), (dict(peak=None), "null"), (dict(total=None), "null"),
    (dict(rows=0), "positive"), (dict(vocab=0), "positive"), (dict(dim=-8), "positive"), (dict(dtype=3), "type"), (dict(rows=1 << 22), "2^22"), (dict(vocab=1 << 28), "2^28"),
    (dict(dim=65537), "65,536"), (dict(x_stride=-8), "negative"), (dict(w_stride=-8), "negative"), (dict(ws=None), "workspace"),
    (dict(vocab=1 << 20, dim=1 << 15), "too many numbers"), (dict(rows=1 << 20, dim=1 << 14), "too many numbers"), (dict(rows=(1 << 22) - 1, vocab=(1 << 28) - 1), "too many logits")])
def test_projected_logprobs(backward, change, word):
    refused(projected(backward, **change), "projected_logprobs_" + ("bwd" if backward else "fwd"), word)


def test_projected_logprobs_workspace():
    size = lambda *sizes: [_lib.load().bmtk_projected_logprobs_workspace_bytes(*sizes, P, 8, P, 8, way) for way in (0, 1)]  # noqa: E731
    assert min(size(100, 500, 8, 0)) >= 100 * 4 and size(100, 50, 8, 0)[0] == 0 < size(100, 50, 8, 0)[1]   # (a small vocabulary's logits are whole in registers)
    for wrong in ((0, 50, 8, 0), (100, 0, 8, 0), (100, 50, 0, 0), (100, 50, 8, 3), (1 << 22, 50, 8, 0), (100, 1 << 28, 8, 0), (100, 50, 65537, 0)):
        assert size(*wrong) == [0, 0]


def calls(x, tokens=None):
    """Every call, x of three dimensions as the argument that is looked at first."""
    rate, shared, tokens = torch.zeros(4, 3), torch.zeros(5, 2, 1, 3), torch.zeros(5, 2, dtype=torch.int64)
    fwd = readout.ProjectedLogProbs(*[torch.zeros(5, 2)] * 4)
    return [lambda: readout.short_conv(x, torch.zeros(4, 2)), lambda: readout.short_conv_bwd(x, torch.zeros(4, 2), x), lambda: readout.selective_scan(x, x, rate, shared, shared),
            lambda: readout.selective_scan_bwd(x, x, rate, shared, shared, torch.zeros(1, 2, 4, 3), x), lambda: readout.projected_logprobs(x, torch.zeros(7, 4), tokens),
            lambda: readout.projected_logprobs_bwd(x, torch.zeros(7, 4), tokens, fwd, torch.zeros(5, 2))]


def test_tensors_on_the_host():
    for call in calls(torch.zeros(5, 2, 4)):
        with pytest.raises(ValueError, match="current device"):
            call()


def test_what_is_no_tensor():
    for call in calls([[[1.0] * 4] * 2] * 5):
        with pytest.raises(TypeError, match="tensor"):
            call()


def test_tangents():
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(5, 2, 4), torch.ones(5, 2, 4))
        for recording in (True, False):
            with torch.set_grad_enabled(recording):
                for call in calls(x):
                    with pytest.raises(ValueError, match="tangent"):
                        call()


def test_negated_views():
    for call in calls(torch.complex(torch.ones(5, 2, 4), torch.ones(5, 2, 4)).conj().imag):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()


def test_sequence_loss():
    bits, labels = torch.zeros(5, 1, dtype=torch.int64), torch.zeros(5, 2, dtype=torch.int64)
    given = lambda **change: [dict(dict(bits=bits, batch=2, weight=torch.zeros(10, 14), conv_weight=torch.zeros(10, 4), rate=torch.zeros(4, 3), out_weight=torch.zeros(7, 4),  # noqa: E731
                                        labels=labels), **change)]
    for change, error, word in ((dict(), ValueError, "current device"), (dict(weight=torch.zeros(10, 13)), ValueError, r"\[neurons, 14\]"), (dict(groups=2), ValueError, r"\[neurons, 20\]"),
                                (dict(groups=0), ValueError, "groups"), (dict(weight=[[1.0]]), ValueError, "weight"), (dict(rate=torch.zeros(4)), ValueError, "rate")):
        with pytest.raises(error, match=word):
            training.sequence_loss(**given(**change)[0])


@pytest.mark.parametrize("dim,states", [((1 << 26) - 2048, 4), (44_800_000, 1), (44_740_000, 3), ((1 << 24) - 1024, 16)])
def test_selective_scan_sums_of_too_many_channels(dim, states):
    """The launch that adds up d_rate, d_skip and d_dt_bias has sixteen threads for each number of a channel, of which there are P and two: 2^32 of them or more are refused."""
    assert 16 * dim * (-(-states // 4) * 4 + 2) >= 1 << 32 > 16 * dim * (-(-states // 4) * 4)
    for backward in (False, True):
        refused(selective(backward, batch=1, dim=dim, states=states), "selective_scan_" + ("bwd" if backward else "fwd"), "too many")
        assert _lib.load().bmtk_selective_scan_workspace_bytes(20, 1, dim, 1, states, backward) == 0
