"""short_conv and selective_scan where they can go wrong: few steps of every number of states, step sizes far from zero, more than 32 bits of offsets, lengths outside the steps, and
the same bits again."""
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from bmtk_amd import readout, training
from test_gpu_readout import DTYPES, close, gen
from test_gpu_sequence import conv_case, conv_run, selective_case, selective_check, selective_reference, selective_run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps,batch,dim,states,groups", [(1, 2, 12, 64, 3), (8, 3, 5, 33, 1), (9, 3, 5, 33, 1), (4, 2, 66, 7, 2), (7, 1, 130, 2, 1), (6, 5, 3, 16, 3), (1, 1, 1, 64, 1), (8, 2, 9, 5, 1)])
def test_few_steps(steps, batch, dim, states, groups, dtype):
    selective_check(selective_case(steps, batch, dim, states, groups, dtype, ragged=True, seed=4))


@pytest.mark.parametrize("steps", [3, 20, 700])
def test_step_sizes_far_from_zero(steps):
    """Softplus from where it is nothing to where it is its argument; decays from 1 to nothing."""
    c = selective_case(steps, 2, 21, 4, 1, torch.float32, seed=6)
    far = torch.tensor([-200.0, -80.0, -30.0, -17.0, -8.0, -1e-3, 0.0, 1e-3, 5.0, 17.0, 30.0, 88.0, 200.0])
    at = torch.randint(0, len(far), c["dt"].shape, generator=gen(3))
    c["dt"], c["dt_bias"] = far[at], None
    c["x"] = c["x"] / (1.0 + far[at].clamp(min=0))
    # (an exponential below 2^-126 is 0, or that: off by at most 2^-126 of what it multiplies, states and gradients of up to 2^10 here)
    got, want = selective_run(c), selective_reference(c)
    for name in want:
        close(got[name], want[name][0], torch.as_tensor(want[name][1]) + 2.0 ** -116, name)


@pytest.mark.parametrize("steps", [5, 40])
def test_lengths_outside_the_steps_count_as_the_nearer(steps):
    s = selective_case(steps, 4, 30, 8, 1, torch.bfloat16)
    v = conv_case(steps, 4, 30, 4, torch.bfloat16)
    near, far = (torch.tensor(n, dtype=torch.int32) for n in ([0, steps, steps, 2], [-7, steps + 1, 2 ** 31 - 1, 2]))
    for run, c in ((selective_run, s), (conv_run, v)):
        a, b = run(dict(c, lengths=near)), run(dict(c, lengths=far))
        assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("dtype", DTYPES)
def test_all_sequences_empty(dtype):
    nothing = torch.zeros(3, dtype=torch.int32)
    c = dict(conv_case(20, 3, 16, 4, dtype), lengths=nothing)
    got = conv_run(c)
    assert not any(got[k].any() for k in ("y", "dx", "d_weight", "d_bias")) and torch.equal(got["last"].cpu(), c["state"]) and torch.equal(got["d_state"].cpu(), c["d_last"])
    for steps in (5, 20, 300):
        c = dict(selective_case(steps, 3, 16, 4, 1, dtype), lengths=nothing)
        got = selective_run(c)
        assert not any(got[k].any() for k in ("y", "dx", "d_dt", "d_rate", "d_write", "d_read", "d_skip", "d_dt_bias"))
        assert torch.equal(got["last"].cpu(), c["state"]) and torch.equal(got["d_state"].cpu(), c["d_last"])


def test_more_than_32_bits_of_offsets():
    """2.7 billion numbers, 0 but for the last steps: those are what a call of the last steps gives."""
    steps, batch, dim, tail = 40_000, 32, 2080, 48
    g = gen(2)
    x = torch.zeros(steps, batch, dim, dtype=torch.bfloat16, device="cuda")
    dt = torch.full((1, 1, dim), -2.0, dtype=torch.bfloat16, device="cuda").expand(steps, batch, dim)
    x[-tail:] = torch.randn(tail, batch, dim, generator=g).bfloat16().cuda()
    weight, rate = torch.randn(dim, 4, generator=g).cuda(), -torch.rand(dim, 2, generator=g).cuda()
    y, last = readout.short_conv(x, weight, silu=True)
    want, want_last = readout.short_conv(x[-tail:], weight, silu=True)
    assert torch.equal(y[-tail:], want) and torch.equal(last, want_last) and not y[:1000].any()
    dx, dw, db, ds = readout.short_conv_bwd(x, weight, x, silu=True)
    want = readout.short_conv_bwd(x[-tail:], weight, x[-tail:], silu=True)
    assert torch.equal(dx[-tail:], want[0]) and not dx[:1000].any()
    # (sums in another order: 2^-24 of the magnitudes for each of at most 64 + 16 + 640 * 32 / 16 additions)
    bound = 1360 * 2.0 ** -24 * 1.1 * (x[-tail:].float().abs().sum((0, 1)) * x[-tail:].float().abs().max()).unsqueeze(1)
    assert ((dw - want[1]).abs() <= 2 * bound).all()
    del dx, y
    torch.cuda.empty_cache()
    shared = torch.randn(1, 1, 1, 2, generator=g).bfloat16().cuda().expand(steps, batch, 1, 2)
    y, last, saved = readout.selective_scan(x, dt, rate, shared, shared, softplus=True, save_state=True)
    want, want_last = readout.selective_scan(x[-tail:], dt[-tail:], rate, shared[-tail:], shared[-tail:], softplus=True)
    scale = want.float().abs().max()
    # (the same steps, cut into other stretches: 2^-8 of a rounding, and fp32 sums)
    assert (y[-tail:].float() - want.float()).abs().max() <= 2.0 ** -8 * scale * 1.01 and (last - want_last).abs().max() <= 1e-5 * want_last.abs().max() and not y[:1000].any()
    d = readout.selective_scan_bwd(x, dt, rate, shared, shared, saved, x, softplus=True)
    some = readout.selective_scan(x[-tail:], dt[-tail:], rate, shared[-tail:], shared[-tail:], softplus=True, save_state=True)
    want = readout.selective_scan_bwd(x[-tail:], dt[-tail:], rate, shared[-tail:], shared[-tail:], some[2], x[-tail:], softplus=True)
    for name in ("dx", "d_dt", "d_write", "d_read"):
        p, q = getattr(d, name)[-tail:].float(), getattr(want, name).float()
        assert (p - q).abs().max() <= 2.0 ** -8 * q.abs().max() * 1.01, name
    for name in ("d_rate", "d_skip", "d_dt_bias"):
        p, q = getattr(d, name), getattr(want, name)
        assert (p - q).abs().max() <= 1e-4 * q.abs().max(), name
    assert not d.dx[:1000, :, :].any() or d.dx[:1000].abs().max() < want.dx.abs().max()


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_bits_again(dtype):
    c, v = selective_case(900, 3, 100, 16, 2, dtype, ragged=True), conv_case(900, 3, 100, 4, dtype, ragged=True)
    for run, case in ((selective_run, c), (conv_run, v)):
        first = run(case)
        for _ in range(3):
            assert all(torch.equal(first[k], q) for k, q in run(case).items())


def calls():
    """Every call with its tensors by name, float32 on the device."""
    ones = lambda *shape: torch.full(shape, 0.5, device="cuda")  # noqa: E731
    conv = dict(x=ones(5, 2, 4), weight=ones(4, 3), bias=ones(4), state=ones(2, 2, 4))
    scan = dict(x=ones(5, 2, 4), dt=ones(5, 2, 4), rate=-ones(4, 3), write=ones(5, 2, 1, 3), read=ones(5, 2, 1, 3), skip=ones(4), dt_bias=ones(4))
    rows, tokens = dict(x=ones(5, 4), weight=ones(7, 4)), torch.zeros(5, dtype=torch.int64, device="cuda")
    loss = dict(weight=ones(10, 14), conv_weight=ones(10, 4), rate=-ones(4, 3), out_weight=ones(7, 4), conv_bias=ones(10), skip=ones(4), dt_bias=ones(4))
    bits, labels = torch.zeros(5, 1, dtype=torch.int64, device="cuda"), torch.zeros(5, 2, dtype=torch.int64, device="cuda")
    back = lambda x, weight, peak, total, d_logp: readout.projected_logprobs_bwd(  # noqa: E731
        x, weight, tokens, readout.ProjectedLogProbs(None, None, peak, total), d_logp)
    return [(readout.short_conv, conv), (readout.short_conv_bwd, dict(conv, dy=ones(5, 2, 4), d_last=ones(2, 2, 4))), (readout.selective_scan, dict(scan, state=ones(2, 4, 3))),
            (readout.selective_scan_bwd, dict(scan, saved=ones(1, 2, 4, 3), dy=ones(5, 2, 4), d_last=ones(2, 4, 3))),
            (lambda **k: readout.projected_logprobs(tokens=tokens, **k), rows), (back, dict(rows, peak=ones(5), total=ones(5), d_logp=ones(5))),
            (lambda **k: training.sequence_loss(bits, 2, labels=labels, **k), loss)]


def test_tensors_that_are_not_what_they_look_like():
    """Each argument of each call in turn: with a tangent, recorded by autograd, or a view of numbers with the other sign."""
    for call, given in calls():
        call(**given)
        for name, t in given.items():
            with forward_ad.dual_level():
                for recording in (True, False):
                    with torch.set_grad_enabled(recording), pytest.raises(ValueError, match="tangent"):
                        call(**dict(given, **{name: forward_ad.make_dual(t, torch.ones_like(t))}))
            with pytest.raises(ValueError, match="requires gradients"):
                call(**dict(given, **{name: t.clone().requires_grad_()}))
            with torch.no_grad():
                call(**dict(given, **{name: t.clone().requires_grad_()}))
            negated = torch.complex(t, -t).conj().imag
            if negated.is_neg():
                with pytest.raises(ValueError, match="resolve_neg|next to one another|contiguous"):
                    call(**dict(given, **{name: negated}))
        for name, t in given.items():
            with pytest.raises(ValueError, match="current device"):
                call(**dict(given, **{name: t.cpu()}))
            with pytest.raises(TypeError):
                call(**dict(given, **{name: t.double()}))
            with pytest.raises((TypeError, ValueError)):
                call(**dict(given, **{name: t[..., :-1]}))
