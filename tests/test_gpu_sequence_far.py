"""Gradients of short_conv and selective_scan at steps that lie more than 2^31 numbers away from where they come from, by the definition."""
import pytest
import torch

from bmtk_amd import readout
from test_gpu_readout import U, close, gen

pytestmark = pytest.mark.gpu


def test_gradients_far_in_front_of_what_they_come_from():
    """2.7 billion inputs, 0 but for the last steps, whose dy alone is not 0: in front of those, where the states and dy are 0, only x has a gradient, what the last steps' state has, decayed."""
    steps, batch, dim, states, tail = 40_000, 32, 2080, 2, 48
    g = gen(12)
    x = torch.zeros(steps, batch, dim, dtype=torch.bfloat16, device="cuda")
    x[-tail:] = torch.randn(tail, batch, dim, generator=g).bfloat16().cuda()
    weight = torch.randn(dim, 4, generator=g).cuda()
    dx, _, _, ds = readout.short_conv_bwd(x, weight, x, silu=True)
    # (the widest of the last steps' taps: three in front of them; z is 0 there, where silu's slope is 1/2)
    assert not dx[:-tail - 3].any() and not ds.any() and dx[-tail - 3:-tail].any()
    del dx
    torch.cuda.empty_cache()
    dt = torch.full((1, 1, dim), -2.0, dtype=torch.bfloat16, device="cuda").expand(steps, batch, dim)
    rate = -torch.rand(dim, states, generator=g).cuda() ** 4
    shared = torch.randn(1, 1, 1, states, generator=g).bfloat16().cuda().expand(steps, batch, 1, states)
    _, _, saved = readout.selective_scan(x, dt, rate, shared, shared, softplus=True, save_state=True)
    assert not saved[:(steps - tail) // 16].any()
    d = readout.selective_scan_bwd(x, dt, rate, shared, shared, saved, x, softplus=True)
    some = readout.selective_scan(x[-tail:], dt[-tail:], rate, shared[-tail:], shared[-tail:], softplus=True, save_state=True)
    entering = readout.selective_scan_bwd(x[-tail:], dt[-tail:], rate, shared[-tail:], shared[-tail:], some[2], x[-tail:], softplus=True).d_state.double()
    for name in ("d_dt", "d_write", "d_read"):
        assert not getattr(d, name)[:-tail].any(), name
    delta = torch.nn.functional.softplus(torch.tensor(-2.0, dtype=torch.float64)).item()
    write = shared[0, 0, 0].double()
    # The last steps' own gradient, in either call: a sum of dy read decay of which each term is off by a rounding for each of up to 48 additions and four for each step that it decays, and
    # by ten of its exponent, below 7: 310 roundings of the terms' magnitudes, twice
    mag = 2 * 310 * U * x[-tail:].double().abs().sum(0).unsqueeze(2) * write.abs()
    for distance in (1, 2, 15, 16, 17, 100, 1000, 5000, 17_000, 33_000, steps - tail):
        by_step = delta * rate.double()
        decay = torch.exp((distance - 1) * by_step)
        part = entering * decay * write
        # a step's decay: its exponent off by ten roundings of itself (of the softplus, the rate, their product), or, of a stretch, whose deltas are added up, by one for each; the exponential
        # and a product for each step; four for what is made of it
        off = distance * 4 * U + (10 + distance) * U * (distance * by_step).abs() + 14 * U
        close(d.dx[steps - tail - distance], delta * part.sum(2), delta * ((part.abs() * off) + (decay * mag + 2.0 ** -126 * entering.abs()) * write.abs()).sum(2) + 2.0 ** -126,
              "dx, {} steps before".format(distance))
    off = steps * 4 * U + (10 + steps) * U * (steps * by_step).abs() + 14 * U
    decay = torch.exp((steps - tail) * by_step)
    close(d.d_state, entering * decay, entering.abs() * (decay * off + 2.0 ** -126) + decay * mag, "d_state")
