"""The readout operations against plain implementations in 64 bits.

Tolerances are bounds, made from the sums themselves: U = 2^-24 is half a step of fp32, a value rounded to type T is off by at most
eps(T) / 2 of itself (and half of the smallest subnormal), and a sum of k terms is off by at most k U times the sum of the terms' magnitudes."""
import math

import numpy as np
import pytest
import torch

from bmtk_amd import _lib, ops, readout, synthetic, training
from bmtk_amd.simulator import Glif3Simulator

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def close(got, want, error, what=""):
    """|got - want| <= error + the rounding to got's type, entry by entry; infinities and NaN at the same places."""
    dtype = got.dtype
    got, want, error = got.double().cpu(), want.double().cpu(), torch.as_tensor(error, dtype=torch.float64).cpu().expand(want.shape)
    assert got.shape == want.shape, what
    # what rounding takes to infinity: half a step above the largest value m = (2 - eps) 2^e, whose steps are eps 2^e, m (1 + eps / 4) and a little
    want = torch.where(want.abs() > torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4), torch.copysign(torch.tensor(math.inf, dtype=torch.float64), want), want)
    finite = torch.isfinite(want)
    assert torch.equal(finite, torch.isfinite(got)), what
    assert torch.equal(want.isnan(), got.isnan()) and torch.equal(want[~finite & ~want.isnan()], got[~finite & ~want.isnan()]), what
    got, want, error = got[finite], want[finite], error[finite]
    room = error + (want.abs() + error) * torch.finfo(dtype).eps / 2 + TINY[dtype]
    over = (got - want).abs() - room
    assert not over.numel() or over.max().item() <= 0, "{}: {:.3g} off where {:.3g} is allowed".format(
        what, (got - want).abs()[over.argmax()].item(), room[over.argmax()].item())


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------------------------------------------------------------
# spikes

def raster(steps, n, batch, p, seed):
    return torch.rand(steps, n, batch, generator=gen(seed)) < p


def pack(z, extra=1, garbage=False):
    """bool [steps, n, batch] -> int64 words on the device, ``extra`` words of padding a row."""
    steps = z.shape[0]
    flat = z.reshape(steps, -1).numpy()
    ne = flat.shape[1]
    words = (ne + 63) // 64
    full = np.ones((steps, (words + extra) * 64), bool) if garbage else np.zeros((steps, (words + extra) * 64), bool)
    full[:, :ne] = flat
    return torch.from_numpy(np.packbits(full, axis=1, bitorder="little").view(np.int64).copy()).cuda()


def spike_case(steps, n, batch, dim, dtype, p, seed=0, garbage=False):
    z = raster(steps, n, batch, p, seed)
    w = (torch.randn(n, dim, generator=gen(seed + 1))).to(dtype)
    dy = (torch.randn(steps, batch, dim, generator=gen(seed + 2))).to(dtype)
    return z, pack(z, garbage=garbage), w.cuda(), dy.cuda()


def spikes_check(z, bits, w, dy, batch):
    zd, wd, dyd = z.double(), w.double().cpu(), dy.double().cpu()
    steps, n = z.shape[:2]
    zt = zd.transpose(1, 2).reshape(steps * batch, n)
    dy2 = dyd.reshape(steps * batch, -1)
    y = readout.spike_readout(bits, w, batch)
    k = zt.sum(1, keepdim=True) + 64   # (joins of wavefronts and slices)
    close(y.view(steps * batch, -1), zt @ wd, k * U * (zt @ wd.abs()), "y")
    d_weight, dl_dz = readout.spike_readout_bwd(bits, w, dy, batch)
    k = zt.sum(0).unsqueeze(1) + 64
    close(d_weight, zt.t() @ dy2, k * U * (zt.t() @ dy2.abs()), "d_weight")
    # products and additions of a row's channels; operands in three parts of 8 bits each leave out products of up to 2^-24 of a term
    want, mag = dy2 @ wd.t(), dy2.abs() @ wd.abs().t()
    order = lambda a: a.view(steps, batch, n).transpose(1, 2).reshape(steps, n * batch)  # noqa: E731
    close(dl_dz, order(want), (w.shape[1] + 8) * 2 * U * order(mag), "dl_dz")
    again = readout.spike_readout_bwd(bits, w, dy, batch)
    assert torch.equal(again[0], d_weight) and torch.equal(again[1], dl_dz) and torch.equal(readout.spike_readout(bits, w, batch), y)
    none = readout.spike_readout_bwd(bits, w, dy, batch, spikes=False)
    assert none[1] is None and torch.equal(none[0], d_weight)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps,n,batch,dim,p", [
    (1, 1, 1, 1, 1.0), (1, 70, 1, 3, 0.3), (5, 450, 1, 64, 0.05), (3, 301, 12, 17, 0.05), (7, 100, 32, 64, 0.02), (4, 33, 45, 130, 0.1), (2, 5, 64, 256, 0.5),
    (2, 9, 100, 5, 0.2), (3, 40, 61, 33, 0.3), (130, 65, 3, 10, 0.01), (1, 20011, 1, 100, 0.01), (2, 3001, 16, 96, 0.003), (66, 2, 200, 4, 0.05), (40, 129, 1, 300, 0.5)])
def test_spikes_against_64_bits(steps, n, batch, dim, p, dtype):
    spikes_check(*spike_case(steps, n, batch, dim, dtype, p), batch)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps,n,batch,dim,p", [(2, 5003, 32, 33, 0.003), (1, 270011, 1, 20, 0.002), (3, 4001, 45, 9, 0.01), (64, 5003, 32, 33, 0.002)])
def test_spikes_of_steps_in_slices(steps, n, batch, dim, p, dtype):
    """And, the last one, a large product of rows that no load of 16 bytes divides."""
    spikes_check(*spike_case(steps, n, batch, dim, dtype, p), batch)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps,n,batch,dim", [(250, 20011, 32, 70), (670, 20011, 12, 128), (8003, 20011, 1, 257), (250, 20016, 32, 20), (671, 20011, 12, 31), (900, 20011, 9, 64), (2801, 20011, 3, 50),
                                                 (331, 20011, 24, 17), (399, 20011, 20, 33), (999, 20011, 8, 64)])
def test_large_products(steps, n, batch, dim, dtype):
    """Several tiles of rows to a workgroup, not a whole number of what it takes at once; the product in 64 bits on the device, step by step."""
    g = gen(steps)
    w, dy = torch.randn(n, dim, generator=g).to(dtype).cuda(), torch.randn(steps, batch, dim, generator=g).to(dtype).cuda()
    bits = torch.zeros(steps, (n * batch + 63) // 64, dtype=torch.int64, device="cuda")
    dl_dz = readout.spike_readout_bwd(bits, w, dy, batch)[1].view(steps, n, batch)
    wd = w.double()
    for t in range(0, steps, 40):
        d = dy[t:t + 40].double().reshape(-1, dim).t().contiguous()
        want, mag = (a.view(n, -1, batch).transpose(0, 1) for a in (wd @ d, wd.abs() @ d.abs()))
        # (products and additions of a row's channels, twice: see spikes_check)
        assert ((dl_dz[t:t + 40].double() - want).abs() <= (dim + 8) * 2 * U * mag).all()


@pytest.mark.parametrize("p", [0.0, 1.0])
@pytest.mark.parametrize("batch,n", [(1, 200), (12, 37), (64, 11), (130, 3)])
def test_nothing_fired_and_everything_fired(batch, n, p):
    z, bits, w, dy = spike_case(9, n, batch, 20, torch.float32, 0.0)
    z = torch.full_like(z, bool(p))
    spikes_check(z, pack(z), w, dy, batch)


def test_bits_behind_the_last_element_are_not_looked_at():
    for batch, n in ((1, 70), (12, 37), (5, 13)):
        z, bits, w, dy = spike_case(6, n, batch, 8, torch.float32, 0.2, garbage=True)
        assert bits[0, -1] == -1
        spikes_check(z, bits, w, dy, batch)


def test_rows_further_apart_and_weights_off_a_boundary():
    z, bits, w, dy = spike_case(5, 90, 12, 16, torch.bfloat16, 0.1)
    wide = torch.full((5, bits.shape[1] + 7), -1, dtype=torch.int64, device="cuda")
    wide[:, 3:3 + bits.shape[1]] = bits
    odd = torch.empty(90 * 16 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(90, 16)
    odd.copy_(w)
    odd_dy = torch.empty(5 * 12 * 16 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(5, 12, 16)
    odd_dy.copy_(dy)
    spikes_check(z, wide[:, 3:3 + bits.shape[1]], odd, odd_dy, 12)


def test_infinite_weights_of_neurons_that_did_not_fire_stay_out():
    z, bits, w, dy = spike_case(3, 50, 4, 8, torch.float32, 0.2)
    z[:, 7] = False
    w[7] = math.inf
    y = readout.spike_readout(pack(z), w, 4)
    assert torch.isfinite(y).all()


def test_infinite_gradients_reach_their_spikes_only():
    z, bits, w, dy = spike_case(3, 50, 4, 8, torch.float32, 0.2)
    dy[1, 2, 3] = math.inf
    w[:, 3] = w[:, 3].abs() + 0.1
    dl_dz = readout.spike_readout_bwd(bits, w, dy, 4)[1].view(3, 50, 4)
    assert (dl_dz[1, :, 2] == math.inf).all()
    dl_dz[1, :, 2] = 0
    assert torch.isfinite(dl_dz).all()


@pytest.mark.parametrize("steps,n,batch,dim", [(20, 9001, 32, 64), (40, 8111, 12, 100), (701, 5003, 1, 128), (30, 10016, 4, 300), (60, 9000, 8, 96), (31, 10000, 16, 65),
                                               (9, 9000, 64, 61), (7, 5003, 45, 260)])
def test_products_in_parts(steps, n, batch, dim):
    """fp32 of more products than are made in fp32 instructions (3e8): every way in which the result reaches memory, one pass over the channels and more,
    partial tiles; then with an infinity in a weight, an infinity and a NaN in a gradient: those reach what they take part in and nothing else."""
    g = gen(steps)
    w, dy = torch.randn(n, dim, generator=g), torch.randn(steps, batch, dim, generator=g)
    bits = torch.zeros(steps, (n * batch + 63) // 64, dtype=torch.int64, device="cuda")

    def dl_dz():
        return readout.spike_readout_bwd(bits, w.cuda(), dy.cuda(), batch)[1].view(steps, n, batch)

    def products(a, b):
        return (b.double().view(steps * batch, dim) @ a.double().t()).view(steps, batch, n).transpose(1, 2)
    first = dl_dz()
    close(first, products(w, dy), (dim + 8) * 2 * U * products(w.abs(), dy.abs()), "dl_dz")
    w[5, dim - 1], dy[steps - 1, batch - 1, 0], dy[0, 0, dim // 2] = math.inf, -math.inf, math.nan
    w[5, 0] = 2.0
    got, want = dl_dz().cpu(), products(w, dy)
    reached = torch.zeros(steps, n, batch, dtype=torch.bool)
    reached[:, 5], reached[steps - 1, :, batch - 1], reached[0, :, 0] = True, True, True
    assert torch.isfinite(got[~reached]).all()
    assert torch.equal(got[reached].isnan(), want[reached].isnan())
    inf = reached & want.isinf()
    assert inf.any() and torch.equal(got[inf].double(), want[inf])
    close(got[~reached], want[~reached], (dim + 8) * 2 * U * products(w.nan_to_num(0, 0, 0).abs(), dy.nan_to_num(0, 0, 0).abs())[~reached], "the rest")


def test_no_steps():
    bits, w = torch.zeros(0, 5, dtype=torch.int64, device="cuda"), torch.ones(20, 3, device="cuda")
    assert readout.spike_readout(bits, w, 4).shape == (0, 4, 3)
    d_weight, dl_dz = readout.spike_readout_bwd(bits, w, torch.zeros(0, 4, 3, device="cuda"), 4)
    assert (d_weight == 0).all() and dl_dz.shape == (0, 80)


# ---------------------------------------------------------------------------------------------------------------------
# recurrence

def scan_reference(x, a, state, lengths, dh, d_last):
    """Everything in 64 bits, step by step, and bounds of the errors: every value passes at most two roundings a step (a product, a sum), two more for
    every 16 steps (the join of wavefronts), and a few at its ends.  Terms are followed with their magnitudes: S the sum of them,
    G the sum of them times the roundings each has passed."""
    x, a, dh = x.double().cpu(), a.double().cpu(), dh.double().cpu()
    steps, batch, dim = x.shape
    lengths = torch.full((batch,), steps) if lengths is None else lengths.cpu().clamp(0, steps)
    gate = lambda t: (a.expand(batch, dim) if a.dim() == 1 else a[t].repeat_interleave(dim // a.shape[2], 1))  # noqa: E731
    s = torch.zeros(batch, dim, dtype=torch.float64) if state is None else state.double().cpu()
    hs, err, before, before_err = (torch.zeros(steps, batch, dim, dtype=torch.float64) for _ in range(4))
    S, G = s.abs(), 12.0 * s.abs()
    for t in range(steps):
        on = (t < lengths).unsqueeze(1)
        g = torch.where(on, gate(t), 1.0)
        xt = torch.where(on, x[t], 0.0)
        before[t], before_err[t] = s, U * G
        s = g * s + xt
        S, G = g.abs() * S + xt.abs(), torch.where(on, g.abs() * (G + 2.2 * S) + 12.0 * xt.abs(), G)
        hs[t], err[t] = torch.where(on, s, 0.0), torch.where(on, U * G, 0.0)
    out = dict(h=hs, h_err=err, last=s, last_err=U * G)
    c = torch.zeros(batch, dim, dtype=torch.float64) if d_last is None else d_last.double().cpu()
    S, G = c.abs(), 12.0 * c.abs()
    dx, dx_err, da, da_err = (torch.zeros(steps, batch, dim, dtype=torch.float64) for _ in range(4))
    for t in range(steps - 1, -1, -1):
        on = (t < lengths).unsqueeze(1)
        dt = torch.where(on, dh[t], 0.0)
        g = dt + c
        S, G = S + dt.abs(), G + 12.0 * dt.abs()
        dx[t], dx_err[t] = torch.where(on, g, 0.0), torch.where(on, U * G, 0.0)
        da[t] = torch.where(on, g * before[t], 0.0)
        da_err[t] = torch.where(on, U * G * before[t].abs() + (g.abs() + U * G) * (before_err[t] + 2 * U * before[t].abs()), 0.0)
        gt = torch.where(on, gate(t), 1.0)
        c = gt * g
        S, G = gt.abs() * S, torch.where(on, gt.abs() * (G + 2.2 * S), G)
    out.update(dx=dx, dx_err=dx_err, d_state=c, d_state_err=U * (G + S))
    if a.dim() == 1:
        # a sum of steps * batch terms in any order
        out.update(d_decay=da.sum((0, 1)), d_decay_err=da_err.sum((0, 1)) + min(steps * batch, 4000) * U * da.abs().sum((0, 1)))
    else:
        split = lambda v: v.view(steps, batch, a.shape[2], -1).sum(3)  # noqa: E731
        out.update(d_decay=split(da), d_decay_err=split(da_err) + (dim // a.shape[2]) * U * split(da.abs()))
    return out


def scan_case(steps, batch, dim, groups, dtype, gates, lengths=None, seed=0, with_state=True):
    g = gen(seed)
    x = torch.randn(steps, batch, dim, generator=g).to(dtype).cuda()
    a = torch.rand(dim, generator=g) * 1.5 - 0.5 if groups == 0 else torch.rand(steps, batch, groups, generator=g) * 1.4 - 0.4
    state = torch.randn(batch, dim, generator=g).cuda() if with_state else None
    dh = torch.randn(steps, batch, dim, generator=g).to(dtype).cuda()
    d_last = torch.randn(batch, dim, generator=g).cuda() if with_state else None
    if lengths is not None:
        lengths = torch.tensor([lengths[b % len(lengths)] for b in range(batch)], dtype=torch.int32).cuda()
    return x, a.clamp(-1, 1).to(gates).cuda(), state, lengths, dh, d_last


def scan_check(x, a, state, lengths, dh, d_last):
    want = scan_reference(x, a, state, lengths, dh, d_last)
    h, last, saved = readout.gated_scan(x, a, state, lengths, save_state=True)
    close(h, want["h"], want["h_err"], "h")
    close(last, want["last"], want["last_err"], "last")
    h2, last2 = readout.gated_scan(x, a, state, lengths)
    assert torch.equal(h2, h) and torch.equal(last2, last)
    dx, d_decay, d_state = readout.gated_scan_bwd(x, a, saved, dh, d_last, lengths)
    close(dx, want["dx"], want["dx_err"], "dx")
    close(d_state, want["d_state"], want["d_state_err"], "d_state")
    close(d_decay, want["d_decay"], want["d_decay_err"], "d_decay")
    again = readout.gated_scan_bwd(x, a, saved, dh, d_last, lengths)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, d_decay, d_state)))
    return h, last, dx, d_decay, d_state


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32)]


@pytest.mark.parametrize("dtype,gates", TYPES)
@pytest.mark.parametrize("steps,batch,dim,groups", [
    (1, 1, 1, 1), (1, 3, 130, 130), (1, 2, 12, 4), (1, 5, 7, 0), (2, 2, 5, 5), (15, 1, 64, 64), (16, 2, 100, 100), (17, 3, 66, 0), (127, 1, 3, 3), (128, 2, 128, 4),
    (129, 2, 128, 1), (257, 3, 99, 3), (300, 2, 10, 5), (300, 1, 192, 2), (100, 4, 33, 1), (700, 1, 40, 0), (1030, 2, 70, 70), (2100, 1, 66, 22)])
def test_recurrence_against_64_bits(steps, batch, dim, groups, dtype, gates):
    scan_check(*scan_case(steps, batch, dim, groups, dtype, gates))


@pytest.mark.parametrize("groups", [0, 40, 4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sequences_of_different_lengths(groups, dtype):
    """... among them none at all and one step; what lies behind them is NaN and is not read."""
    steps = 530
    x, a, state, lengths, dh, d_last = scan_case(steps, 7, 40, groups, dtype, torch.float32, lengths=[0, 1, 530, 16, 17, 255, 529])
    for b, n in enumerate(lengths.tolist()):
        for t in (x, dh) + ((a,) if groups else ()):
            t[n:, b] = math.nan
    clean = [torch.nan_to_num(t, nan=0.0) for t in (x, a, dh)]
    h, last, dx, d_decay, d_state = scan_check(x, a, state, lengths, dh, d_last)
    got = scan_check(clean[0], clean[1], state, lengths, clean[2], d_last)
    assert all(torch.equal(p, q) for p, q in zip(got, (h, last, dx, d_decay, d_state)))
    assert (h[0, 0] == 0).all() and torch.equal(last[0], state[0]) and torch.equal(d_state[0], d_last[0])


def test_lengths_outside_count_as_the_nearer_end():
    x, a, state, _, dh, d_last = scan_case(40, 3, 8, 8, torch.float32, torch.float32)
    outside, inside = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([-5, 41, 1 << 30], [0, 40, 40]))
    got, want = (readout.gated_scan(x, a, state, n, save_state=True) for n in (outside, inside))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    one = [readout.gated_scan(x[:1], a[:1], state, n) for n in (outside, inside.clamp(max=1))]
    assert torch.equal(one[0][0], one[1][0]) and torch.equal(one[0][1], one[1][1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,dim,groups", [(1, 64, 64), (1, 3, 0), (2, 96, 3), (1, 1000, 1000), (3, 50, 25)])
def test_long_sequences_in_stretches(batch, dim, groups, dtype):
    scan_check(*scan_case(6007, batch, dim, groups, dtype, torch.float32, lengths=[6007, 3111]))


@pytest.mark.parametrize("dtype,gates,batch,dim,groups,lengths", [
    (torch.bfloat16, torch.bfloat16, 2, 260, 260, None), (torch.float32, torch.float32, 2, 260, 0, [8200, 5001]), (torch.bfloat16, torch.float32, 1, 520, 8, [8200]),
    (torch.float16, torch.float16, 2, 260, 26, [4099, 8200]), (torch.bfloat16, torch.bfloat16, 2, 261, 9, [8199, 0])])
def test_long_sequences_in_one_pass(dtype, gates, batch, dim, groups, lengths):
    """65 stretches of a chain in five groups, the last one not whole."""
    scan_check(*scan_case(8200, batch, dim, groups, dtype, gates, lengths=lengths))


@pytest.mark.parametrize("dtype,batch,dim,groups", [(torch.float32, 4, 100, 0), (torch.bfloat16, 20, 64, 64), (torch.float16, 7, 60, 5), (torch.float32, 33, 30, 30)])
@pytest.mark.parametrize("steps", [300, 2433, 2432])
def test_between_stretches_and_one_pass(steps, batch, dim, groups, dtype):
    """Three stretches of few and of many columns; 19 and 20 of them."""
    scan_check(*scan_case(steps, batch, dim, groups, dtype, dtype, lengths=[steps, 0, 257, steps - 1, 129]))


@pytest.mark.parametrize("steps", [128, 129, 144, 200, 256, 257])
@pytest.mark.parametrize("dtype,gates,dim,groups", [(torch.float32, torch.float32, 33, 0), (torch.bfloat16, torch.float32, 64, 64), (torch.bfloat16, torch.bfloat16, 96, 6),
                                                    (torch.float16, torch.float16, 31, 31)])
def test_one_round_of_many_wavefronts(steps, dtype, gates, dim, groups):
    """And what is just too short or too long for it."""
    scan_check(*scan_case(steps, 5, dim, groups, dtype, gates, lengths=[steps, 0, 1, 127, steps - 1]))


@pytest.mark.parametrize("dtype,dim,groups", [(torch.float32, 128, 128), (torch.bfloat16, 256, 0), (torch.bfloat16, 256, 4), (torch.float16, 129, 43)])
def test_stretches_of_several_rounds(dtype, dim, groups):
    """Many columns: two or three stretches of two rounds and more."""
    scan_check(*scan_case(700, 64, dim, groups, dtype, dtype, lengths=[700, 300, 0, 511]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    """[sequences, steps, channels] transposed, parts of wider rows, rows on odd addresses, gates that sequences share, no state."""
    x, a, state, _, dh, d_last = scan_case(150, 3, 20, 20, dtype, dtype)
    plain = scan_check(x, a, state, None, dh, d_last)

    def other(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def wider(t, left):
        w = torch.full((t.shape[0], t.shape[1], t.shape[2] + 5), math.nan, dtype=t.dtype, device="cuda")
        w[:, :, left:left + t.shape[2]] = t
        return w[:, :, left:left + t.shape[2]]
    for change in (other, lambda t: wider(t, 1), lambda t: wider(t, 2)):
        got = scan_check(change(x), change(a), state, None, change(dh), d_last)
        for p, q in zip(got, plain):   # (16-bit types: a lane takes two channels of even rows; the arithmetic is the same)
            assert torch.equal(p, q)
    shared = a[:, :1].expand(150, 3, 20)
    scan_check(x, shared, None, None, dh, None)


def test_decays_of_nothing_and_of_everything():
    x, a, state, _, dh, d_last = scan_case(400, 2, 8, 8, torch.float32, torch.float32)
    for v in (0.0, 1.0, -1.0):
        scan_check(x, torch.full_like(a, v), state, None, dh, d_last)
    # gates above 1 whose products leave fp32: a state of nothing stays nothing until there is an input
    a = torch.full_like(a, 1.0e3)
    x.zero_()
    x[-1] = 2.0
    h, last = readout.gated_scan(x, a, None)
    assert (h[:-1] == 0).all() and (h[-1] == 2.0).all() and (last == 2.0).all()


def test_steps_one_at_a_time_are_a_whole_run():
    x, a, state, _, _, _ = scan_case(20, 3, 24, 24, torch.float32, torch.float32)
    whole, last = readout.gated_scan(x, a, state)
    now = state
    for t in range(20):
        h, now = readout.gated_scan(x[t:t + 1], a[t:t + 1], now)
        # the same products and sums, those of a run's first 16 steps in the same order
        assert torch.equal(h[0], now)
        close(h[0], whole[t].double(), 64 * U * (whole[t].double().abs() + 1))


@pytest.mark.parametrize("groups", [0, 6, 2])
def test_recurrence_gradients_are_differences(groups):
    """The change of a loss, computed in 64 bits from the definition, along a random direction of all inputs at once."""
    x, a, state, lengths, dh, d_last = scan_case(60, 3, 6, groups, torch.float32, torch.float32, lengths=[60, 23, 0])
    _, _, saved = readout.gated_scan(x, a, state, lengths, save_state=True)
    dx, d_decay, d_state = readout.gated_scan_bwd(x, a, saved, dh, d_last, lengths)
    g = gen(9)
    vx, va, vs = (torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (x, a, state))

    def loss(e):
        r = scan_reference(x.cpu().double() + e * vx, a.cpu().double() + e * va, state.cpu().double() + e * vs, lengths, dh, d_last)
        return ((r["h"] * dh.cpu().double()).sum() + (r["last"] * d_last.cpu().double()).sum()).item()
    slope = (loss(1e-6) - loss(-1e-6)) / 2e-6
    along = sum((d.cpu().double() * v).sum().item() for d, v in ((dx, vx), (d_decay, va), (d_state, vs)))
    size = sum((d.cpu().double() * v).abs().sum().item() for d, v in ((dx, vx), (d_decay, va), (d_state, vs)))
    assert abs(slope - along) <= 1e-5 * size   # (fp32 gradients, some hundred roundings; 1e-6^2 of the third derivative)


def test_no_steps_of_a_sequence():
    state = torch.randn(2, 3, device="cuda")
    x = torch.zeros(0, 2, 3, device="cuda")
    h, last, saved = readout.gated_scan(x, torch.ones(3, device="cuda"), state, save_state=True)
    assert h.shape == (0, 2, 3) and torch.equal(last, state)
    dx, d_decay, d_state = readout.gated_scan_bwd(x, torch.ones(3, device="cuda"), saved, x, state)
    assert dx.shape == x.shape and (d_decay == 0).all() and torch.equal(d_state, state)
    assert (readout.gated_scan(x, torch.ones(3, device="cuda"))[1] == 0).all()


# ---------------------------------------------------------------------------------------------------------------------
# log probabilities

def logprobs_reference(logits, tokens, top, ignore=-100, d_logp=None, d_entropy=None):
    x, tokens = logits.double().cpu(), tokens.cpu()
    lead, vocab = x.shape[:-1], x.shape[-1]
    x, token = x.reshape(-1, vocab), tokens.reshape(-1)
    lse = torch.logsumexp(x, 1)
    lse = torch.where(x.isnan().any(1) | (x == math.inf).any(1), math.nan, lse)
    lp = torch.where((x == -math.inf) & ~lse.isnan().unsqueeze(1), -math.inf, x - lse.unsqueeze(1))
    p = torch.exp(lp)
    H = -torch.where(p > 0, p * lp, torch.where(p.isnan(), math.nan, 0.0)).sum(1)
    inside = (token >= 0) & (token < vocab)
    at = torch.where(inside, token, 0)
    logp = torch.where(token == ignore, 0.0, torch.where(inside, lp.gather(1, at.unsqueeze(1)).squeeze(1), math.nan))
    # (numpy's sort puts NaN last, so ascending order of -x would too: they are made the largest)
    order = torch.sort(torch.where(x.isnan(), math.inf, x) + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    out = dict(lse=lse.view(lead), entropy=H.view(lead), logp=logp.view(lead), top_index=order.view(lead + (top,)), top_logp=lp.gather(1, order).view(lead + (top,)))
    # errors: sums of positive terms, each off by 3 roundings and that of its exponent (up to 40 in magnitude, or it does not count), added in at most
    # vocab / 64 + 64 additions; lse and logits round at their own size
    n = (vocab / 64 + 64 + 3 + 2 * 40) * U
    big = torch.where(torch.isfinite(lse), lse.abs(), 0.0) + torch.where(torch.isfinite(x), x.abs(), 0.0).amax(1)
    spread = torch.where(p > 0, p * lp.abs(), 0.0).sum(1) + 1
    out.update(lse_err=(n + 4 * U * big).view(lead), entropy_err=(4 * n * spread + 4 * U * big).view(lead))
    out["logp_err"] = out["lse_err"]
    out["top_err"] = out["lse_err"].unsqueeze(-1).expand(lead + (top,))
    if d_logp is not None or d_entropy is not None:
        dl = torch.zeros(lead, dtype=torch.float64) if d_logp is None else d_logp.double().cpu()
        de = torch.zeros(lead, dtype=torch.float64) if d_entropy is None else d_entropy.double().cpu()
        dl, de = torch.where(token == ignore, 0.0, dl.reshape(-1)).unsqueeze(1), de.reshape(-1).unsqueeze(1)
        lq = torch.where(p > 0, lp, 0.0)
        d = -p * dl - de * p * (lq + H.unsqueeze(1))
        d[torch.arange(len(at)), at] += torch.where((lse > -math.inf) & inside, dl.squeeze(1), 0.0)
        out["d"] = d.view(logits.shape)
        per = (lq.abs() + 40) * 2 * U + out["lse_err"].reshape(-1, 1) * 2
        err = p * per * (dl.abs() + de.abs() * (lq.abs() + H.unsqueeze(1) + 1)) + p * de.abs() * (out["entropy_err"].reshape(-1, 1) + out["lse_err"].reshape(-1, 1))
        out["d_err"] = (err + 4 * U * (dl.abs() * p)).view(logits.shape)
        out["d_err"].view(-1, vocab)[torch.arange(len(at)), at] += 2 * U * dl.squeeze(1).abs()
    return out


def logprobs_check(logits, tokens, top, d_logp=None, d_entropy=None, ignore=-100):
    want = logprobs_reference(logits, tokens, top, ignore, d_logp, d_entropy)
    r = readout.token_logprobs(logits, tokens, top=top, ignore=ignore)
    close(r.lse, want["lse"], want["lse_err"], "lse")
    close(r.logp, want["logp"], want["logp_err"], "logp")
    close(r.entropy, want["entropy"], want["entropy_err"], "entropy")
    if top:
        assert torch.equal(r.top_index.cpu(), want["top_index"])
        close(r.top_logp, want["top_logp"], want["top_err"], "top_logp")
    else:
        assert r.top_logp is None and r.top_index is None
    again = readout.token_logprobs(logits, tokens, top=top, ignore=ignore)
    assert all(torch.equal(torch.nan_to_num(p), torch.nan_to_num(q)) for p, q in zip(again, r) if p is not None)
    if d_logp is not None or d_entropy is not None:
        d = readout.token_logprobs_bwd(logits, tokens, r, d_logp, d_entropy, ignore=ignore)
        close(d, want["d"], want["d_err"], "d_logits")
    return r


def logits_case(rows, vocab, dtype, seed=0, masked=0.0, ignored=0.1, scale=3.0):
    g = gen(seed)
    x = scale * torch.randn(rows, vocab, generator=g)
    if masked:
        x[torch.rand(rows, vocab, generator=g) < masked] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    tokens[torch.rand(rows, generator=g) < ignored] = -100
    return x.to(dtype).cuda(), tokens.cuda(), torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 2, 2), (5, 10, 3), (33, 16, 16), (7, 17, 5), (20, 64, 64), (3, 65, 1), (9, 511, 64), (4, 512, 0), (4, 1000, 20), (3, 2048, 7), (6, 2049, 64), (3, 5003, 33),
    (1000, 10, 0), (2, 40000, 20), (1, 131072, 64), (3, 100003, 5), (770, 4097, 2)])
def test_logprobs_against_64_bits(rows, vocab, top, dtype):
    x, tokens, dl, de = logits_case(rows, vocab, dtype)
    logprobs_check(x, tokens, top, dl, de)


@pytest.mark.parametrize("vocab", [12, 60, 700, 9001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits(vocab, dtype):
    """Half of them -inf; a row with one left, a row with none, a row of the type's lowest value; tokens among the masked."""
    x, tokens, dl, de = logits_case(9, vocab, dtype, masked=0.5, ignored=0.0)
    x[1] = -math.inf
    x[1, vocab // 2] = 1.5
    x[2] = -math.inf
    x[3] = torch.finfo(dtype).min
    x[4] = torch.finfo(dtype).min
    x[4, 3] = 2.0
    x[5, tokens[5]] = -math.inf
    x[6] = torch.finfo(dtype).max
    x[6, 1] = torch.finfo(dtype).min
    r = logprobs_check(x, tokens, min(vocab, 64), dl, de)
    assert r.lse[2] == -math.inf and r.entropy[2] == 0 and r.logp[2] == -math.inf
    assert (readout.token_logprobs_bwd(x, tokens, r, dl, de)[2] == 0).all()


@pytest.mark.parametrize("vocab", [10, 64, 300, 5000])
def test_rows_with_nan_or_infinity(vocab):
    x, tokens, dl, de = logits_case(5, vocab, torch.float32, ignored=0.0)
    x[1, 7] = math.nan
    x[2, 3] = math.inf
    x[3] = math.nan
    r = logprobs_check(x, tokens, 4)
    assert r.top_index[1, 0] == 7 and r.top_index[2, 0] == 3 and r.top_index[3].tolist() == [0, 1, 2, 3]
    d = readout.token_logprobs_bwd(x, tokens, r, dl, de)
    assert d[1:4].isnan().all() and torch.isfinite(d[[0, 4]]).all()


@pytest.mark.parametrize("vocab", [16, 64, 1500, 20001])
@pytest.mark.parametrize("shape", ["equal", "zeros of both signs", "rising", "falling", "few values"])
def test_orders_that_are_hard_on_the_alternatives(vocab, shape):
    i = torch.arange(vocab, dtype=torch.float32)
    x = {"equal": torch.full((vocab,), 0.25), "zeros of both signs": torch.where(i % 2 == 0, -0.0, 0.0), "rising": i / 512, "falling": -i / 512,
         "few values": (i * 7919 % 5)}[shape].expand(3, vocab).contiguous().cuda()
    logprobs_check(x, torch.tensor([0, vocab // 2, vocab - 1]).cuda(), min(vocab, 64))


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_that_are_ignored_or_outside(dtype):
    x, tokens, dl, de = logits_case(6, 700, dtype, ignored=0.0)
    tokens[:] = torch.tensor([-100, 3, -1, 700, 699, 0])
    r = logprobs_check(x, tokens, 2)
    assert r.logp[0] == 0 and r.logp[2].isnan() and r.logp[3].isnan()
    d = readout.token_logprobs_bwd(x, tokens, r, dl)
    assert (d[0] == 0).all() and d[2:4].isnan().all()
    tokens[2:4] = 5
    logprobs_check(x, torch.where(tokens == -100, 7, tokens), 2, dl, de, ignore=7)
    logprobs_check(x, tokens, 2, None, de)
    logprobs_check(x, tokens, 2, dl, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [10, 300, 3001])
def test_padding_of_any_content(dtype, vocab):
    """Rows without a token that hold NaN and infinities: what nobody asks about has no gradient."""
    x, tokens, dl, de = logits_case(6, vocab, dtype, ignored=0.0)
    x[1], x[2, 3], x[4, 0] = math.nan, math.inf, math.nan
    tokens[1:3] = -100
    r = readout.token_logprobs(x, tokens)
    de[1:3] = 0.0
    for d_entropy in (None, de):
        d = readout.token_logprobs_bwd(x, tokens, r, dl, d_entropy)
        assert (d[1:3] == 0).all() and d[4].isnan().all()
        kept = torch.tensor([0, 3, 5])
        part = readout.LogProbs(*(None if t is None else t[kept] for t in r))
        assert torch.equal(d[kept], readout.token_logprobs_bwd(x[kept], tokens[kept], part, dl[kept], None if d_entropy is None else de[kept]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [30, 333, 3000, 20000])
def test_rows_of_any_distance_and_address(vocab, dtype):
    x, tokens, dl, de = logits_case(6, vocab, dtype)
    want = readout.token_logprobs(x, tokens, top=3)
    d = readout.token_logprobs_bwd(x, tokens, want, dl, de)
    for left, wide in ((0, 3), (1, 8), (3, 16)):
        w = torch.full((6, vocab + wide), math.nan, dtype=dtype, device="cuda")
        part = w[:, left:left + vocab]
        part.copy_(x)
        r = logprobs_check(part, tokens, 3, dl, de)
        assert torch.equal(r.top_index, want.top_index)
        # in place, among neighbours that stay as they are
        got = readout.token_logprobs_bwd(part, tokens, want, dl, de, out=part)
        assert got is part and torch.equal(part, d) and w[:, :left].isnan().all() and w[:, left + vocab:].isnan().all()
    out = torch.full((6, vocab + 1), 3.0, dtype=dtype, device="cuda")
    readout.token_logprobs_bwd(x, tokens, want, dl, de, out=out[:, 1:])
    assert torch.equal(out[:, 1:], d) and (out[:, 0] == 3.0).all()
    cube = x.view(2, 3, vocab)
    r = readout.token_logprobs(cube, tokens.view(2, 3), top=3)
    assert r.logp.shape == (2, 3) and r.top_index.shape == (2, 3, 3) and torch.equal(r.logp.view(-1), want.logp)
    assert torch.equal(readout.token_logprobs_bwd(cube, tokens.view(2, 3), r, dl.view(2, 3), de.view(2, 3)).view(6, vocab), d)


def test_logprobs_gradients_are_differences():
    x, tokens, dl, de = logits_case(6, 50, torch.float32, masked=0.2)
    r = readout.token_logprobs(x, tokens)
    d = readout.token_logprobs_bwd(x, tokens, r, dl, de).cpu().double()
    v = torch.randn(x.shape, generator=gen(4), dtype=torch.float64)

    def loss(e):
        w = logprobs_reference(x.cpu().double() + e * v, tokens, 0)
        at = torch.isfinite(w["logp"])   # (a masked token's log probability stays -inf)
        return ((w["logp"] * dl.cpu().double())[at].sum() + (w["entropy"] * de.cpu().double()).sum()).item()
    masked_token = (r.logp == -math.inf).cpu()
    d[masked_token] = readout.token_logprobs_bwd(x, tokens, r, None, de).cpu().double()[masked_token]
    slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
    assert abs(slope - (d * v).sum().item()) <= 1e-5 * (d * v).abs().sum().item()


def test_no_rows():
    r = readout.token_logprobs(torch.zeros(0, 5, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), top=2)
    assert r.logp.shape == (0,) and r.top_index.shape == (0, 2)
    d = readout.token_logprobs_bwd(torch.zeros(0, 5, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), r, r.logp)
    assert d.shape == (0, 5)


# ---------------------------------------------------------------------------------------------------------------------
# as they are used

def test_refusals_of_device_tensors():
    w, bits = torch.ones(20, 4, device="cuda"), torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    x, a = torch.ones(5, 2, 6, device="cuda"), torch.ones(6, device="cuda")
    logits, tokens = torch.ones(3, 9, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    r = readout.token_logprobs(logits, tokens)
    one = torch.ones(3, device="cuda")
    saved = torch.zeros(1, 2, 6, device="cuda")
    for error, word, call in [
            (ValueError, "words per step", lambda: readout.spike_readout(bits, w, 8)), (TypeError, "bits", lambda: readout.spike_readout(bits.int(), w, 4)),
            (TypeError, "weight", lambda: readout.spike_readout(bits, w.double(), 4)), (ValueError, "batch", lambda: readout.spike_readout(bits, w, 0)),
            (ValueError, "contiguous", lambda: readout.spike_readout(bits, w.t().contiguous().t(), 4)), (ValueError, "next to", lambda: readout.spike_readout(torch.zeros(2, 3, dtype=torch.int64, device="cuda").t(), w, 4)),
            (ValueError, "dy must be", lambda: readout.spike_readout_bwd(bits, w, torch.ones(3, 4, 5, device="cuda"), 4)),
            (TypeError, "dy", lambda: readout.spike_readout_bwd(bits, w, torch.ones(3, 4, 4, device="cuda").half(), 4)),
            (ValueError, "requires gradients", lambda: readout.spike_readout(bits, w.clone().requires_grad_(), 4)),
            (ValueError, "decay", lambda: readout.gated_scan(x, a[:3])), (ValueError, "decay", lambda: readout.gated_scan(x, torch.ones(5, 2, 4, device="cuda"))),
            (ValueError, "decay", lambda: readout.gated_scan(x, torch.ones(4, 2, 6, device="cuda"))), (TypeError, "decay", lambda: readout.gated_scan(x, a.half())),
            (ValueError, "x must be", lambda: readout.gated_scan(x[0], a)), (ValueError, "next to", lambda: readout.gated_scan(x.transpose(1, 2).contiguous().transpose(1, 2), a)),
            (ValueError, "state", lambda: readout.gated_scan(x, a, torch.ones(6, device="cuda"))), (TypeError, "state", lambda: readout.gated_scan(x, a, torch.ones(2, 6, device="cuda").half())),
            (TypeError, "lengths", lambda: readout.gated_scan(x, a, None, torch.ones(2, dtype=torch.int64, device="cuda"))),
            (ValueError, "lengths", lambda: readout.gated_scan(x, a, None, torch.ones(3, dtype=torch.int32, device="cuda"))),
            (ValueError, "saved", lambda: readout.gated_scan_bwd(x, a, saved[:, :1], x)), (ValueError, "dh", lambda: readout.gated_scan_bwd(x, a, saved, x[:4])),
            (ValueError, "d_last", lambda: readout.gated_scan_bwd(x, a, saved, x, torch.ones(2, 5, device="cuda"))),
            (ValueError, "tokens", lambda: readout.token_logprobs(logits, tokens[:2])), (TypeError, "tokens", lambda: readout.token_logprobs(logits, tokens.int())),
            (ValueError, "top", lambda: readout.token_logprobs(logits, tokens, top=10)), (ValueError, "top", lambda: readout.token_logprobs(torch.ones(3, 99, device="cuda"), tokens, top=65)),
            (ValueError, "next to", lambda: readout.token_logprobs(torch.ones(9, 3, device="cuda").t(), tokens)),
            (ValueError, "d_logp", lambda: readout.token_logprobs_bwd(logits, tokens, r)), (ValueError, "d_logp", lambda: readout.token_logprobs_bwd(logits, tokens, r, one[:2])),
            (ValueError, "shares memory", lambda: _shifted(r, tokens, one)),
            (TypeError, "out", lambda: readout.token_logprobs_bwd(logits, tokens, r, one, out=logits.half()))]:
        with pytest.raises(error, match=word):
            call()
    leaf = w.clone().requires_grad_()
    with torch.no_grad():
        assert not readout.spike_readout(bits, leaf, 4).requires_grad


def _shifted(r, tokens, one):
    both = torch.ones(4, 9, device="cuda")
    return readout.token_logprobs_bwd(both[:3], tokens, r, one, out=both[1:])


def test_decays_further_apart():
    """One decay per channel, every other entry of a tensor: what is computed from must outlive the call's results being made."""
    dim = 1 << 20
    g = gen(11)
    x = torch.randn(2, 1, dim, generator=g).bfloat16().cuda()
    decay = torch.rand(2 * dim, generator=g).cuda()[::2]
    for _ in range(3):
        h, last, saved = readout.gated_scan(x, decay, save_state=True)
        got = readout.gated_scan_bwd(x, decay, saved, x)
        want_h, want_last, want_saved = readout.gated_scan(x, decay.clone(), save_state=True)
        want = readout.gated_scan_bwd(x, decay.clone(), want_saved, x)
        for p, q in zip((h, last, saved, *got), (want_h, want_last, want_saved, *want)):
            assert torch.equal(p, q)
        del h, last, saved, got, want_h, want_last, want_saved, want, p, q


def everything(s):
    """One pass of all operations, as a training step makes them; what it returns."""
    y = readout.spike_readout(s["bits"], s["w"], s["batch"])
    h, last, saved = readout.gated_scan(y, s["decay"], s["state"], save_state=True)
    r = readout.token_logprobs(h, s["labels"], top=2)
    dh = readout.token_logprobs_bwd(h, s["labels"], r, s["d_logp"])
    dy, d_decay, d_state = readout.gated_scan_bwd(y, s["decay"], saved, dh, last)
    d_weight, dl_dz = readout.spike_readout_bwd(s["bits"], s["w"], dy, s["batch"])
    big = readout.token_logprobs(s["logits"], s["tokens"], top=5)   # in slices, with a workspace
    one = readout.spike_readout(s["wide"], s["w_wide"], 1)          # likewise
    return [y, h, last, *r, dh, dy, d_decay, d_state, d_weight, dl_dz, *big, one]


def chain_case(seed, steps=700, n=60, batch=4, dim=10):
    z, bits, w, _ = spike_case(steps, n, batch, dim, torch.float32, 0.05, seed=seed)
    g = gen(seed + 5)
    x, tokens, _, _ = logits_case(2, 50001, torch.bfloat16, seed=seed)
    zw, wide, w_wide, _ = spike_case(1, 30000, 1, 8, torch.float32, 0.01, seed=seed)
    return dict(bits=bits, w=w, batch=batch, decay=torch.rand(dim, generator=g).cuda(), state=torch.randn(batch, dim, generator=g).cuda(),
                labels=torch.randint(0, dim, (steps, batch), generator=g).cuda(), d_logp=torch.randn(steps, batch, generator=g).cuda(), logits=x, tokens=tokens,
                wide=wide, w_wide=w_wide)


def test_captured_and_replayed():
    """Two graphs of the same operations, replayed in turn with eager work between, on inputs that change."""
    cases = [chain_case(s) for s in (0, 1, 2)]
    want = [[t.clone() for t in everything(c)] for c in cases]
    graphs = []
    for k in (0, 1):
        held = {name: t.clone() if torch.is_tensor(t) else t for name, t in cases[k].items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            everything(held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = everything(held)
        graphs.append((graph, held, out))
    for turn in range(4):
        for k, (graph, held, _) in enumerate(graphs):
            for name, t in cases[(turn + k) % 3].items():
                if torch.is_tensor(t):
                    held[name].copy_(t)
            graph.replay()
        everything(cases[2])
        torch.cuda.synchronize()
        for k, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(p, q) for p, q in zip(out, want[(turn + k) % 3]))


def test_label_loss_captured_and_replayed():
    """Of more labels than one launch sums up."""
    cases = [chain_case(s, steps=2000, batch=16, n=24) for s in (0, 1)]
    for c in cases:
        c["labels"][::3] = -100

    def run(c):
        loss, dl_dz, grads, answer = training.label_loss(c["bits"], c["batch"], c["w"], c["decay"], c["labels"], state=c["state"], top=1)
        return [loss, dl_dz, *grads.values(), *answer]
    want = [[t.clone() for t in run(c)] for c in cases]
    mean = -(want[0][5].double().sum() / (cases[0]["labels"] != -100).sum()).cpu()
    close(want[0][0], mean, 20 * U * mean.abs())   # (sums of 1,024, of those and their share: at most 10 + 5 + 3 half steps each way)
    held = {name: t.clone() if torch.is_tensor(t) else t for name, t in cases[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(held)
    for turn in range(5):
        for name, t in cases[turn % 2].items():
            if torch.is_tensor(t):
                held[name].copy_(t)
        graph.replay()
        run(cases[0])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[turn % 2]))


def test_two_streams_at_once():
    cases = [chain_case(s) for s in (3, 4)]
    want = [everything(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(everything(cases[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for out in got[k]:
            assert all(torch.equal(p, q) for p, q in zip(out, want[k]))


def test_calls_in_native_code_and_in_python_are_the_same(monkeypatch):
    case = chain_case(6)
    native = everything(case)
    assert readout._native.gated_scan.__name__ == "gated_scan" and readout._native.gated_scan(None, None, None, None, False) is None
    monkeypatch.setattr(readout, "_native", type("Nothing", (), {name: staticmethod(lambda *_: None) for name in readout._Native.NAMES}))
    assert all(torch.equal(p, q) and p.dtype == q.dtype and p.shape == q.shape for p, q in zip(everything(case), native))


def test_label_loss_trains_a_network_down_to_its_spikes():
    """A run of a small network, its readout's loss, and the gradients of readout and synapses: the readout's against float64 autograd of the
    definition, the synapses' as what Glif3Bptt makes of that dl_dz."""
    n, batch, steps, classes = 96, 4, 120, 7
    cfg = synthetic.small_glif3_network(n=n, n_in=200, steps=steps, seed=3, in_w_scale=4.0)
    sim = Glif3Simulator(n, cfg["par"], 1.0, batch=batch, rec=cfg["rec_src"], inp=cfg["inp_src"], ring_slots=cfg["L"])
    in_ptr, in_events = ops.poisson_events(200, 60.0, 1.0, steps, batch=batch, seed=5)
    sim.set_input_events(in_ptr, in_events)
    fwd = sim.run(steps, save_state=True)
    z = sim.raster(fwd["bits"]).cpu().view(steps, n, batch).double()
    assert z.sum() > 100
    g = gen(8)
    weight = torch.randn(n, classes, generator=g).cuda()
    decay = (0.5 + 0.45 * torch.rand(classes, generator=g)).cuda()
    labels = torch.randint(0, classes, (steps, batch), generator=g)
    labels[torch.rand(steps, batch, generator=g) < 0.3] = -100
    loss, dl_dz, grads, answer = training.label_loss(fwd["bits"], batch, weight, decay, labels.cuda(), top=3)

    zd, wd, ad = z.clone().requires_grad_(), weight.cpu().double().requires_grad_(), decay.cpu().double().requires_grad_()
    h, hs = torch.zeros(batch, classes, dtype=torch.float64, requires_grad=True), []
    h0 = h
    for t in range(steps):
        h = ad * h + zd[t].t() @ wd
        hs.append(h)
    hs = torch.stack(hs)
    want = torch.nn.functional.cross_entropy(hs.view(-1, classes), labels.view(-1), ignore_index=-100)
    want.backward()
    # sums of some hundred terms of one sign or another, each a chain of some hundred roundings: a thousand half steps of the largest entry
    for got, ref in ((loss, want.detach()), (dl_dz.view(steps, n, batch), zd.grad), (grads["weight"], wd.grad), (grads["decay"], ad.grad), (grads["state"], h0.grad)):
        close(got, ref, 1000 * U * ref.abs().max().clamp(min=1e-6))
    assert torch.equal(answer.top_index[..., 0].cpu(), hs.argmax(2)) or (answer.top_index[..., 0].cpu() == hs.argmax(2)).double().mean() > 0.99
    bptt = training.Glif3Bptt(sim)
    bptt.backward(fwd, dl_dz=dl_dz)
    assert torch.isfinite(bptt.d_rec_w).all() and bptt.d_rec_w.abs().sum() > 0
    other = training.Glif3Bptt(sim)
    other.backward(fwd, dl_dz=zd.grad.reshape(steps, n * batch).float().cuda())
    scale = other.d_rec_w.abs().max().item()
    assert (bptt.d_rec_w - other.d_rec_w).abs().max().item() <= 1e-4 * scale   # (the same pass of a dl_dz that is 1e-5 off at most)
