"""short_conv and selective_scan against plain implementations in 64 bits, and their gradients against autograd of those and against differences.

Tolerances are bounds, made from the sums themselves: U = 2^-24 is half a step of fp32, a value rounded to type T is off by at most eps(T) / 2 of itself (and
half of the smallest subnormal), and a sum of k terms is off by at most k U times the sum of the terms' magnitudes."""
import math

import pytest
import torch

from bmtk_amd import readout
from test_gpu_readout import DTYPES, U, close, gen

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------------
# short convolution

def conv_case(steps, batch, dim, width, dtype, weights=None, silu=True, bias=True, state=True, ragged=False, seed=0):
    g = gen(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    weights = weights or dtype
    c = dict(x=normal(steps, batch, dim).to(dtype), weight=normal(dim, width).to(weights), bias=normal(dim).to(weights) if bias else None,
             state=normal(width - 1, batch, dim).to(dtype) if state else None, lengths=None, silu=silu, dy=normal(steps, batch, dim).to(dtype),
             d_last=normal(width - 1, batch, dim).to(dtype))
    if ragged:
        c["lengths"] = torch.randint(0, steps + 1, (batch,), generator=g, dtype=torch.int32)
    return c


def conv_reference(c):
    """The definition in 64 bits, step by step and sequence by sequence, its gradients by autograd, and bounds of what fp32 arithmetic is off by."""
    x, w = c["x"].double(), c["weight"].double()
    steps, batch, dim = x.shape
    width = w.shape[1]
    leaf = lambda t, shape: (torch.zeros(shape, dtype=torch.float64) if t is None else t.double()).clone().requires_grad_()  # noqa: E731
    x, w, bias, state = leaf(x, None), leaf(w, None), leaf(c["bias"], (dim,)), leaf(c["state"], (width - 1, batch, dim))
    ends = [steps] * batch if c["lengths"] is None else [min(max(n, 0), steps) for n in c["lengths"].tolist()]
    y, z_mag = torch.zeros(steps, batch, dim, dtype=torch.float64), torch.zeros(steps, batch, dim, dtype=torch.float64)
    zs = torch.zeros(steps, batch, dim, dtype=torch.float64)
    columns, last = [], []
    for b, end in enumerate(ends):
        given = torch.cat([state[:, b], x[:end, b]])
        last.append(given[end:])
        rows = []
        for t in range(end):
            window = given[t:t + width]
            z = bias + (window * w.t()).sum(0)
            z_mag[t, b] = (bias.abs() + (window * w.t()).abs().sum(0)).detach()
            zs[t, b] = z.detach()
            rows.append(z * torch.sigmoid(z) if c["silu"] else z)
        rows += [torch.zeros(dim, dtype=torch.float64)] * (steps - end)
        columns.append(torch.stack(rows) if rows else torch.zeros(0, dim, dtype=torch.float64))
    y, last = torch.stack(columns, 1), torch.stack(last, 1)
    grads = torch.autograd.grad((y * c["dy"].double()).sum() + (last * c["d_last"].double()).sum(), (x, w, bias, state), allow_unused=True)
    grads = [torch.zeros_like(v) if d is None else d for v, d in zip((x, w, bias, state), grads)]
    # z: width fmas.  silu'(z) is at most 1.1, silu'' at most 0.5; the sigmoid itself is off by 4 roundings and by what its exponent is, up to |z| U
    e_z = (width + 1) * U * z_mag
    p = torch.sigmoid(zs)
    e_y = 1.1 * e_z + (zs * p).abs() * (6 + 2 * zs.abs()) * U if c["silu"] else e_z
    dy = c["dy"].double().abs()
    dz_mag = 1.1 * dy if c["silu"] else dy
    e_dz = dy * (0.5 * e_z + (p + (zs * p * (1 - p)).abs()) * (10 + 3 * zs.abs()) * U) if c["silu"] else torch.zeros_like(dy)
    inside = torch.zeros(steps, batch, 1, dtype=torch.float64)
    for b, end in enumerate(ends):
        inside[:end, b] = 1
    e_dz, dz_mag = e_dz * inside, dz_mag * inside
    wa = w.detach().abs()
    e_dx = torch.zeros(steps + width - 1, batch, dim, dtype=torch.float64)
    e_dw, e_db = torch.zeros(dim, width, dtype=torch.float64), torch.zeros(dim, dtype=torch.float64)
    long = torch.cat([state, x]).detach().abs()
    # sums over a stretch of up to 64 steps, then over stretches and sequences, a sixteenth of them in each of sixteen wavefronts
    k = 64 + 16 + math.ceil(math.ceil(steps / 8) * batch / 16)
    for j in range(width):
        e_dx[j:j + steps] += wa[:, j] * (e_dz + (width + 2) * U * dz_mag)
        e_dw[:, j] = (long[j:j + steps] * (e_dz + k * U * dz_mag)).sum((0, 1))
    e_db = (e_dz + k * U * dz_mag).sum((0, 1))
    for b, end in enumerate(ends):
        e_dx[end:end + width - 1, b] += U * c["d_last"][:, b].double().abs()
    return dict(y=(y.detach(), e_y * inside), last=(last.detach(), 0.0), dx=(grads[0], e_dx[width - 1:]), d_weight=(grads[1], e_dw), d_bias=(grads[2], e_db),
                d_state=(grads[3], e_dx[:width - 1]))


def conv_run(c):
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    y, last = readout.short_conv(d["x"], d["weight"], d["bias"], d["state"], d["lengths"], silu=c["silu"])
    dx, dw, db, ds = readout.short_conv_bwd(d["x"], d["weight"], d["dy"], d["bias"], d["state"], d["d_last"], d["lengths"], silu=c["silu"])
    return dict(y=y, last=last, dx=dx, d_weight=dw, d_bias=db, d_state=ds)


def conv_check(c):
    got, want = conv_run(c), conv_reference(c)
    for name in want:
        close(got[name], *want[name], name)
    again = conv_run(c)
    assert all(torch.equal(got[k], again[k]) for k in got)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps,batch,dim,width,silu,ragged", [
    (1, 1, 1, 2, True, False), (1, 5, 64, 4, True, False), (2, 3, 7, 4, False, True), (3, 2, 8, 8, True, False), (9, 4, 17, 3, True, True), (40, 3, 33, 4, True, True),
    (130, 2, 9, 5, False, True), (70, 2, 64, 8, True, True), (300, 1, 20, 2, True, False), (33, 7, 12, 6, True, True), (17, 1, 3, 7, False, False), (5, 2, 4, 4, True, True),
    (65, 40, 11, 4, True, True)])
def test_conv_against_64_bits(steps, batch, dim, width, silu, ragged, dtype):
    conv_check(conv_case(steps, batch, dim, width, dtype, None if width % 2 else torch.float32, silu, ragged=ragged))


@pytest.mark.parametrize("bias,state", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("dim", [5, 24])
def test_conv_without_bias_or_state(dim, bias, state):
    conv_check(conv_case(11, 3, dim, 4, torch.bfloat16, bias=bias, state=state, ragged=True))


@pytest.mark.parametrize("dtype", DTYPES)
def test_conv_of_views_and_of_what_begins_anywhere(dtype):
    c = conv_case(21, 3, 30, 4, dtype, ragged=True)
    want = conv_run(c)
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    wide = torch.full((3, 21, 71), math.nan, dtype=dtype, device="cuda")
    x, dy = wide[:, :, 1:31].transpose(0, 1), wide[:, :, 33:63].transpose(0, 1)
    x.copy_(d["x"])
    dy.copy_(d["dy"])
    odd = torch.empty(30 * 4 + 1, dtype=dtype, device="cuda")[1:].view(30, 4)
    odd.copy_(d["weight"])
    y, last = readout.short_conv(x, odd, d["bias"], d["state"], d["lengths"], silu=True)
    got = (y, last) + readout.short_conv_bwd(x, odd, dy, d["bias"], d["state"], d["d_last"], d["lengths"], silu=True)
    for g, name in zip(got, ("y", "last", "dx", "d_weight", "d_bias", "d_state")):
        assert torch.equal(g, want[name]), name


@pytest.mark.parametrize("dim,width", [(24, 4), (3, 3)])
def test_conv_goes_on_from_its_last_inputs(dim, width):
    """Steps in one call and one after the other give the same bits; what lies behind a sequence's end changes nothing, whatever it is."""
    c = conv_case(12, 4, dim, width, torch.bfloat16, torch.float32)
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    y, last = readout.short_conv(d["x"], d["weight"], d["bias"], d["state"], silu=True)
    state, rows = d["state"], []
    for t in range(12):
        r, state = readout.short_conv(d["x"][t:t + 1], d["weight"], d["bias"], state, silu=True)
        rows.append(r)
    assert torch.equal(torch.cat(rows), y) and torch.equal(state, last)
    lengths = torch.tensor([12, 0, 5, 1], dtype=torch.int32, device="cuda")
    outs = []
    for filler in (0.0, math.nan, math.inf):
        x, dy = d["x"].clone(), d["dy"].clone()
        for b, n in enumerate(lengths.tolist()):
            x[n:, b], dy[n:, b] = filler, filler
        outs.append(readout.short_conv(x, d["weight"], d["bias"], d["state"], lengths, silu=True)
                    + readout.short_conv_bwd(x, d["weight"], dy, d["bias"], d["state"], d["d_last"], lengths, silu=True))
    assert all(torch.equal(p, q) for o in outs[1:] for p, q in zip(o, outs[0]))
    assert not outs[0][0][5:, 2].any() and not outs[0][2][5:, 2].any() and torch.equal(outs[0][1][:, 1], d["state"][:, 1])
    far = torch.tensor([2 ** 31 - 1, -5, 5, 1], dtype=torch.int32, device="cuda")
    assert all(torch.equal(p, q) for p, q in zip(readout.short_conv(d["x"], d["weight"], d["bias"], d["state"], far, silu=True),
                                                 readout.short_conv(d["x"], d["weight"], d["bias"], d["state"], lengths, silu=True)))


def test_conv_of_no_steps():
    c = conv_case(4, 2, 5, 3, torch.float32)
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    y, last = readout.short_conv(d["x"][:0], d["weight"], d["bias"], d["state"])
    assert y.shape == (0, 2, 5) and torch.equal(last, d["state"]) and not readout.short_conv(d["x"][:0], d["weight"])[1].any()
    dx, dw, db, ds = readout.short_conv_bwd(d["x"][:0], d["weight"], d["dy"][:0], d["bias"], d["state"], d["d_last"])
    assert dx.shape == (0, 2, 5) and not dw.any() and not db.any() and torch.equal(ds, d["d_last"])


def test_conv_of_far_values():
    """silu of numbers whose exponential is 0 or infinite, and of infinities: z sigmoid(z) as it is, -inf gives NaN there."""
    z = torch.tensor([-3e38, -200.0, -100.0, -87.0, 0.0, 50.0, 200.0, 3e38, math.inf]).cuda().view(1, 1, -1)
    w = torch.tensor([0.0, 1.0]).repeat(9, 1).cuda()
    y, _ = readout.short_conv(z, w, silu=True)
    zd = z.double()
    want = zd * torch.sigmoid(zd)
    # below -87 the result is under the smallest normal number, and 0 is as near as need be
    assert torch.allclose(y.double(), want, rtol=2e-5, atol=1.2e-38 * 100)


# ---------------------------------------------------------------------------------------------------------------------
# selective scan

def selective_case(steps, batch, dim, states, groups, dtype, gates=None, softplus=True, skip=True, bias=True, state=True, ragged=False, seed=0):
    g = gen(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    c = dict(x=normal(steps, batch, dim).to(dtype), dt=(normal(steps, batch, dim) if softplus else 0.3 * torch.rand(steps, batch, dim, generator=g)).to(gates or dtype),
             rate=-torch.rand(dim, states, generator=g) * 3 - 0.05, write=normal(steps, batch, groups, states).to(dtype), read=normal(steps, batch, groups, states).to(dtype),
             skip=normal(dim) if skip else None, dt_bias=(normal(dim) - 1 if softplus else 0.1 * torch.rand(dim, generator=g)) if bias else None, softplus=softplus,
             state=normal(batch, dim, states) if state else None, lengths=None, dy=normal(steps, batch, dim).to(dtype), d_last=normal(batch, dim, states))
    if ragged:
        c["lengths"] = torch.randint(0, steps + 1, (batch,), generator=g, dtype=torch.int32)
    return c


def selective_reference(c):
    """The definition in 64 bits, its gradients by autograd, and bounds of the errors of fp32 arithmetic.

    Bounds: a state is a sum of terms, each of which passed some decays.  A decay e^(delta rate) is off by its argument's error (delta's, 16 half steps of
    its softplus and its sum, and two more, of up to |delta rate|) and 2 half steps; a term that is older has passed more of them, and m |v| e^-v of its
    decay is at most m / e.  S: sum of the terms' magnitudes; G: the same, each times the roundings that it went through."""
    d64 = lambda k, shape=None: torch.zeros(shape, dtype=torch.float64) if c[k] is None else c[k].double()  # noqa: E731
    x, dt, rate, write, read = (d64(k).clone().requires_grad_() for k in ("x", "dt", "rate", "write", "read"))
    steps, batch, dim = x.shape
    groups, states = write.shape[2:]
    skip, bias, state = (d64(k, s).clone().requires_grad_() for k, s in (("skip", (dim,)), ("dt_bias", (dim,)), ("state", (batch, dim, states))))
    lengths = torch.full((batch,), steps) if c["lengths"] is None else c["lengths"].clamp(0, steps)
    wide = lambda v: v.repeat_interleave(dim // groups, dim=1)  # noqa: E731
    h, ys = state, []
    S, G = state.detach().abs(), torch.zeros_like(state.detach())
    e_y, keep = [], []
    for t in range(steps):
        there = (t < lengths).view(-1, 1)
        v = dt[t] + bias
        delta = torch.nn.functional.softplus(v, threshold=200) if c["softplus"] else v
        a = delta.unsqueeze(2) * rate
        u = (delta * x[t]).unsqueeze(2) * wide(write[t])
        new = torch.exp(a) * h + u
        h = torch.where(there.unsqueeze(2), new, h)
        ys.append(torch.where(there, (h * wide(read[t])).sum(2) + skip * x[t], 0.0))
        with torch.no_grad():
            e, k = torch.exp(a), 20 * a.abs() + 4   # roundings of a decay
            if not c["softplus"]:
                k = 20 * a.abs() + 4 + 4 * (dt[t].abs() + bias.abs()).unsqueeze(2) * rate.abs()
            S1, G1 = e * S + u.abs(), e * (G + k * S) + 20 * u.abs()
            S, G = torch.where(there.unsqueeze(2), S1, S), torch.where(there.unsqueeze(2), G1, G)
            # (stretches joined: the same decays again, once)
            e_y.append(torch.where(there, ((2 * G + (states + 8) * S) * wide(read[t]).abs()).sum(2) + 4 * (skip * x[t]).abs(), 0.0) * U)
            keep.append((e, k, S, G, u.abs(), delta, v, there))
    y = torch.stack(ys)
    e_last = (2 * G + 8 * S) * U
    leaves = (x, dt, rate, write, read, skip, bias, state)
    grads = torch.autograd.grad((y * c["dy"].double()).sum() + (h * c["d_last"].double()).sum(), leaves, allow_unused=True)
    grads = [torch.zeros_like(v) if d is None else d for v, d in zip(leaves, grads)]
    # back: R, H as S, G of g
    with torch.no_grad():
        R, H = c["d_last"].double().abs(), torch.zeros_like(S)
        out = {k: torch.zeros_like(v) for k, v in zip(("dx", "d_dt", "d_rate", "d_write", "d_read", "d_skip", "d_dt_bias"), leaves)}
        mag = {k: torch.zeros_like(out[k]) for k in ("d_rate", "d_skip", "d_dt_bias")}
        first = (state.detach().abs(), torch.zeros_like(S))
        for t in range(steps - 1, -1, -1):
            e, k, S1, G1, u, delta, v, there = keep[t]
            S0, G0 = (keep[t - 1][2], keep[t - 1][3]) if t else first
            dy = c["dy"][t].double().abs()
            w, r = wide(write[t]).abs(), wide(read[t]).abs()
            g, Gg = dy.unsqueeze(2) * r + R, 3 * dy.unsqueeze(2) * r + 2 * H + 2 * R
            in3 = there.unsqueeze(2)
            dx_abs, delta_abs = x[t].abs(), delta.abs()
            eh, Geh = e * S0, e * (2 * G0 + (k + 4) * S0)     # |e h[t-1]| and its roundings
            q, Gq = g * eh, g * Geh + Gg * eh
            s1, e_s1 = (g * w).sum(2), ((Gg + (states + 4) * g) * w).sum(2)
            s2, e_s2 = (q * rate.abs()).sum(2), ((Gq + (states + 4) * q) * rate.abs()).sum(2)
            slope = torch.sigmoid(v) if c["softplus"] else torch.ones_like(v)
            out["dx"][t] = torch.where(there, delta_abs * e_s1 + 24 * delta_abs * s1 + 4 * (skip.abs() * dy), 0.0) * U
            e_dt = torch.where(there, slope * (dx_abs * e_s1 + e_s2 + (24 + 2 * v.abs()) * (dx_abs * s1 + s2)), 0.0)
            m_dt = torch.where(there, slope * (dx_abs * s1 + s2), 0.0)
            out["d_dt"][t] = e_dt * U
            by_group = lambda p: torch.where(in3, p, 0.0).view(batch, groups, dim // groups, states).sum(2)  # noqa: E731
            n = 64 + math.ceil(dim / groups / 64) + 8
            h_now, G_now = S1, 2 * G1 + 8 * S1
            out["d_read"][t] = by_group(dy.unsqueeze(2) * (G_now + n * h_now)) * U
            out["d_write"][t] = by_group((delta_abs * dx_abs).unsqueeze(2) * (Gg + (n + 24) * g)) * U
            out["d_rate"] += torch.where(in3, Gq * delta_abs.unsqueeze(2) + 24 * q * delta_abs.unsqueeze(2), 0.0).sum(0) * U
            mag["d_rate"] += torch.where(in3, q * delta_abs.unsqueeze(2), 0.0).sum(0)
            mag["d_skip"] += torch.where(there, dy * dx_abs, 0.0).sum(0)
            out["d_dt_bias"] += e_dt.sum(0) * U
            mag["d_dt_bias"] += m_dt.sum(0)
            R, H = torch.where(in3, e * g, R), torch.where(in3, e * (Gg + (k + 2) * g), H)
        terms = min(steps * batch, 4000)
        for name in mag:
            out[name] += (terms + 40) * U * mag[name]
        out["d_state"] = (2 * H + 8 * R) * U
    names = ("dx", "d_dt", "d_rate", "d_write", "d_read", "d_skip", "d_dt_bias", "d_state")
    return dict(y=(y.detach(), torch.stack(e_y)), last=(h.detach(), e_last), **{k: (g, out[k]) for k, g in zip(names, grads)})


def selective_run(c):
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    given = tuple(d[k] for k in ("x", "dt", "rate", "write", "read"))
    more = dict(skip=d["skip"], dt_bias=d["dt_bias"], softplus=c["softplus"], lengths=d["lengths"])
    y, last, saved = readout.selective_scan(*given, state=d["state"], save_state=True, **more)
    r = readout.selective_scan_bwd(*given, saved, d["dy"], d_last=d["d_last"], **more)
    plain = readout.selective_scan(*given, state=d["state"], **more)
    assert torch.equal(plain[0], y) and torch.equal(plain[1], last)
    return dict(y=y, last=last, **r._asdict())


def selective_check(c):
    got, want = selective_run(c), selective_reference(c)
    for name in want:
        close(got[name], *want[name], name)
    again = selective_run(c)
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps,batch,dim,states,groups,softplus,ragged", [
    (1, 1, 1, 1, 1, True, False), (1, 3, 70, 16, 1, True, False), (2, 2, 5, 4, 1, False, True), (16, 2, 64, 16, 1, True, False), (17, 3, 65, 16, 1, True, True),
    (40, 2, 130, 5, 2, False, True), (63, 1, 24, 8, 4, True, False), (150, 2, 10, 16, 1, True, True), (333, 1, 66, 3, 1, True, False), (50, 3, 40, 32, 2, True, True),
    (37, 2, 12, 64, 1, False, True), (33, 1, 9, 20, 9, True, False), (20, 2, 8, 40, 1, True, True), (5, 2, 16, 12, 1, True, True), (3, 70, 6, 16, 1, True, True)])
def test_selective_against_64_bits(steps, batch, dim, states, groups, softplus, ragged, dtype):
    selective_check(selective_case(steps, batch, dim, states, groups, dtype, torch.float32 if states % 2 else None, softplus, ragged=ragged))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steps,batch,dim,states", [(1500, 1, 20, 16), (700, 2, 66, 4), (1031, 1, 64, 33)])
def test_selective_of_many_stretches(steps, batch, dim, states, dtype):
    selective_check(selective_case(steps, batch, dim, states, 1, dtype, ragged=True, seed=2))


@pytest.mark.parametrize("without", [("skip",), ("bias",), ("state",), ("skip", "bias", "state")])
def test_selective_without_some_inputs(without):
    selective_check(selective_case(23, 2, 20, 6, 1, torch.float32, **{k: False for k in without}))


@pytest.mark.parametrize("dtype", DTYPES)
def test_selective_of_views(dtype):
    c = selective_case(19, 3, 30, 4, 2, dtype, ragged=True)
    want = selective_run(c)
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    wide = torch.full((3, 19, 131), math.nan, dtype=dtype, device="cuda")
    at = {}
    for name, first, n in (("x", 1, 30), ("dt", 32, 30), ("dy", 65, 30), ("write", 97, 8), ("read", 107, 8)):
        at[name] = wide[:, :, first:first + n].transpose(0, 1)
        at[name].copy_(d[name].reshape(19, 3, n))
    write, read = (at[k].unflatten(2, (2, 4)) for k in ("write", "read"))
    more = dict(skip=d["skip"], dt_bias=d["dt_bias"], softplus=True, lengths=d["lengths"])
    y, last, saved = readout.selective_scan(at["x"], at["dt"], d["rate"], write, read, state=d["state"], save_state=True, **more)
    r = readout.selective_scan_bwd(at["x"], at["dt"], d["rate"], write, read, saved, at["dy"], d_last=d["d_last"], **more)
    for name, got in dict(y=y, last=last, **r._asdict()).items():
        assert torch.equal(got, want[name]), name


@pytest.mark.parametrize("states", [4, 16, 5])
def test_selective_goes_on_from_its_last_state(states):
    """Steps in one call and one after the other: within the bounds of both.  What lies behind a sequence's end changes nothing, whatever it is."""
    c = selective_case(40, 4, 20, states, 1, torch.bfloat16, torch.float32)
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    more = dict(skip=d["skip"], dt_bias=d["dt_bias"], softplus=True)
    state, rows = d["state"], []
    for t in range(40):
        r, state = readout.selective_scan(d["x"][t:t + 1], d["dt"][t:t + 1], d["rate"], d["write"][t:t + 1], d["read"][t:t + 1], state=state, **more)
        rows.append(r)
    want = selective_reference(c)
    close(torch.cat(rows), *want["y"], "y")
    close(state, *want["last"], "last")
    lengths = torch.tensor([40, 0, 17, 1], dtype=torch.int32, device="cuda")
    outs = []
    for filler in (0.0, math.nan, math.inf):
        at = {k: d[k].clone() for k in ("x", "dt", "write", "read", "dy")}
        for b, n in enumerate(lengths.tolist()):
            for v in at.values():
                v[n:, b] = filler
        y, last, saved = readout.selective_scan(at["x"], at["dt"], d["rate"], at["write"], at["read"], state=d["state"], lengths=lengths, save_state=True, **more)
        outs.append((y, last) + tuple(readout.selective_scan_bwd(at["x"], at["dt"], d["rate"], at["write"], at["read"], saved, at["dy"], d_last=d["d_last"], lengths=lengths,
                                                                 **more)))
    assert all(torch.equal(p, q) for o in outs[1:] for p, q in zip(o, outs[0]))
    assert torch.equal(outs[0][1][1], d["state"][1]) and not outs[0][0][17:, 2].any()
    assert all(not v[17:, 2].any() and not v[:, 1].any() for v in outs[0][2:4])


def test_selective_of_no_steps():
    c = selective_case(4, 2, 5, 3, 1, torch.float32)
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    given = [d[k][:0] if k != "rate" else d[k] for k in ("x", "dt", "rate", "write", "read")]
    y, last, saved = readout.selective_scan(*given, state=d["state"], save_state=True)
    assert y.shape == (0, 2, 5) and torch.equal(last, d["state"]) and saved.shape == (0, 2, 5, 3) and not readout.selective_scan(*given)[1].any()
    r = readout.selective_scan_bwd(*given, saved, d["dy"][:0], d_last=d["d_last"])
    assert torch.equal(r.d_state, d["d_last"]) and not any(v.any() for v in r[:7])
    assert not readout.selective_scan_bwd(*given, saved, d["dy"][:0]).d_state.any()


@pytest.mark.parametrize("steps", [16, 700])
def test_selective_of_infinite_states(steps):
    """An infinite state stays infinite, behind decays that fp32 does not hold too, and stays in its own channel."""
    c = selective_case(steps, 1, 70, 4, 1, torch.float32, softplus=False)
    c["dt"] = c["dt"] + 0.2
    c["state"][0, 3, 1] = math.inf
    got = selective_run(dict(c, dy=torch.ones_like(c["dy"])))
    assert got["last"][0, 3, 1] == math.inf
    c["state"][0, 3, 1] = 0.0
    want = selective_run(dict(c, dy=torch.ones_like(c["dy"])))
    others = torch.arange(70) != 3
    assert torch.equal(got["y"][:, :, others], want["y"][:, :, others]) and torch.equal(got["last"][:, others], want["last"][:, others])
    assert torch.equal(got["dx"][:, :, others], want["dx"][:, :, others])


def test_selective_by_differences():
    """The gradient against differences of the definition's own loss in 64 bits, in the direction of the gradient's and of random numbers."""
    c = selective_case(21, 2, 6, 3, 2, torch.float32, ragged=True, seed=5)
    got = selective_run(c)
    names = dict(x="dx", dt="d_dt", rate="d_rate", write="d_write", read="d_read", skip="d_skip", dt_bias="d_dt_bias", state="d_state")

    def loss(at):
        lengths = at["lengths"]
        h, total = at["state"], 0.0
        wide = lambda v: v.repeat_interleave(3, dim=1)  # noqa: E731
        for t in range(21):
            there = (t < lengths).view(-1, 1)
            delta = torch.log1p(torch.exp(at["dt"][t] + at["dt_bias"]))
            new = torch.exp(delta.unsqueeze(2) * at["rate"]) * h + (delta * at["x"][t]).unsqueeze(2) * wide(at["write"][t])
            h = torch.where(there.unsqueeze(2), new, h)
            total = total + torch.where(there, ((h * wide(at["read"][t])).sum(2) + at["skip"] * at["x"][t]) * at["dy"][t], 0.0).sum()
        return total + (h * at["d_last"]).sum()
    at = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in c.items()}
    for name, grad in names.items():
        v = torch.randn(at[name].shape, generator=gen(7), dtype=torch.float64)
        step = 1e-5
        diff = (loss(dict(at, **{name: at[name] + step * v})) - loss(dict(at, **{name: at[name] - step * v}))) / (2 * step)
        along = (got[grad].double().cpu() * v).sum()
        size = (got[grad].double().cpu() * v).abs().sum()
        # differences of second order: 1e-10 times a third derivative, and 1e-16 / 1e-5 of the loss; fp32 gradients: 100 roundings of the terms
        assert (along - diff).abs() <= 100 * 2 * U * size + 1e-6 * (1 + size), name
