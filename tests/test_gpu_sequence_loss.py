"""short_conv, selective_scan and projected_logprobs together: the loss of a trained readout with a memory, all gradients down to the spikes, and the answers step by step;
captured and replayed, on two streams, and by native calls and Python's alike."""
import math

import pytest
import torch

from bmtk_amd import readout, training
from test_gpu_readout import U, gen, pack

pytestmark = pytest.mark.gpu


def case(steps, batch, n, channels, states, groups, vocab, dtype, width=4, seed=0):
    g = gen(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    mixed = channels + 2 * groups * states
    labels = torch.randint(0, vocab, (steps, batch), generator=g)
    return dict(z=torch.rand(steps, n * batch, generator=g) < 0.1, batch=batch, groups=groups, weight=(normal(n, mixed + channels) / math.sqrt(0.1 * n)).to(dtype),
                conv_weight=(normal(mixed, width) / math.sqrt(width)).to(dtype), conv_bias=(0.1 * normal(mixed)).to(dtype), rate=-(0.5 + 2.0 * torch.rand(channels, states, generator=g)),
                skip=normal(channels), dt_bias=0.3 * normal(channels) - 1.0, out_weight=(2.0 / math.sqrt(channels) * normal(vocab, channels)).to(dtype),
                labels=torch.where(torch.rand(steps, batch, generator=g) < 0.2, -100, labels),
                memory=(normal(width - 1, batch, mixed).to(dtype), normal(batch, channels, states)))


PARAMETERS = ("weight", "conv_weight", "conv_bias", "rate", "out_weight", "skip", "dt_bias")


def on_device(c):
    d = {k: tuple(t.cuda() for t in v) if isinstance(v, tuple) else v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    d["bits"] = pack(c["z"])
    return d


def run(d):
    return training.sequence_loss(d["bits"], d["batch"], d["weight"], d["conv_weight"], d["rate"], d["out_weight"], d["labels"], conv_bias=d["conv_bias"], skip=d["skip"],
                                  dt_bias=d["dt_bias"], groups=d["groups"], memory=d["memory"])


class Rounded(torch.autograd.Function):
    """A stage's result and its gradient, in the type between the stages."""
    @staticmethod
    def forward(ctx, t, dtype):
        ctx.dtype = dtype
        return t.to(dtype).double()

    @staticmethod
    def backward(ctx, d):
        return d.to(ctx.dtype).double(), None


def reference(c):
    """The definition in 64 bits, rounded to the type between the stages where that is bf16, and its gradients by autograd."""
    dtype = torch.bfloat16 if c["weight"].dtype == torch.bfloat16 else torch.float64
    between = lambda t: Rounded.apply(t, dtype)  # noqa: E731
    p = {k: c[k].double().clone().requires_grad_() for k in PARAMETERS}
    conv_state, state = (t.double().clone().requires_grad_() for t in c["memory"])
    steps, batch, groups = len(c["z"]), c["batch"], c["groups"]
    channels, states = p["rate"].shape
    mixed = channels + 2 * groups * states
    n = p["weight"].shape[0]
    z = c["z"].double().view(steps, n, batch).clone().requires_grad_()
    y = between((z.transpose(1, 2).reshape(steps * batch, n) @ p["weight"]).view(steps, batch, -1))
    given, width = torch.cat([conv_state, y[:, :, :mixed]]), p["conv_weight"].shape[1]
    m = p["conv_bias"] + sum(p["conv_weight"][:, j] * given[j:j + steps] for j in range(width))
    m = between(m * torch.sigmoid(m))
    x, write, read = m.split((channels, groups * states, groups * states), 2)
    write, read = (t.unflatten(2, (groups, states)).repeat_interleave(channels // groups, 2) for t in (write, read))
    delta = torch.nn.functional.softplus(y[:, :, mixed:] + p["dt_bias"], threshold=1e9)
    h, rows = state, []
    for t in range(steps):
        h = torch.exp(delta[t].unsqueeze(2) * p["rate"]) * h + (delta[t] * x[t]).unsqueeze(2) * write[t]
        rows.append((h * read[t]).sum(2) + p["skip"] * x[t])
    out = between(torch.stack(rows)) if rows else torch.zeros(0, batch, channels, dtype=torch.float64)
    logp = torch.log_softmax(out @ p["out_weight"].t(), 2)
    there = c["labels"] != -100
    logp = torch.where(there, logp.gather(2, c["labels"].clamp(min=0).unsqueeze(2)).squeeze(2), 0.0)
    loss = -logp.sum() / max(1, int(there.sum()))
    leaves = dict(p, conv_state=conv_state, state=state, z=z)
    grads = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))
    return loss.detach(), logp.detach(), grads, (given[steps:].detach(), h.detach())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("steps,batch,n,channels,states,groups,vocab", [(1, 1, 40, 8, 4, 1, 10), (6, 3, 50, 12, 5, 2, 9), (40, 4, 70, 24, 16, 1, 33), (90, 2, 30, 66, 3, 3, 300)])
def test_loss_and_gradients_against_64_bits(steps, batch, n, channels, states, groups, vocab, dtype):
    c = case(steps, batch, n, channels, states, groups, vocab, dtype)
    loss, dl_dz, grads, answer, memory = run(on_device(c))
    want_loss, want_logp, want, want_memory = reference(c)
    # Everything is of order one.  fp32 (and fp16, whose call is in fp32): as many roundings as the longest sums one behind the other have terms, twice: forward and back;
    # terms are up to some four times the largest result.  bf16: the stages' results are rounded as the reference's are, but where they lie next to the middle of two numbers, to the
    # other one, a step; p and what is rounded of it, and gradients in bf16, half a step each: eight half steps of the largest entry.
    single = 4 * 2 * (steps + batch + n + channels * states + vocab) * U
    tolerance = single + (8 * torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 0.0)
    assert (loss.double().cpu() - want_loss).abs() <= tolerance * (1 + want_loss)
    assert (answer.logp.double().cpu() - want_logp).abs().max() <= tolerance * (1 + want_logp.abs().max())
    for got, wanted in zip(memory, want_memory):
        assert (got.double().cpu() - wanted).abs().max() <= tolerance * (1 + wanted.abs().max())
    got = dict(grads, z=dl_dz.view(steps, n, batch))
    assert set(got) == set(want)
    for name, g in got.items():
        last = torch.finfo(torch.float16).eps / 2 if g.dtype == torch.float16 else 0.0
        off = (g.double().cpu() - want[name]).abs().max()
        size = want[name].abs().max()
        assert off <= (tolerance + last) * size + (2.0 ** -25 if last else 0.0), (name, float(off), float(size))
    assert all(grads[k].dtype == c[k].dtype and grads[k].shape == c[k].shape for k in PARAMETERS)
    assert dl_dz.dtype == torch.float32 and dl_dz.shape == (steps, n * batch)


def test_goes_on_from_its_memory():
    """Steps in two calls, and the answers of the second one step at a time from the first one's memory."""
    c = case(30, 3, 40, 16, 8, 1, 20, torch.float32)
    c["labels"].clamp_(min=0)
    d = on_device(c)
    whole = run(d)
    first = run(dict(d, bits=d["bits"][:17], labels=d["labels"][:17]))
    second = run(dict(d, bits=d["bits"][17:], labels=d["labels"][17:], memory=first[4]))
    tolerance = 4 * 2 * (30 + 3 + 40 + 16 * 8 + 20) * U
    joined = torch.cat([first[3].logp, second[3].logp])
    assert (joined - whole[3].logp).abs().max() <= tolerance * (1 + whole[3].logp.abs().max())
    conv_state, state = first[4]
    for t in range(17, 30):
        y = readout.spike_readout(d["bits"][t:t + 1], d["weight"], 3)
        m, conv_state = readout.short_conv(y[:, :, :32], d["conv_weight"], d["conv_bias"], conv_state, silu=True)
        h, state = readout.selective_scan(m[:, :, :16], y[:, :, 32:], d["rate"], m[:, :, 16:24].unflatten(2, (1, 8)), m[:, :, 24:].unflatten(2, (1, 8)), d["skip"], d["dt_bias"],
                                          softplus=True, state=state)
        logp = readout.projected_logprobs(h, d["out_weight"], d["labels"][t:t + 1]).logp
        assert (logp[0] - joined[t]).abs().max() <= tolerance * (1 + joined.abs().max())
    for got, wanted in zip((conv_state, state), whole[4]):
        assert (got - wanted).abs().max() <= tolerance * (1 + wanted.abs().max())


def test_no_steps_and_no_labels():
    d = on_device(case(5, 2, 40, 16, 8, 1, 20, torch.bfloat16))
    loss, dl_dz, grads, answer, memory = run(dict(d, bits=d["bits"][:0], labels=d["labels"][:0]))
    assert loss == 0 and dl_dz.shape == (0, 80) and answer.logp.shape == (0, 2) and not any(g.any() for g in grads.values())
    assert all(torch.equal(p, q) for p, q in zip(memory, d["memory"]))
    loss, dl_dz, grads, answer, memory = run(dict(d, labels=torch.full_like(d["labels"], -100)))
    assert loss == 0 and not dl_dz.any() and not any(g.any() for g in grads.values()) and not answer.logp.any() and answer.lse.isfinite().all()


def tensors(r):
    loss, dl_dz, grads, answer, memory = r
    return [loss, dl_dz, *grads.values(), *answer, *memory]


def copy(d, to):
    for name, t in d.items():
        for p, q in zip(to[name] if isinstance(t, tuple) else (to[name],), t if isinstance(t, tuple) else (t,)):
            if torch.is_tensor(p):
                p.copy_(q)


def clones(d):
    return {k: tuple(t.clone() for t in v) if isinstance(v, tuple) else v.clone() if torch.is_tensor(v) else v for k, v in d.items()}


SIZES = [(50, 8, 60, 32, 16, 1, 40), (300, 2, 100, 64, 8, 2, 700), (4, 3, 60, 32, 16, 1, 40)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", SIZES)
def test_captured_and_replayed(sizes, dtype):
    """Two graphs, replayed in turn on other inputs, eager work and synchronizations in between."""
    cases = [on_device(case(*sizes, dtype, seed=s)) for s in range(3)]
    want = [[t.clone() for t in tensors(run(d))] for d in cases]
    graphs = []
    for k in (0, 1):
        held = clones(cases[k])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = tensors(run(held))
        graphs.append((graph, held, out))
    for turn in range(5):
        for k, (graph, held, _) in enumerate(graphs):
            copy(cases[(turn + k) % 3], held)
            graph.replay()
        run(cases[2])
        torch.cuda.synchronize()
        for k, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(p, q) for p, q in zip(out, want[(turn + k) % 3])), (turn, k)


def test_two_streams_at_once():
    cases = [on_device(case(*SIZES[1], torch.bfloat16, seed=s)) for s in (3, 4)]
    want = [[t.clone() for t in tensors(run(d))] for d in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(tensors(run(cases[k])))
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(p, q) for r in got[k] for p, q in zip(r, want[k]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_python_calls_and_native_ones(monkeypatch, dtype):
    """The same bits from both, with and without what is optional."""
    d = on_device(case(*SIZES[1], dtype, seed=5))
    lengths = torch.tensor([300, 123], dtype=torch.int32, device="cuda")
    g = gen(1)
    x, dt, dy = (torch.randn(300, 2, 64, generator=g).to(dtype).cuda() for _ in range(3))
    write, read = (torch.randn(300, 2, 2, 8, generator=g).to(dtype).cuda() for _ in range(2))
    w, bias = torch.randn(64, 3, generator=g).to(dtype).cuda(), torch.randn(64, generator=g).to(dtype).cuda()
    state, last = torch.randn(2, 2, 64, generator=g).to(dtype).cuda(), torch.randn(2, 64, 8, generator=g).cuda()
    tokens, scale = torch.randint(-1, 700, (300,), generator=g).cuda(), torch.randn(300, generator=g).cuda()

    def everything():
        out = tensors(run(d))
        for some in (True, False):
            of = lambda t: t if some else None  # noqa: E731, B023
            out += readout.short_conv(x, w, of(bias), of(state), of(lengths), silu=some)
            out += readout.short_conv_bwd(x, w, dy, of(bias), of(state), of(state), of(lengths), silu=some)
            for n in (300, 5):
                given = x[:n], dt[:n], d["rate"], write[:n], read[:n]
                more = dict(skip=of(d["skip"]), dt_bias=of(d["dt_bias"]), softplus=some, lengths=of(lengths))
                scan = readout.selective_scan(*given, state=of(last), save_state=True, **more)
                out += [*scan, *readout.selective_scan(*given, state=of(last), **more), *readout.selective_scan_bwd(*given, scan[2], dy[:n], d_last=of(last), **more)]
        for n in (300, 9):
            r = readout.projected_logprobs(x[:n, 0], d["out_weight"].to(dtype), tokens[:n], ignore=-1)
            out += [*r, *readout.projected_logprobs_bwd(x[:n, 0], d["out_weight"].to(dtype), tokens[:n], r, scale[:n], ignore=-1)]
        return out
    torch.cuda.init()
    readout._native.first()
    native = readout._native
    assert native.projected_logprobs is not None and native.projected_logprobs(x[:, 0], d["out_weight"].to(dtype), tokens, -1) is not None
    assert native.short_conv(x, w, None, None, None, False) is not None and native.selective_scan(x, dt, d["rate"], write, read, None, None, True, None, None, False) is not None
    want = [t.clone() for t in everything()]
    for name in readout._Native.NAMES:
        monkeypatch.setattr(native, name, lambda *_: None)
    # (step sizes without softplus are of either sign here, and some of 300 steps' states pass what 32 bits hold: NaN is the same as NaN)
    for k, (p, q) in enumerate(zip(everything(), want)):
        assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p[~p.isnan()], q[~q.isnan()]), k


def test_trains():
    """Gradients that autograd's optimizer takes, for some steps: it runs and stays finite."""
    d = on_device(case(60, 4, 50, 32, 8, 1, 25, torch.float32))
    parameters = [d[k].requires_grad_() for k in PARAMETERS]
    optimizer = torch.optim.Adam(parameters, lr=1e-2)
    for _ in range(5):
        with torch.no_grad():
            loss, dl_dz, grads, _, _ = run(d)
        for name, p in zip(PARAMETERS, parameters):
            p.grad = grads[name]
        optimizer.step()
        assert math.isfinite(loss) and dl_dz.isfinite().all() and all(p.isfinite().all() for p in parameters)
