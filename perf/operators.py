"""What is measured of the operators that train and use a readout of a spiking network: the work, through the calls that a program makes.

spikes    ``readout.spike_readout`` / ``spike_readout_bwd``: y[t, b] = sum of the weight rows of the neurons that fired in step t of trial b,
          from the spike bits of a run; its gradients by the weights and by every spike (what ``Glif3Bptt.backward`` takes as ``dl_dz``)
scan      ``readout.gated_scan`` / ``gated_scan_bwd``: h[t] = decay[t] * h[t - 1] + x[t], the leaky or gated memory behind such a
          readout, over the steps of many sequences, from a given state to a new one
logprobs  ``readout.token_logprobs`` / ``token_logprobs_bwd``: log probability of each row's token, the row's entropy, its most
          probable alternatives, and the gradient by the logits

Inputs are made on the GPU from the seed alone.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
IGNORED = -100   # the token of a row without one: padding


def listed():
    return [
        # one step of the V1 model's neurons, read out while it runs: latency
        dict(name="spikes_step_v1", kind="spikes", steps=1, n=230924, batch=1, dim=64, dtype="float32", rate=3.0, train=False),
        # a stretch of the V1 model into a wide readout with weights in 16 bits
        dict(name="spikes_v1", kind="spikes", steps=1000, n=230924, batch=1, dim=256, dtype="bfloat16", rate=3.0, train=False),
        # a training step of a small network, a batch that is no power of two and trials that straddle words
        dict(name="spikes_train_3k", kind="spikes", steps=100, n=3001, batch=12, dim=17, dtype="float32", rate=5.0, train=True),
        # a training step at the size of the V1 model's core: 600 steps, 32 trials
        dict(name="spikes_train_52k", kind="spikes", steps=600, n=51978, batch=32, dim=64, dtype="float32", rate=3.0, train=True),
        # one step of a readout's memory while the network runs: latency
        dict(name="scan_step", kind="scan", steps=1, batch=32, dim=1024, groups=1024, dtype="bfloat16", gates="float32", ragged=False, train=False),
        # leaky integrators over 600 steps of 32 trials, one time constant per channel, all learned
        dict(name="scan_leaky_train", kind="scan", steps=600, batch=32, dim=64, groups=0, dtype="float32", gates="float32", ragged=False, train=True),
        # one long recording: the time axis is all there is to spread over the chip
        dict(name="scan_long", kind="scan", steps=65536, batch=1, dim=1000, groups=1000, dtype="bfloat16", gates="bfloat16", ragged=False, train=False),
        # training a gated layer, a gate for each 64 channels, sequences of different lengths
        dict(name="scan_heads_train", kind="scan", steps=4096, batch=8, dim=2048, groups=32, dtype="bfloat16", gates="float32", ragged=True, train=True),
        # the answer of a few sequences with their alternatives: few rows, a long vocabulary
        dict(name="logprobs_answer", kind="logprobs", rows=4, vocab=131072, dtype="bfloat16", top=20, masked=0.1, ignored=0.0, train=False),
        # the label of each step and trial of a training step: many rows of ten classes
        dict(name="logprobs_classes_train", kind="logprobs", rows=19200, vocab=10, dtype="float32", top=2, masked=0.0, ignored=0.2, train=True),
        # training on tokens, an odd vocabulary, so that rows begin on any address
        dict(name="logprobs_tokens_train", kind="logprobs", rows=4096, vocab=50021, dtype="bfloat16", top=0, masked=0.0, ignored=0.1, train=True),
        # scoring given text
        dict(name="logprobs_score", kind="logprobs", rows=8192, vocab=131072, dtype="bfloat16", top=5, masked=0.0, ignored=0.05, train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("spikes", "scan", "logprobs"))
    train = rng.random() < 0.5
    dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
    if kind == "spikes":
        batch = rng.choice((1, 1, 4, 10, 12, 16, 20, 32, 32, 45, 64, 100))
        n = max(10, _log(rng, 450, 250000) // (1 if batch == 1 else 4))
        steps = _log(rng, 1, 1000)
        while steps * n * batch > 900_000_000:
            steps //= 2
        dim = _log(rng, 2, 300)
        while steps * n * batch * dim > 50_000_000_000:
            dim = max(2, dim // 2)
        return dict(kind=kind, steps=max(1, steps), n=n, batch=batch, dim=dim, dtype=dtype, rate=round(math.exp(rng.uniform(math.log(0.3), math.log(20.0))), 2),
                    train=train)
    if kind == "scan":
        steps, batch, dim = _log(rng, 1, 65536), _log(rng, 1, 64), _log(rng, 3, 4096)
        shared = rng.choice((0, 1, 1, 1, 2, 8, 33, 64, 128))   # channels of a gate; 0: one decay a channel for all steps
        if shared > 1:
            dim = max(1, dim // shared) * shared
        while steps * batch * dim > 60_000_000:
            steps, batch = max(1, steps // 2), max(1, batch // 2)
        return dict(kind=kind, steps=steps, batch=batch, dim=dim, groups=dim // shared if shared else 0, dtype=dtype,
                    gates="float32" if shared == 0 or rng.random() < 0.5 else dtype, ragged=rng.random() < 0.4, train=train)
    rows, vocab = _log(rng, 1, 20000), _log(rng, 2, 200000)
    while rows * vocab > (200_000_000 if train else 1_000_000_000):
        rows = max(1, rows // 2)
    return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, top=min(vocab, rng.choice((0, 1, 2, 5, 10, 20, 50))), masked=rng.choice((0.0, 0.0, 0.1, 0.5)),
                ignored=rng.choice((0.0, 0.1, 0.3)), train=train)


# ---------------------------------------------------------------------------------------------------------------------
# inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_spikes(case, seed):
    g = _generator(seed)
    steps, n, batch, dim, dtype = case["steps"], case["n"], case["batch"], case["dim"], DTYPES[case["dtype"]]
    ne = n * batch
    words = (ne + 63) // 64
    bits = torch.zeros(steps, words + 1, dtype=torch.int64, device="cuda")   # as Glif3Simulator.run returns them: one word of padding
    # independent spikes of a few Hz at steps of 1 ms, made from their number and places (a place drawn twice is one spike)
    per_row = max(1, int(round(ne * case["rate"] * 1e-3)))
    rows = max(1, 16_000_000 // per_row)
    for t in range(0, steps, rows):
        k = min(rows, steps - t)
        at = (torch.randint(0, ne, (k, per_row), device="cuda", generator=g)
              + torch.arange(k, device="cuda").view(-1, 1) * (words * 64)).view(-1).sort().values
        at = at[torch.cat([at.new_ones(1, dtype=torch.bool), at[1:] != at[:-1]])]
        bits[t:t + k, :words] = torch.zeros(k * words, dtype=torch.int64, device="cuda").index_add_(
            0, at >> 6, torch.ones_like(at) << (at & 63)).view(k, words)
    s = dict(bits=bits, batch=batch, weight=(torch.randn(n, dim, device="cuda", generator=g) / math.sqrt(dim)).to(dtype))
    if case["train"]:
        s["dy"] = (0.01 * torch.randn(steps, batch, dim, device="cuda", generator=g)).to(dtype)
    return s


def _prepare_scan(case, seed):
    g = _generator(seed)
    steps, batch, dim, groups = case["steps"], case["batch"], case["dim"], case["groups"]
    dtype, gates = DTYPES[case["dtype"]], DTYPES[case["gates"]]
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    s = dict(x=normal(steps, batch, dim).to(dtype), state=normal(batch, dim), lengths=None)
    # time constants of 5 to 200 steps; gates that forget within one step up to hundreds
    s["decay"] = (torch.exp(-1.0 / (5.0 * 40.0 ** torch.rand(dim, device="cuda", generator=g))) if groups == 0
                  else torch.sigmoid(2.0 + 2.0 * normal(steps, batch, groups))).to(gates)
    if case["ragged"]:
        lengths = torch.randint(0, steps + 1, (batch,), device="cuda", generator=g)
        lengths[0] = steps
        s["lengths"] = lengths.to(torch.int32)
    if case["train"]:
        s["dh"], s["d_last"] = normal(steps, batch, dim).to(dtype), normal(batch, dim)
    return s


def _prepare_logprobs(case, seed):
    g = _generator(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    logits = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    some = max(1, 64_000_000 // vocab)
    for r in range(0, rows, some):
        part = 2.5 * torch.randn(min(some, rows - r), vocab, device="cuda", generator=g)
        if case["masked"]:
            part.masked_fill_(torch.rand(part.shape, device="cuda", generator=g) < case["masked"], -math.inf)
        logits[r:r + some] = part
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    tokens = torch.where(torch.rand(rows, device="cuda", generator=g) < case["ignored"], IGNORED, tokens)
    s = dict(logits=logits, tokens=tokens, top=case["top"])
    if case["train"]:
        # a mean over the rows, and a little entropy asked for; scaled up where 16 bits would lose small gradients
        scale = 1000.0 if case["dtype"] == "float16" else 1.0 / rows
        s["d_logp"] = -scale * torch.rand(rows, device="cuda", generator=g)
        s["d_entropy"] = -0.01 * scale * torch.rand(rows, device="cuda", generator=g)
    return s


_PREPARE = {"spikes": _prepare_spikes, "scan": _prepare_scan, "logprobs": _prepare_logprobs}


def prepare(case, seed):
    case = dict(case)
    return case["kind"], case["train"], _PREPARE[case["kind"]](case, int(seed))


# ---------------------------------------------------------------------------------------------------------------------
# passes: the plain forms

def _plain_spikes(s, train):
    bits, w, batch = s["bits"], s["weight"].float(), s["batch"]
    (n, dim), steps = w.shape, bits.shape[0]
    words = (n * batch + 63) // 64
    z = (bits[:, :words, None] >> torch.arange(64, device="cuda")) & 1
    z = z.view(steps, words * 64)[:, :n * batch].view(steps, n, batch).transpose(1, 2).float().reshape(steps * batch, n)
    y = (z @ w).view(steps, batch, dim).to(s["weight"].dtype)
    if not train:
        return dict(y=y)
    dy = s["dy"].float().view(steps * batch, dim)
    return dict(y=y, d_weight=(z.t() @ dy).to(s["weight"].dtype),
                dl_dz=(dy @ w.t()).view(steps, batch, n).transpose(1, 2).reshape(steps, n * batch))


def _recurrence(a, x):
    """h[t] = a[t] * h[t - 1] + x[t] from h[-1] = 0: neighbouring steps are joined, the half as long recurrence gives every second h,
    one more step each the others."""
    steps = x.shape[0]
    if steps == 1:
        return x
    even = steps - steps % 2
    h_odd = _recurrence(a[1:even:2] * a[0:even:2], a[1:even:2] * x[0:even:2] + x[1:even:2])
    h = torch.empty_like(x)
    h[0] = x[0]
    h[1::2] = h_odd
    h[2::2] = a[2::2] * h_odd[:(steps - 1) // 2] + x[2::2]
    return h


def _plain_scan(s, train):
    x, decay, state, lengths = s["x"].float(), s["decay"].float(), s["state"], s["lengths"]
    steps, batch, dim = x.shape
    per_step = decay.dim() == 3
    a = decay.repeat_interleave(dim // decay.shape[2], dim=2) if per_step else decay.expand(steps, batch, dim)
    there = None
    if lengths is not None:
        there = (torch.arange(steps, device="cuda").view(-1, 1) < lengths).unsqueeze(2)
        a, x = torch.where(there, a, 1.0), torch.where(there, x, 0.0)
    x = torch.cat([(a[0] * state + x[0]).unsqueeze(0), x[1:]])
    h = _recurrence(a, x)
    out = (h if there is None else torch.where(there, h, 0.0)).to(s["x"].dtype)
    if not train:
        return dict(h=out, last=h[-1])
    dh = s["dh"].float()
    if there is not None:
        dh = torch.where(there, dh, 0.0)
    dh = torch.cat([dh[:-1], (dh[-1] + s["d_last"]).unsqueeze(0)])
    g = _recurrence(torch.cat([torch.ones_like(a[:1]), a[1:].flip(0)]), dh.flip(0)).flip(0)
    da = g * torch.cat([state.unsqueeze(0), h[:-1]])
    d_state = a[0] * g[0]
    if there is not None:
        g, da = torch.where(there, g, 0.0), torch.where(there, da, 0.0)
    da = da.view(steps, batch, decay.shape[2], -1).sum(3) if per_step else da.sum((0, 1))
    return dict(h=out, last=h[-1], dx=g.to(s["x"].dtype), d_decay=da.to(s["decay"].dtype), d_state=d_state)


def _plain_logprobs(s, train):
    logits, tokens, top = s["logits"], s["tokens"], s["top"]
    x = logits.float()
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    lp = torch.where(x == -math.inf, -math.inf, x - lse)
    p = torch.exp(lp)
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(1)
    given = tokens != IGNORED
    at = torch.where(given, tokens, 0).unsqueeze(1)
    out = dict(logp=torch.where(given, lp.gather(1, at).squeeze(1), 0.0), entropy=entropy, lse=lse.squeeze(1))
    if top:
        # the largest logits, of equal ones those with the lowest index: whole numbers in that order
        order = (x + 0.0).view(torch.int32).long()
        order = torch.where(order < 0, order ^ 0x7FFFFFFF, order)
        order = (order << 32) + (0xFFFFFFFF - torch.arange(x.shape[1], device="cuda"))
        out["top_index"] = torch.topk(order, top, dim=1).indices
        out["top_logp"] = lp.gather(1, out["top_index"])
    if train:
        by_logp = torch.where(given, s["d_logp"], 0.0).unsqueeze(1)
        d = -p * (by_logp + s["d_entropy"].unsqueeze(1) * (torch.where(p > 0, lp, 0.0) + entropy.unsqueeze(1)))
        d.scatter_add_(1, at, torch.where(lse == -math.inf, 0.0, by_logp))
        out["d_logits"] = d.to(logits.dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# passes: the framework's calls

def _own_spikes(s, train):
    from bmtk_amd import readout
    y = readout.spike_readout(s["bits"], s["weight"], s["batch"])
    if not train:
        return dict(y=y)
    d_weight, dl_dz = readout.spike_readout_bwd(s["bits"], s["weight"], s["dy"], s["batch"])
    return dict(y=y, d_weight=d_weight, dl_dz=dl_dz)


def _own_scan(s, train):
    from bmtk_amd import readout
    if not train:
        h, last = readout.gated_scan(s["x"], s["decay"], s["state"], s["lengths"])
        return dict(h=h, last=last)
    h, last, saved = readout.gated_scan(s["x"], s["decay"], s["state"], s["lengths"], save_state=True)
    dx, d_decay, d_state = readout.gated_scan_bwd(s["x"], s["decay"], saved, s["dh"], s["d_last"], s["lengths"])
    return dict(h=h, last=last, dx=dx, d_decay=d_decay, d_state=d_state)


def _own_logprobs(s, train):
    from bmtk_amd import readout
    r = readout.token_logprobs(s["logits"], s["tokens"], top=s["top"])
    out = dict(logp=r.logp, entropy=r.entropy, lse=r.lse)
    if s["top"]:
        out.update(top_index=r.top_index, top_logp=r.top_logp)
    if train:
        out["d_logits"] = readout.token_logprobs_bwd(s["logits"], s["tokens"], r, s["d_logp"], s["d_entropy"])
    return out


_PLAIN = {"spikes": _plain_spikes, "scan": _plain_scan, "logprobs": _plain_logprobs}
_OWN = {"spikes": _own_spikes, "scan": _own_scan, "logprobs": _own_logprobs}


def run(state):
    kind, train, s = state
    if own:
        return _OWN[kind](s, train)
    return _PLAIN[kind](s, train)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    size, train = SIZE[case["dtype"]], case["train"]
    if case["kind"] == "spikes":
        steps, n, batch, dim = case["steps"], case["n"], case["batch"], case["dim"]
        ne = n * batch
        spikes = steps * ne * case["rate"] * 1e-3
        # of the weights, the rows of the neurons that fired at all
        rows = n * (1.0 - math.exp(-steps * batch * case["rate"] * 1e-3))
        bytes_ = steps * ne / 8 + (n if train else rows) * dim * size + steps * batch * dim * size
        flops = spikes * dim
        if train:
            bytes_ += steps * batch * dim * size + n * dim * size + 4.0 * steps * ne
            flops += spikes * dim + 2.0 * steps * ne * dim
        return {"bytes": bytes_, "flops": flops}
    if case["kind"] == "scan":
        steps, batch, dim = case["steps"], case["batch"], case["dim"]
        share = 0.55 if case["ragged"] and batch > 1 else 1.0   # of the steps that are read, about
        cells, states = steps * batch * dim, batch * dim * 4
        gates = (steps * batch * case["groups"] if case["groups"] else dim) * SIZE[case["gates"]]
        bytes_ = share * (cells * size + gates) + cells * size + 2 * states
        flops = 2.0 * share * cells
        if train:
            bytes_ += share * cells * size + cells * size + gates + 2 * states
            flops += 6.0 * share * cells
        return {"bytes": bytes_, "flops": flops}
    rows, cells = case["rows"], case["rows"] * case["vocab"]
    bytes_ = cells * size + rows * (8 + 12 + 12 * case["top"])
    flops = 5.0 * cells
    if train:
        bytes_ += cells * size + rows * 8
        flops += 6.0 * cells
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits

def _exact_spikes(s, train):
    bits, batch = s["bits"], s["batch"]
    w = s["weight"].double()
    (n, dim), steps = w.shape, bits.shape[0]
    y = torch.zeros(steps, batch, dim, dtype=torch.float64, device="cuda")
    d_weight = torch.zeros_like(w)
    dl_dz = torch.empty(steps, n * batch, dtype=torch.float64, device="cuda") if train else None
    one = torch.arange(64, device="cuda")
    for t in range(steps):
        fired = bits[t].nonzero().squeeze(1)
        word, bit = ((bits[t][fired].unsqueeze(1) >> one) & 1).nonzero(as_tuple=True)
        element = fired[word] * 64 + bit
        element = element[element < n * batch]
        neuron, trial = element // batch, element % batch
        y[t].index_add_(0, trial, w[neuron])
        if train:
            dy = s["dy"][t].double()
            d_weight.index_add_(0, neuron, dy[trial])
            dl_dz[t] = (w @ dy.t().contiguous()).view(-1)
    return dict(y=y, d_weight=d_weight, dl_dz=dl_dz) if train else dict(y=y)


def _exact_scan(s, train):
    x, decay, lengths = s["x"], s["decay"], s["lengths"]
    steps, batch, dim = x.shape
    if lengths is None:
        lengths = torch.full((batch,), steps, dtype=torch.int32, device="cuda")
    gate = lambda t: (decay[t].double().unsqueeze(2).expand(-1, -1, dim // decay.shape[2]).reshape(batch, dim)  # noqa: E731
                      if decay.dim() == 3 else decay.double().expand(batch, dim))
    h = torch.zeros(steps, batch, dim, dtype=torch.float64, device="cuda")
    now = s["state"].double()
    for t in range(steps):
        there = (t < lengths).unsqueeze(1)
        now = torch.where(there, gate(t) * now + x[t].double(), now)
        h[t] = now * there
    out = dict(h=h, last=now)
    if train:
        dx = torch.zeros_like(h)
        d_decay = torch.zeros(decay.shape, dtype=torch.float64, device="cuda")
        back = s["d_last"].double()
        for t in range(steps - 1, -1, -1):
            there = (t < lengths).unsqueeze(1)
            g = torch.where(there, back + s["dh"][t].double(), 0.0)
            da = g * (h[t - 1] if t else s["state"].double())
            dx[t] = g
            if decay.dim() == 3:
                d_decay[t] = da.view(batch, decay.shape[2], -1).sum(2)
            else:
                d_decay += da.sum(0)
            back = torch.where(there, gate(t) * g, back)
        out.update(dx=dx, d_decay=d_decay, d_state=back)
    return out


def _exact_logprobs(s, train):
    logits, tokens, top = s["logits"], s["tokens"], s["top"]
    rows, vocab = logits.shape
    kinds = ["logp", "entropy", "lse"] + ["top_logp"] * (top > 0) + ["d_logits"] * train
    parts = {k: [] for k in kinds}
    some = max(1, 32_000_000 // vocab)
    for r in range(0, rows, some):
        x, token = logits[r:r + some].double(), tokens[r:r + some]
        lse = torch.logsumexp(x, 1)
        lp = x - lse.unsqueeze(1)
        lp = torch.where(lp.isnan(), -math.inf, lp)   # (rows of nothing but -inf)
        p = torch.exp(lp)
        entropy = torch.special.entr(p).sum(1)
        given = (token != IGNORED).double()
        at = token.clamp(min=0)
        parts["lse"].append(lse)
        parts["entropy"].append(entropy)
        parts["logp"].append(torch.where(given > 0, lp[torch.arange(len(at), device="cuda"), at], 0.0))
        if top:
            parts["top_logp"].append(torch.topk(lp, top, dim=1).values)
        if train:
            by_logp = s["d_logp"][r:r + some].double() * given
            d = torch.special.entr(p) - p * entropy.unsqueeze(1)
            d = d * s["d_entropy"][r:r + some].double().unsqueeze(1) - p * by_logp.unsqueeze(1)
            d[torch.arange(len(at), device="cuda"), at] += by_logp * (lse > -math.inf)
            parts["d_logits"].append(d)
    out = {k: torch.cat(v) for k, v in parts.items()}
    if top:
        out["top_index"] = None
    return out


_EXACT = {"spikes": _exact_spikes, "scan": _exact_scan, "logprobs": _exact_logprobs}


def exact(case, seed):
    kind, train, s = prepare(case, seed)
    return _EXACT[kind](s, train)
