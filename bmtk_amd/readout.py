"""A readout of a spiking network that is trained on what it answers: the operations between the spike bits of a run and a loss
on labels, and their gradients down to the ``dl_dz`` that ``training.Glif3Bptt.backward`` takes.

``spike_readout``    spikes -> sums of weight rows, per step and trial
``gated_scan``       sums -> a memory that leaks, or that gates of the caller's own empty: h[t] = decay[t] * h[t - 1] + x[t]
``token_logprobs``   logits -> log probability of each row's token (label), entropy, most probable alternatives

Each has its backward pass under its name with ``_bwd``, called by the caller as ``Glif3Bptt`` is: autograd does not follow any of
them (arguments that require gradients are refused while it records, those with a forward-mode tangent always).  Tensors are on the current device, work is enqueued on the current stream;
nothing synchronises, so all of it can be captured.  float32, bfloat16 and float16; arithmetic in 32 bits, what is returned in 16 bits is rounded
once.  The same call gives the same bits.  The reference has no counterpart (bmtk has no gradients).
"""
import ctypes as C
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _stream

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Native:
    """The same calls in native code for arguments that are as they should be, where that has been built for this torch and library; None for all others."""
    NAMES = ("spike_readout", "spike_readout_bwd", "gated_scan", "gated_scan_bwd", "token_logprobs", "token_logprobs_bwd")
    LIBRARY = ("spike_readout_workspace_bytes", "spike_readout_fwd", "spike_readout_bwd_weight", "spike_readout_bwd_spikes", "gated_scan_workspace_bytes",
               "gated_scan_fwd", "gated_scan_bwd", "token_logprobs_workspace_bytes", "token_logprobs_fwd", "token_logprobs_bwd")

    def __init__(self):
        for name in self.NAMES:
            setattr(self, name, self.first)

    def first(self, *_):
        """Looks for the module, once, when the library is needed on a GPU."""
        if not torch.cuda.is_initialized():
            return None
        lib = _lib.load()
        try:
            from . import _readout
        except ImportError:
            _readout = None
        # (it calls the library by the signatures and sizes of the header that it was built with)
        if (getattr(_readout, "built_for", None), getattr(_readout, "abi_version", None)) != (str(torch.__version__), _lib.ABI_VERSION):
            _readout = None
        if _readout is not None:
            _readout.set_library(tuple(C.cast(getattr(lib, "bmtk_" + name), C.c_void_p).value for name in self.LIBRARY), torch._C._cuda_getCurrentRawStream)
        for name in self.NAMES:
            setattr(self, name, getattr(_readout, name, lambda *_: None))
        return None


_native = _Native()


def _given(t, name, dtype=None, shape=None):
    """``t`` after the checks that every argument gets."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("{} must be a tensor".format(name))
    if forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError("{} carries a tangent, which forward-mode differentiation cannot take through this operation".format(name))
    if t.is_neg():
        raise ValueError("{} is a view of numbers with the other sign: call resolve_neg() on it".format(name))
    if not t.is_cuda or t.get_device() != torch.cuda.current_device():
        raise ValueError("{} must be on the current device".format(name))
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("{} requires gradients, which autograd cannot take through this operation: detach it, or call under torch.no_grad()".format(name))
    if dtype is None:
        if t.dtype not in _CODE:
            raise TypeError("{} must be float32, bfloat16 or float16, got {}".format(name, t.dtype))
    elif t.dtype != dtype:
        raise TypeError("{} must be {}, got {}".format(name, dtype, t.dtype))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("{} must be {}, got {}".format(name, tuple(shape), tuple(t.shape)))
    return t


def _contiguous(t, name, dtype=None, shape=None):
    if not _given(t, name, dtype, shape).is_contiguous():
        raise ValueError("{} must be contiguous".format(name))
    return t


class _Workspace:
    """Device memory of a call.  (Held until its kernels are enqueued: before that, another call of this stream could be given it.)"""

    def __init__(self, n_bytes, device):
        self.memory = torch.empty(n_bytes, dtype=torch.uint8, device=device) if n_bytes else None
        self.ptr = self.memory.data_ptr() if n_bytes else None


# ---------------------------------------------------------------------------------------------------------------------

def _spikes(bits, weight, batch):
    """(steps, neurons, channels, words of a row) after the checks of what both directions take."""
    _contiguous(weight, "weight")
    _given(bits, "bits", torch.int64)
    if weight.dim() != 2 or bits.dim() != 2 or weight.numel() == 0:
        raise ValueError("weight must be [neurons, channels] and bits [steps, words]")
    if type(batch) is not int or batch < 1:
        raise ValueError("batch must be a positive whole number")
    steps, (n, dim) = bits.shape[0], weight.shape
    if bits.shape[1] < (n * batch + 63) // 64:
        raise ValueError("bits has {} words per step, {} neurons x {} trials need {}".format(bits.shape[1], n, batch, (n * batch + 63) // 64))
    if bits.stride(1) != 1 and bits.shape[1] > 1:
        raise ValueError("the words of a step must lie next to one another in bits")
    return steps, n, dim, bits.stride(0) if steps > 1 else bits.shape[1]


def spike_readout(bits, weight, batch=1):
    """y [steps, batch, channels]: the sum of the rows of ``weight`` [neurons, channels] of the neurons that fired, for each step and trial.

    bits: int64 [steps, words] spike bits as ``Glif3Simulator.run`` returns them (bit e = neuron * batch + trial; what lies behind the last element
    is not looked at; rows may be further apart than they are long).  y has the type of ``weight``; the sums are in 32 bits."""
    y = _native.spike_readout(bits, weight, batch)
    if y is not None:
        return y
    steps, n, dim, stride = _spikes(bits, weight, batch)
    y = torch.empty(steps, batch, dim, dtype=weight.dtype, device=weight.device)
    if steps:
        lib = _lib.load()
        ws = _Workspace(lib.bmtk_spike_readout_workspace_bytes(steps, n, batch, dim, 0), weight.device)
        _lib.check(lib.bmtk_spike_readout_fwd(bits.data_ptr(), stride, steps, n, batch, weight.data_ptr(), dim, _CODE[weight.dtype], y.data_ptr(), ws.ptr, _stream()))
    return y


def spike_readout_bwd(bits, weight, dy, batch=1, spikes=True):
    """(d_weight, dl_dz) from ``dy`` [steps, batch, channels], of the type of ``weight``, the gradient of ``spike_readout``'s result.

    d_weight: as ``weight``.  dl_dz: float32 [steps, neurons * batch], the gradient by every spike, as ``Glif3Bptt.backward`` takes it;
    None with ``spikes=False`` (a network that is not trained itself)."""
    r = _native.spike_readout_bwd(bits, weight, dy, batch, spikes)
    if r is not None:
        return r
    steps, n, dim, stride = _spikes(bits, weight, batch)
    _contiguous(dy, "dy", weight.dtype, (steps, batch, dim))
    dev = weight.device
    d_weight = torch.empty_like(weight) if steps else torch.zeros_like(weight)
    dl_dz = torch.empty(steps, n * batch, dtype=torch.float32, device=dev) if spikes else None
    if steps:
        lib, code = _lib.load(), _CODE[weight.dtype]
        _lib.check(lib.bmtk_spike_readout_bwd_weight(bits.data_ptr(), stride, steps, n, batch, dy.data_ptr(), dim, code, d_weight.data_ptr(), _stream()))
        if spikes:
            ws = _Workspace(lib.bmtk_spike_readout_workspace_bytes(steps, n, batch, dim, 1) if code == 0 else 0, dev)
            _lib.check(lib.bmtk_spike_readout_bwd_spikes(weight.data_ptr(), dy.data_ptr(), steps, n, batch, dim, code, dl_dz.data_ptr(), ws.ptr, _stream()))
    return d_weight, dl_dz


# ---------------------------------------------------------------------------------------------------------------------

def _rows(t, name):
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError("the channels of {} must lie next to one another".format(name))
    return t.data_ptr(), t.stride(0), t.stride(1)


def _scan(x, decay, lengths):
    """(steps, sequences, channels, gates, arguments that both directions share, the decays that those point to)"""
    _given(x, "x")
    _given(decay, "decay")
    if x.dim() != 3 or x.shape[1] == 0 or x.shape[2] == 0:
        raise ValueError("x must be [steps, sequences, channels]")
    steps, batch, dim = x.shape
    if decay.dtype != torch.float32 and decay.dtype != x.dtype:
        raise TypeError("decay must be float32 or of the type of x, {}, got {}".format(x.dtype, decay.dtype))
    if decay.dim() == 1 and decay.shape[0] == dim:
        decay = decay.contiguous()
        groups, a = 0, (decay.data_ptr(), 0, 0)
    elif decay.dim() == 3 and decay.shape[0] == steps and decay.shape[1] == batch and decay.shape[2] and dim % decay.shape[2] == 0:
        groups, a = decay.shape[2], _rows(decay, "decay")
    else:
        raise ValueError("decay must be [channels], or [steps, sequences, gates] with a number of gates that divides the channels; got {} for x {}".format(
            tuple(decay.shape), tuple(x.shape)))
    if lengths is not None:
        _contiguous(lengths, "lengths", torch.int32, (batch,))
    return steps, batch, dim, groups, (steps, batch, dim, groups, _CODE[x.dtype], _CODE[decay.dtype]) + _rows(x, "x") + a, decay


def gated_scan(x, decay, state=None, lengths=None, save_state=False):
    """h[t] = decay[t] * h[t - 1] + x[t] over the steps of every sequence: (h, last), with ``save_state`` (h, last, saved).

    x       [steps, sequences, channels]; steps and sequences at any distance in memory (a transposed [sequences, steps, channels] is fine), the channels next
            to one another
    decay   [channels]: one per channel for all steps (a leaky integrator), or [steps, sequences, gates]: the gates of each step, each
            for channels / gates neighbouring channels; of the type of ``x`` or float32.  Of magnitude up to 1
    state   float32 [sequences, channels]: the state before the first step (None: zero)
    lengths int32 [sequences]: steps of each sequence (None: all).  h is 0 behind them, and nothing of x and decay counts there; values
            outside 0..steps count as the nearer of the two
    h has the type and shape of ``x``, last is float32 [sequences, channels], the state behind each sequence's last step: the ``state``
    of the next call.  saved: what ``gated_scan_bwd`` takes, float32, a sixteenth of h's entries."""
    r = _native.gated_scan(x, decay, state, lengths, save_state)
    if r is not None:
        return r
    steps, batch, dim, groups, args, decay = _scan(x, decay, lengths)
    if state is not None:
        _contiguous(state, "state", torch.float32, (batch, dim))
    dev = x.device
    h = torch.empty(steps, batch, dim, dtype=x.dtype, device=dev)
    last = torch.empty(batch, dim, dtype=torch.float32, device=dev)
    saved = torch.empty(-(-steps // _lib.SCAN_MARK), batch, dim, dtype=torch.float32, device=dev) if save_state else None
    if steps:
        lib = _lib.load()
        ws = _Workspace(lib.bmtk_gated_scan_workspace_bytes(steps, batch, dim, groups, 0), dev)
        _lib.check(lib.bmtk_gated_scan_fwd(*args, state.data_ptr() if state is not None else None, lengths.data_ptr() if lengths is not None else None,
                                           h.data_ptr(), last.data_ptr(), saved.data_ptr() if save_state else None, ws.ptr, _stream()))
    elif state is not None:
        last.copy_(state)
    else:
        last.zero_()
    return (h, last, saved) if save_state else (h, last)


def gated_scan_bwd(x, decay, saved, dh, d_last=None, lengths=None):
    """(dx, d_decay, d_state) from the gradients of ``gated_scan``'s h, ``dh`` (the type of ``x``, strides as ``x`` may have), and last, ``d_last`` (float32,
    None: zero).  x, decay, lengths: as they were; saved: what the forward pass returned.  The states are computed again from it in 32 bits, so
    h itself need not be kept.

    dx: as ``x``, 0 behind a sequence's end.  d_decay: as ``decay``, summed over the channels of a gate, and over all steps and
    sequences where there is one decay for them.  d_state: float32 [sequences, channels].

    Gates for an odd number of channels (33) take four bytes of device memory for each entry of ``x`` meanwhile, and up to ten times as long as gates for 32 or 64."""
    r = _native.gated_scan_bwd(x, decay, saved, dh, d_last, lengths)
    if r is not None:
        return r
    steps, batch, dim, groups, args, decay = _scan(x, decay, lengths)
    if _given(dh, "dh", x.dtype).shape != x.shape:
        raise ValueError("dh must be {}, got {}".format(tuple(x.shape), tuple(dh.shape)))
    _contiguous(saved, "saved", torch.float32, (-(-steps // _lib.SCAN_MARK), batch, dim))
    if d_last is not None:
        _contiguous(d_last, "d_last", torch.float32, (batch, dim))
    dev = x.device
    dx = torch.empty(steps, batch, dim, dtype=x.dtype, device=dev)
    d_decay = (torch.empty if steps else torch.zeros)(decay.shape, dtype=decay.dtype, device=dev)
    d_state = torch.empty(batch, dim, dtype=torch.float32, device=dev)
    if steps:
        lib = _lib.load()
        ws = _Workspace(lib.bmtk_gated_scan_workspace_bytes(steps, batch, dim, groups, 1), dev)
        _lib.check(lib.bmtk_gated_scan_bwd(*args, saved.data_ptr(), lengths.data_ptr() if lengths is not None else None, *_rows(dh, "dh"),
                                           d_last.data_ptr() if d_last is not None else None, dx.data_ptr(), d_decay.data_ptr(), d_state.data_ptr(), ws.ptr, _stream()))
    elif d_last is not None:
        d_state.copy_(d_last)
    else:
        d_state.zero_()
    return dx, d_decay, d_state


# ---------------------------------------------------------------------------------------------------------------------

class LogProbs(NamedTuple):
    """What ``token_logprobs`` returns, float32 and of the shape of the tokens; top_logp and top_index (int64) have one more dimension, or are None."""
    logp: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    top_logp: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


def _logits(logits, tokens, name="logits"):
    """Logits as rows, (rows, vocabulary, distance of rows)."""
    _given(logits, name)
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError("{} must be [..., vocabulary]".format(name))
    if tuple(tokens.shape) != tuple(logits.shape[:-1]):
        raise ValueError("tokens must be {}, got {}".format(tuple(logits.shape[:-1]), tuple(tokens.shape)))
    vocab = logits.shape[-1]
    rows = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    if vocab > 1 and rows.stride(1) != 1:
        raise ValueError("the entries of a row of {} must lie next to one another".format(name))
    return rows, rows.shape[0], vocab, rows.stride(0) if rows.shape[0] > 1 else vocab


def token_logprobs(logits, tokens, top=0, ignore=-100):
    """Log probability of each row's token under the softmax of its logits, the row's entropy, and its ``top`` (up to 64) most probable alternatives.

    logits  [..., vocabulary]; the entries of a row next to one another.  -inf: no probability
    tokens  int64 [...]; ``ignore`` where a row has none (padding): its logp is 0.  A token outside the vocabulary has logp NaN
    Returns ``LogProbs``: logp, entropy, lse (log of the sum of e^logit), top_logp and top_index: of equal logits the one with the
    lower index comes first.  A row of nothing but -inf: lse and logp -inf, entropy 0; one with NaN or +inf: NaN."""
    r = _native.token_logprobs(logits, tokens, top, ignore)
    if r is not None:
        return LogProbs(*r)
    _given(tokens, "tokens", torch.int64)
    rows, n, vocab, stride = _logits(logits, tokens)
    if type(top) is not int or not 0 <= top <= min(_lib.LOGPROBS_MAX_TOP, vocab):
        raise ValueError("top must lie in 0..{}".format(min(_lib.LOGPROBS_MAX_TOP, vocab)))
    dev, shape = logits.device, tokens.shape
    r = LogProbs(*(torch.empty(shape, dtype=torch.float32, device=dev) for _ in range(3)),
                 torch.empty(shape + (top,), dtype=torch.float32, device=dev) if top else None,
                 torch.empty(shape + (top,), dtype=torch.int64, device=dev) if top else None)
    if n:
        lib, code = _lib.load(), _CODE[logits.dtype]
        tokens = tokens.contiguous()
        ws = _Workspace(lib.bmtk_token_logprobs_workspace_bytes(n, vocab, code, top), dev)
        _lib.check(lib.bmtk_token_logprobs_fwd(n, vocab, code, rows.data_ptr(), stride, tokens.data_ptr(), ignore, top, r.logp.data_ptr(), r.entropy.data_ptr(),
                                               r.lse.data_ptr(), r.top_logp.data_ptr() if top else None, r.top_index.data_ptr() if top else None, ws.ptr, _stream()))
    return r


def token_logprobs_bwd(logits, tokens, fwd, d_logp=None, d_entropy=None, ignore=-100, out=None):
    """Gradient by the logits, of their type and shape, from those of logp and entropy (float32, of the shape of the tokens; one may be None).

    logits, tokens, ignore: as they were; fwd: what ``token_logprobs`` returned.  The alternatives are not differentiated.  Rows without a token get
    their entropy's gradient only (0, whatever their logits, where there is none), rows of nothing but -inf none.  out: where to write
    it; ``logits`` itself is allowed, which then are gone.  float16 holds no gradient below 6e-8: give it a scaled d_logp, as a mean over many rows needs."""
    if out is None:
        r = _native.token_logprobs_bwd(logits, tokens, fwd.lse, fwd.entropy, d_logp, d_entropy, ignore)
        if r is not None:
            return r
    _given(tokens, "tokens", torch.int64)
    rows, n, vocab, stride = _logits(logits, tokens)
    if d_logp is None and d_entropy is None:
        raise ValueError("give d_logp, d_entropy or both")
    shape = tokens.shape
    for t, name in ((fwd.lse, "lse"), (fwd.entropy, "entropy"), (d_logp, "d_logp"), (d_entropy, "d_entropy")):
        if t is not None:
            _contiguous(t, name, torch.float32, shape)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        to, to_stride = out, vocab
    else:
        _given(out, "out", logits.dtype, logits.shape)
        to, _, _, to_stride = _logits(out, tokens, "out")
        if n and (to.data_ptr() != out.data_ptr() or to_stride < vocab):
            raise ValueError("the rows of out must lie at one distance, and apart")
        if n and _overlap(rows, to) and (rows.data_ptr() != to.data_ptr() or stride != to_stride):
            raise ValueError("out shares memory with logits: it must be the same tensor, or another one")
    if n:
        tokens = tokens.contiguous()
        _lib.check(_lib.load().bmtk_token_logprobs_bwd(
            n, vocab, _CODE[logits.dtype], rows.data_ptr(), stride, tokens.data_ptr(), ignore, fwd.lse.data_ptr(), fwd.entropy.data_ptr(),
            d_logp.data_ptr() if d_logp is not None else None, d_entropy.data_ptr() if d_entropy is not None else None, to.data_ptr(), to_stride, _stream()))
    return out


def _overlap(a, b):
    first = [t.data_ptr() for t in (a, b)]
    end = [p + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size() for p, t in zip(first, (a, b))]
    return first[0] < end[1] and first[1] < end[0]
