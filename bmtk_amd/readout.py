"""A readout of a spiking network that is trained on what it answers: the operations between the spike bits of a run and a loss
on labels, and their gradients down to the ``dl_dz`` that ``training.Glif3Bptt.backward`` takes.

``spike_readout``       spikes -> sums of weight rows, per step and trial
``short_conv``          sums -> weighted sums of the last few of them, a channel at a time
``gated_scan``          sums -> a memory that leaks, or that gates of the caller's own empty: h[t] = decay[t] * h[t - 1] + x[t]
``selective_scan``      sums -> a memory of several states a channel, whose step size, input and output weights come with every step
``token_logprobs``      logits -> log probability of each row's token (label), entropy, most probable alternatives
``projected_logprobs``  a memory's output -> log probability of each row's token under the softmax of its product with a vocabulary's weights, without the logits

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
    NAMES = ("spike_readout", "spike_readout_bwd", "gated_scan", "gated_scan_bwd", "token_logprobs", "token_logprobs_bwd", "short_conv", "short_conv_bwd", "selective_scan",
             "selective_scan_bwd", "projected_logprobs", "projected_logprobs_bwd")
    LIBRARY = ("spike_readout_workspace_bytes", "spike_readout_fwd", "spike_readout_bwd_weight", "spike_readout_bwd_spikes", "gated_scan_workspace_bytes",
               "gated_scan_fwd", "gated_scan_bwd", "token_logprobs_workspace_bytes", "token_logprobs_fwd", "token_logprobs_bwd", "short_conv_workspace_bytes", "short_conv_fwd",
               "short_conv_bwd", "selective_scan_workspace_bytes", "selective_scan_fwd", "selective_scan_bwd", "projected_logprobs_workspace_bytes", "projected_logprobs_fwd",
               "projected_logprobs_bwd")

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

def _ptr(t):
    return None if t is None else t.data_ptr()


def _sequences(x, name="x"):
    if x.dim() != 3 or x.shape[1] == 0 or x.shape[2] == 0:
        raise ValueError("{} must be [steps, sequences, channels]".format(name))
    return x.shape


def _conv(x, weight, bias, state, lengths, silu):
    """(steps, sequences, channels, width, sizes and what both directions point to)"""
    _given(x, "x")
    _contiguous(weight, "weight")
    steps, batch, dim = _sequences(x)
    if weight.dim() != 2 or weight.shape[0] != dim or not 2 <= weight.shape[1] <= _lib.CONV_MAX_WIDTH:
        raise ValueError("weight must be [{}, 2..{}], got {}".format(dim, _lib.CONV_MAX_WIDTH, tuple(weight.shape)))
    if weight.dtype != torch.float32 and weight.dtype != x.dtype:
        raise TypeError("weight must be float32 or of the type of x, {}, got {}".format(x.dtype, weight.dtype))
    width = weight.shape[1]
    if bias is not None:
        _contiguous(bias, "bias", weight.dtype, (dim,))
    if state is not None:
        _contiguous(state, "state", x.dtype, (width - 1, batch, dim))
    if lengths is not None:
        _contiguous(lengths, "lengths", torch.int32, (batch,))
    return steps, batch, dim, width, ((steps, batch, dim, width, _CODE[x.dtype], _CODE[weight.dtype], int(bool(silu))) + _rows(x, "x")
                                      + (weight.data_ptr(), _ptr(bias), _ptr(state), _ptr(lengths)))


def short_conv(x, weight, bias=None, state=None, lengths=None, silu=False):
    """y[t] = bias + the sum of the last few x, each with a weight of its channel, and with ``silu`` that times its sigmoid: (y, last).

    x       [steps, sequences, channels]; steps and sequences at any distance in memory, the channels next to one another
    weight  [channels, width], width 2 to 8; weight[:, width - 1] is for the present step.  Of the type of ``x`` or float32
    bias    [channels], of the type of ``weight`` (None: zero)
    state   [width - 1, sequences, channels], of the type of ``x``: the inputs before the first step (None: zero)
    lengths int32 [sequences]: steps of each sequence (None: all).  y is 0 behind them and nothing of x counts there; values outside
            0..steps count as the nearer of the two
    y has the type and shape of ``x``; last, of the state's shape: the last inputs of each sequence, the ``state`` of the next call, of a single step or
    of many."""
    r = _native.short_conv(x, weight, bias, state, lengths, silu)
    if r is not None:
        return r
    steps, batch, dim, width, args = _conv(x, weight, bias, state, lengths, silu)
    y = torch.empty(steps, batch, dim, dtype=x.dtype, device=x.device)
    last = torch.empty(width - 1, batch, dim, dtype=x.dtype, device=x.device)
    if steps:
        _lib.check(_lib.load().bmtk_short_conv_fwd(*args, y.data_ptr(), last.data_ptr(), _stream()))
    elif state is not None:
        last.copy_(state)
    else:
        last.zero_()
    return y, last


def short_conv_bwd(x, weight, dy, bias=None, state=None, d_last=None, lengths=None, silu=False):
    """(dx, d_weight, d_bias, d_state) from the gradients of ``short_conv``'s y, ``dy`` (the type of ``x``, strides as ``x`` may have), and last, ``d_last``
    (of last's type and shape, None: zero).  x, weight, bias, state, lengths, silu: as they were.

    dx: as ``x``, 0 behind a sequence's end; d_weight, d_bias: as ``weight`` and ``bias``, summed over steps and sequences; d_state: as ``state``.  All four are
    returned, where there was no bias or state too."""
    r = _native.short_conv_bwd(x, weight, dy, bias, state, d_last, lengths, silu)
    if r is not None:
        return r
    steps, batch, dim, width, args = _conv(x, weight, bias, state, lengths, silu)
    if _given(dy, "dy", x.dtype).shape != x.shape:
        raise ValueError("dy must be {}, got {}".format(tuple(x.shape), tuple(dy.shape)))
    if d_last is not None:
        _contiguous(d_last, "d_last", x.dtype, (width - 1, batch, dim))
    dev = x.device
    dx = torch.empty(steps, batch, dim, dtype=x.dtype, device=dev)
    make = torch.empty if steps else torch.zeros
    d_weight, d_bias = make(dim, width, dtype=weight.dtype, device=dev), make(dim, dtype=weight.dtype, device=dev)
    d_state = torch.empty(width - 1, batch, dim, dtype=x.dtype, device=dev)
    if steps:
        lib = _lib.load()
        ws = _Workspace(lib.bmtk_short_conv_workspace_bytes(steps, batch, dim, width, _CODE[x.dtype]), dev)
        _lib.check(lib.bmtk_short_conv_bwd(*args, *_rows(dy, "dy"), _ptr(d_last), dx.data_ptr(), d_weight.data_ptr(), d_bias.data_ptr(), d_state.data_ptr(), ws.ptr, _stream()))
    elif d_last is not None:
        d_state.copy_(d_last)
    else:
        d_state.zero_()
    return dx, d_weight, d_bias, d_state


# ---------------------------------------------------------------------------------------------------------------------

class SelectiveGrads(NamedTuple):
    """What ``selective_scan_bwd`` returns: gradients of the types and shapes of the inputs that they are named for."""
    dx: torch.Tensor
    d_dt: torch.Tensor
    d_rate: torch.Tensor
    d_write: torch.Tensor
    d_read: torch.Tensor
    d_skip: torch.Tensor
    d_dt_bias: torch.Tensor
    d_state: torch.Tensor


def _selective(x, dt, rate, write, read, skip, dt_bias, softplus, lengths):
    """(steps, sequences, channels, groups, states, sizes and what both directions point to)"""
    _given(x, "x")
    _given(dt, "dt")
    _contiguous(rate, "rate", torch.float32)
    steps, batch, dim = _sequences(x)
    if dt.dtype != torch.float32 and dt.dtype != x.dtype:
        raise TypeError("dt must be float32 or of the type of x, {}, got {}".format(x.dtype, dt.dtype))
    if tuple(dt.shape) != tuple(x.shape):
        raise ValueError("dt must be {}, got {}".format(tuple(x.shape), tuple(dt.shape)))
    if rate.dim() != 2 or rate.shape[0] != dim or not 1 <= rate.shape[1] <= _lib.SELECTIVE_MAX_STATES:
        raise ValueError("rate must be [{}, 1..{}], got {}".format(dim, _lib.SELECTIVE_MAX_STATES, tuple(rate.shape)))
    states = rate.shape[1]
    _given(write, "write", x.dtype)
    if write.dim() != 4 or tuple(write.shape[:2]) != (steps, batch) or write.shape[3] != states or not write.shape[2] or dim % write.shape[2]:
        raise ValueError("write must be [{}, {}, groups, {}] with a number of groups that divides the channels; got {}".format(steps, batch, states, tuple(write.shape)))
    groups = write.shape[2]
    _given(read, "read", x.dtype, write.shape)
    shared = ()
    for t, name in ((write, "write"), (read, "read")):
        if (states > 1 and t.stride(3) != 1) or (groups > 1 and t.stride(2) != states):
            raise ValueError("the groups' states of {} must lie next to one another".format(name))
        shared += (t.data_ptr(), t.stride(0), t.stride(1))
    for t, name in ((skip, "skip"), (dt_bias, "dt_bias")):
        if t is not None:
            _contiguous(t, name, torch.float32, (dim,))
    if lengths is not None:
        _contiguous(lengths, "lengths", torch.int32, (batch,))
    return steps, batch, dim, groups, states, ((steps, batch, dim, groups, states, _CODE[x.dtype], _CODE[dt.dtype], int(bool(softplus))) + _rows(x, "x") + _rows(dt, "dt")
                                               + shared + (rate.data_ptr(), _ptr(skip), _ptr(dt_bias)))


def selective_scan(x, dt, rate, write, read, skip=None, dt_bias=None, softplus=False, state=None, lengths=None, save_state=False):
    """A memory of several states a channel whose step size and whose input and output weights come with every step: (y, last), with ``save_state`` (y, last, saved).
    With delta = dt + dt_bias, or with ``softplus`` log(1 + e^(dt + dt_bias)),

        h[t, c, n] = e^(delta[t, c] rate[c, n]) h[t - 1, c, n] + delta[t, c] x[t, c] write[t, n]
        y[t, c]    = sum over n of read[t, n] h[t, c, n] + skip[c] x[t, c]

    x       [steps, sequences, channels]; steps and sequences at any distance in memory, the channels next to one another; dt likewise, of the type of ``x``
            or float32
    rate    float32 [channels, states], finite, up to 64 states; delta * rate is meant to be 0 or less, or at least such that e to its sum over any steps in a row
            stays in 32 bits: the decay of many steps is one exponential, and what it cannot hold makes NaN of a state that is still 0
    write, read  [steps, sequences, groups, states], of the type of ``x``, the states of a step next to one another; each group is for
            channels / groups neighbouring channels
    skip, dt_bias  float32 [channels] (None: zero)
    state   float32 [sequences, channels, states]: the state before the first step (None: zero)
    lengths int32 [sequences]: steps of each sequence (None: all).  y is 0 behind them and nothing of the inputs counts there; values outside
            0..steps count as the nearer of the two
    y has the type and shape of ``x``; last is float32 and of the state's shape: the ``state`` of the next call, of a single step or of many.  Where delta * x is infinite, y is
    NaN or infinite: NaN where the states are no multiple of four, too.
    saved: what ``selective_scan_bwd`` takes, float32 [steps / 16, sequences, channels, states]."""
    r = _native.selective_scan(x, dt, rate, write, read, skip, dt_bias, softplus, state, lengths, save_state)
    if r is not None:
        return r
    steps, batch, dim, groups, states, args = _selective(x, dt, rate, write, read, skip, dt_bias, softplus, lengths)
    if state is not None:
        _contiguous(state, "state", torch.float32, (batch, dim, states))
    dev = x.device
    y = torch.empty(steps, batch, dim, dtype=x.dtype, device=dev)
    last = torch.empty(batch, dim, states, dtype=torch.float32, device=dev)
    saved = torch.empty(-(-steps // _lib.SCAN_MARK), batch, dim, states, dtype=torch.float32, device=dev) if save_state else None
    if steps:
        lib = _lib.load()
        ws = _Workspace(lib.bmtk_selective_scan_workspace_bytes(steps, batch, dim, groups, states, 0), dev)
        _lib.check(lib.bmtk_selective_scan_fwd(*args, _ptr(state), _ptr(lengths), y.data_ptr(), last.data_ptr(), _ptr(saved), ws.ptr, _stream()))
    elif state is not None:
        last.copy_(state)
    else:
        last.zero_()
    return (y, last, saved) if save_state else (y, last)


def selective_scan_bwd(x, dt, rate, write, read, saved, dy, skip=None, dt_bias=None, softplus=False, d_last=None, lengths=None):
    """``SelectiveGrads`` from the gradients of ``selective_scan``'s y, ``dy`` (the type of ``x``, strides as ``x`` may have), and last, ``d_last`` (float32, None:
    zero).  The other arguments as they were; saved: what the forward pass returned.  The states are computed again from it in 32 bits.

    Gradients behind a sequence's end are 0.  d_write and d_read are summed over the channels of a group, d_rate, d_skip and d_dt_bias over steps and sequences.  All
    are returned, where there was no skip, dt_bias or state too."""
    r = _native.selective_scan_bwd(x, dt, rate, write, read, saved, dy, skip, dt_bias, softplus, d_last, lengths)
    if r is not None:
        return SelectiveGrads(*r)
    steps, batch, dim, groups, states, args = _selective(x, dt, rate, write, read, skip, dt_bias, softplus, lengths)
    if _given(dy, "dy", x.dtype).shape != x.shape:
        raise ValueError("dy must be {}, got {}".format(tuple(x.shape), tuple(dy.shape)))
    _contiguous(saved, "saved", torch.float32, (-(-steps // _lib.SCAN_MARK), batch, dim, states))
    if d_last is not None:
        _contiguous(d_last, "d_last", torch.float32, (batch, dim, states))
    dev = x.device
    make = lambda like, shape: (torch.empty if steps else torch.zeros)(shape, dtype=like.dtype, device=dev)  # noqa: E731
    d = SelectiveGrads(make(x, x.shape), make(dt, dt.shape), make(rate, rate.shape), make(write, write.shape), make(read, read.shape), make(rate, (dim,)),
                       make(rate, (dim,)), make(rate, (batch, dim, states)))
    if steps:
        lib = _lib.load()
        ws = _Workspace(lib.bmtk_selective_scan_workspace_bytes(steps, batch, dim, groups, states, 1), dev)
        _lib.check(lib.bmtk_selective_scan_bwd(*args, saved.data_ptr(), _ptr(lengths), *_rows(dy, "dy"), _ptr(d_last), d.dx.data_ptr(), d.d_dt.data_ptr(), d.d_write.data_ptr(),
                                               d.d_read.data_ptr(), d.d_rate.data_ptr(), d.d_skip.data_ptr(), d.d_dt_bias.data_ptr(), d.d_state.data_ptr(), ws.ptr, _stream()))
    elif d_last is not None:
        d.d_state.copy_(d_last)
    return d


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


# ---------------------------------------------------------------------------------------------------------------------

class ProjectedLogProbs(NamedTuple):
    """What ``projected_logprobs`` returns, float32 and of the shape of the tokens.  peak and total are for the backward pass: a multiple of 1/8 next to the row's
    largest logit times log2(e), and the sum of 2^(logit log2(e) - peak)."""
    logp: torch.Tensor
    lse: torch.Tensor
    peak: torch.Tensor
    total: torch.Tensor


def _projected(x, weight, tokens):
    """x as rows, (rows, vocabulary, channels, what both directions point to)."""
    _given(x, "x")
    _given(weight, "weight", x.dtype)
    _given(tokens, "tokens", torch.int64)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("x must be [..., channels]")
    dim = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] != dim:
        raise ValueError("weight must be [vocabulary, {}], got {}".format(dim, tuple(weight.shape)))
    if tuple(tokens.shape) != tuple(x.shape[:-1]):
        raise ValueError("tokens must be {}, got {}".format(tuple(x.shape[:-1]), tuple(tokens.shape)))
    flat = x if x.dim() == 2 else x.reshape(-1, dim)
    strides = []
    for t, name in ((flat, "x"), (weight, "weight")):
        if dim > 1 and t.stride(1) != 1:
            raise ValueError("the channels of {} must lie next to one another".format(name))
        strides.append(t.stride(0) if t.shape[0] > 1 else dim)
    rows, vocab = flat.shape[0], weight.shape[0]
    return flat, rows, vocab, dim, (flat.data_ptr(), strides[0], weight.data_ptr(), strides[1])


def projected_logprobs(x, weight, tokens, ignore=-100):
    """Log probability of each row's token under the softmax of ``x @ weight.T``, without the logits in memory: ``ProjectedLogProbs``.

    x       [..., channels], the channels of a row next to one another
    weight  [vocabulary, channels], of the type of ``x``: a row for each token, the channels next to one another
    tokens  int64 [...]; ``ignore`` where a row has none (padding): its logp is 0.  A token outside the vocabulary has logp NaN
    Rows whose logits hold NaN or +inf have lse and logp NaN, rows of nothing but -inf -inf; 2^124 and more counts as infinite.  Weights are meant to be finite: one that is not makes every row NaN.  float32 arguments of more than
    64 rows, with more than 128 in the vocabulary, are multiplied in three parts of 16 bits that hold all their bits; a row of those that holds an infinity has NaN where its logits would be -inf."""
    r = _native.projected_logprobs(x, weight, tokens, ignore)
    if r is not None:
        return ProjectedLogProbs(*r)
    flat, rows, vocab, dim, at = _projected(x, weight, tokens)
    r = ProjectedLogProbs(*(torch.empty(tokens.shape, dtype=torch.float32, device=x.device) for _ in range(4)))
    if rows:
        lib, code = _lib.load(), _CODE[x.dtype]
        tokens = tokens.contiguous()
        ws = _Workspace(lib.bmtk_projected_logprobs_workspace_bytes(rows, vocab, dim, code, *at, 0), x.device)
        _lib.check(lib.bmtk_projected_logprobs_fwd(rows, vocab, dim, code, *at, tokens.data_ptr(), ignore, *(t.data_ptr() for t in r), ws.ptr, _stream()))
    return r


def projected_logprobs_bwd(x, weight, tokens, fwd, d_logp, ignore=-100):
    """(dx, d_weight), of the types and shapes of ``x`` and ``weight``, from the gradient of logp, ``d_logp`` (float32, of the shape of the tokens).

    x, weight, tokens, ignore: as they were; fwd: what ``projected_logprobs`` returned.  Rows without a token, and rows of nothing but -inf, have a
    gradient of 0 and no part in d_weight, whatever they hold; a row whose token lies outside the vocabulary, or whose logits hold NaN or +inf, makes its own gradient and all of
    d_weight NaN, with a d_logp of 0 too.  The logits are made again, in pieces of the vocabulary of up to 512 MB of p - delta (or of 256 words for all rows, where that is
    more: 2 GB of four million rows of 16 bits, 6 of float32), which, times the mantissa of d_logp over the largest, is rounded to 16 bits (of float32: kept);
    float16 holds no gradient below 6e-8: give it a scaled d_logp, as a mean over many rows needs."""
    r = _native.projected_logprobs_bwd(x, weight, tokens, fwd.peak, fwd.total, d_logp, ignore)
    if r is not None:
        return r
    flat, rows, vocab, dim, at = _projected(x, weight, tokens)
    for t, name in ((fwd.peak, "peak"), (fwd.total, "total"), (d_logp, "d_logp")):
        _contiguous(t, name, torch.float32, tokens.shape)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    d_weight = (torch.empty if rows else torch.zeros)(vocab, dim, dtype=x.dtype, device=x.device)
    if rows:
        lib, code = _lib.load(), _CODE[x.dtype]
        tokens = tokens.contiguous()
        ws = _Workspace(lib.bmtk_projected_logprobs_workspace_bytes(rows, vocab, dim, code, *at, 1), x.device)
        _lib.check(lib.bmtk_projected_logprobs_bwd(rows, vocab, dim, code, *at, tokens.data_ptr(), ignore, fwd.peak.data_ptr(), fwd.total.data_ptr(), d_logp.data_ptr(), dx.data_ptr(),
                                                   d_weight.data_ptr(), ws.ptr, _stream()))
    return dx, d_weight
