"""What the readout operations refuse, before any launch: by the C ABI's checks and by the Python functions' own."""
import ctypes as C
import os
import re

import pytest
import torch

from bmtk_amd import _lib, readout

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUF = C.create_string_buffer(256)
P = C.addressof(BUF)


def refused(code, *words):
    message = _lib.load().bmtk_amd_last_error().decode()
    assert code == -1, code
    for w in words:
        assert w in message, message


def test_constants_are_the_headers():
    txt = open(os.path.join(ROOT, "include", "bmtk_amd.h")).read()
    value = lambda name: int(re.search(r"#define {} (\d+)".format(name), txt).group(1))  # noqa: E731
    assert value("BMTK_SCAN_MARK") == _lib.SCAN_MARK
    assert value("BMTK_LOGPROBS_MAX_TOP") == _lib.LOGPROBS_MAX_TOP
    assert [value("BMTK_F32"), value("BMTK_BF16"), value("BMTK_F16")] == [readout._CODE[t] for t in (torch.float32, torch.bfloat16, torch.float16)]


def spikes_fwd(bits=P, stride=100, steps=3, n=10, batch=4, weight=P, dim=8, dtype=0, y=P, ws=P):
    return _lib.load().bmtk_spike_readout_fwd(bits, stride, steps, n, batch, weight, dim, dtype, y, ws, None)


@pytest.mark.parametrize("change,word", [
    (dict(bits=None), "null"), (dict(weight=None), "null"), (dict(y=None), "null"), (dict(steps=0), "positive"), (dict(n=0), "positive"), (dict(batch=0), "positive"),
    (dict(dim=0), "positive"), (dict(dim=-1), "positive"), (dict(dtype=3), "type"), (dict(dtype=-1), "type"), (dict(stride=0), "stride"), (dict(n=1 << 31), "2^31"),
    (dict(n=1 << 29, batch=4), "2^31"), (dict(steps=1 << 23), "2^23"), (dict(steps=1 << 22, batch=1 << 9), "2^31"), (dict(dim=65537), "65,536"), (dict(batch=65537), "65,536"),
    (dict(steps=1 << 20, batch=1, n=10, dim=4096), "too large"), (dict(n=1 << 20, batch=1, steps=1, stride=1 << 20, ws=None), "workspace")])
def test_spike_readout_fwd(change, word):
    refused(spikes_fwd(**change), "spike_readout_fwd", word)


def test_spike_readout_bwd():
    lib = _lib.load()
    refused(lib.bmtk_spike_readout_bwd_weight(P, 1, 3, 10, 4, None, 8, 0, P, None), "null")
    refused(lib.bmtk_spike_readout_bwd_weight(P, 0, 3, 10, 4, P, 8, 0, P, None), "stride")
    refused(lib.bmtk_spike_readout_bwd_weight(P, 1, 3, 10, 4, P, 8, 7, P, None), "type")
    refused(lib.bmtk_spike_readout_bwd_spikes(P, P, 3, 10, 4, 8, 0, None, P, None), "null")
    refused(lib.bmtk_spike_readout_bwd_spikes(P, P, 3, 1 << 30, 4, 8, 0, P, P, None), "2^31")
    refused(lib.bmtk_spike_readout_bwd_spikes(P, P, 300, 10000, 32, 8, 0, P, None, None), "workspace")
    assert lib.bmtk_spike_readout_workspace_bytes(0, 10, 4, 8, 0) == 0
    assert lib.bmtk_spike_readout_workspace_bytes(1000, 10000, 1, 8, 0) == 0            # steps enough
    assert lib.bmtk_spike_readout_workspace_bytes(1, 1 << 20, 1, 8, 0) % (8 * 4) == 0 < lib.bmtk_spike_readout_workspace_bytes(1, 1 << 20, 1, 8, 0)


def scan_fwd(steps=5, batch=2, dim=8, groups=0, dtype=0, gates=0, x=P, decay=P, h=P, last=P, ws=P):
    return _lib.load().bmtk_gated_scan_fwd(steps, batch, dim, groups, dtype, gates, x, batch * dim, dim, decay, batch * dim, dim, None, None, h, last, None, ws, None)


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "null"), (dict(decay=None), "null"), (dict(h=None), "null"), (dict(last=None), "null"), (dict(steps=0), "positive"), (dict(batch=0), "positive"),
    (dict(dim=0), "positive"), (dict(groups=-1), "positive"), (dict(groups=3), "evenly"), (dict(groups=16), "evenly"), (dict(dtype=5), "type"), (dict(gates=1), "decays"),
    (dict(dtype=1, gates=2), "decays"), (dict(steps=(1 << 31) - 1), "too many"), (dict(batch=1 << 30), "too many"), (dict(steps=1 << 20, ws=None), "workspace")])
def test_gated_scan_fwd(change, word):
    refused(scan_fwd(**change), "gated_scan_fwd", word)


def test_gated_scan_bwd():
    lib = _lib.load()

    def bwd(groups, marks=P, ws=P, dh=P):
        return lib.bmtk_gated_scan_bwd(5, 2, 8, groups, 0, 0, P, 16, 8, P, 16, 8, marks, None, dh, 16, 8, None, P, P, None, ws, None)
    refused(bwd(0, marks=None), "null")
    refused(bwd(0, dh=None), "null")
    refused(bwd(0, ws=None), "workspace")    # parts of the decays' gradient
    refused(bwd(5), "evenly")
    assert lib.bmtk_gated_scan_workspace_bytes(5, 2, 8, 8, 1) == 0
    assert lib.bmtk_gated_scan_workspace_bytes(5, 2, 8, 3, 1) == 0
    assert lib.bmtk_gated_scan_workspace_bytes(5, 2, 8, 0, 1) >= 2 * 8 * 4


def logprobs(rows=2, vocab=10, dtype=0, logits=P, tokens=P, top=0, logp=P, top_logp=P, top_index=P, ws=P):
    return _lib.load().bmtk_token_logprobs_fwd(rows, vocab, dtype, logits, vocab, tokens, -100, top, logp, P, P, top_logp, top_index, ws, None)


@pytest.mark.parametrize("change,word", [
    (dict(logits=None), "null"), (dict(tokens=None), "null"), (dict(logp=None), "null"), (dict(rows=0), "positive"), (dict(vocab=0), "positive"), (dict(dtype=9), "type"),
    (dict(top=-1), "top"), (dict(top=11), "top"), (dict(top=65, vocab=100), "top"), (dict(top=2, top_logp=None), "nowhere"), (dict(top=2, top_index=None), "nowhere"),
    (dict(rows=1 << 24), "2^24"), (dict(vocab=1 << 30), "2^30"), (dict(rows=1, vocab=200000, ws=None), "workspace")])
def test_token_logprobs_fwd(change, word):
    refused(logprobs(**change), "token_logprobs_fwd", word)


def test_token_logprobs_bwd():
    lib = _lib.load()
    refused(lib.bmtk_token_logprobs_bwd(2, 10, 0, P, 10, P, -100, P, P, None, None, P, 10, None), "no gradient")
    refused(lib.bmtk_token_logprobs_bwd(2, 10, 0, P, 10, P, -100, None, P, P, None, P, 10, None), "null")


def test_tensors_on_the_host_are_refused():
    bits, w = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(10, 4)
    for call in (lambda: readout.spike_readout(bits, w, 4), lambda: readout.spike_readout_bwd(bits, w, torch.zeros(3, 4, 4), 4),
                 lambda: readout.gated_scan(torch.zeros(3, 2, 4), torch.zeros(4)), lambda: readout.token_logprobs(w, torch.zeros(10, dtype=torch.int64))):
        with pytest.raises(ValueError, match="current device"):
            call()
    with pytest.raises(TypeError, match="tensor"):
        readout.gated_scan([[[1.0]]], torch.zeros(1))
