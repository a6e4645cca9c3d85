"""What the readout operations do not take for what it looks like: arguments, refused before anything is asked of a device, and calls in native code."""
import ctypes as C
import sys
import types

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import bmtk_amd
from bmtk_amd import _lib, readout


def test_tangents():
    bits, tokens = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(10, dtype=torch.int64)
    with forward_ad.dual_level():
        w = forward_ad.make_dual(torch.ones(10, 4), torch.ones(10, 4))
        for call in (lambda: readout.spike_readout(bits, w, 4), lambda: readout.spike_readout_bwd(bits, w, torch.zeros(3, 4, 4), 4),
                     lambda: readout.gated_scan(w.view(5, 2, 4), torch.zeros(4))):
            for recording in (True, False):
                with torch.set_grad_enabled(recording), pytest.raises(ValueError, match="tangent"):
                    call()


def test_negated_views():
    x = torch.complex(torch.ones(3, 2, 1), torch.ones(3, 2, 1)).conj().imag
    assert x.is_neg()
    with pytest.raises(ValueError, match="resolve_neg"):
        readout.gated_scan(x, torch.ones(1))
    with pytest.raises(ValueError, match="current device"):
        readout.gated_scan(x.resolve_neg(), torch.ones(1))


@pytest.mark.parametrize("torch_version,abi,taken", [(torch.__version__, _lib.ABI_VERSION, True), (torch.__version__, _lib.ABI_VERSION - 1, False), (torch.__version__, None, False),
                                                     ("1.0", _lib.ABI_VERSION, False)])
def test_calls_in_native_code_of_another_header(monkeypatch, torch_version, abi, taken):
    """Compiled with another bmtk_amd.h than the library, they would call its functions by other signatures: the Python functions are used then."""
    handed = []
    module = types.ModuleType("bmtk_amd._readout")
    module.built_for, module.set_library = str(torch_version), lambda *a: handed.append(a)
    if abi is not None:
        module.abi_version = abi
    for name in readout._Native.NAMES:
        setattr(module, name, lambda *_: "native")
    monkeypatch.setitem(sys.modules, "bmtk_amd._readout", module)
    monkeypatch.setattr(bmtk_amd, "_readout", module, raising=False)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    native = readout._Native()
    assert native.spike_readout() is None
    assert len(handed) == taken and native.gated_scan() == ("native" if taken else None)


def test_native_code_that_is_built_names_its_header():
    native = pytest.importorskip("bmtk_amd._readout")
    assert native.abi_version == _lib.ABI_VERSION and native.built_for == str(torch.__version__)


def test_launches_of_too_many_threads():
    """2^32 threads are more than a launch takes: refused before anything of the call is enqueued."""
    lib, buf = _lib.load(), C.create_string_buffer(256)
    p = C.addressof(buf)

    def refused(code, *words):
        message = lib.bmtk_amd_last_error().decode()
        assert code == -1 and all(w in message for w in words), (code, message)
    # gates of three channels each, whose parts of the gradient are joined
    refused(lib.bmtk_gated_scan_bwd(1 << 22, 32, 96, 32, 1, 1, p, 32 * 96, 96, p, 32 * 32, 32, p, None, p, 32 * 96, 96, None, p, p, None, p, None), "gated_scan_bwd", "too many gates")
    # single trials, 128 neurons a workgroup
    n = (1 << 31) - 65
    refused(lib.bmtk_spike_readout_bwd_weight(p, (n + 63) // 64, 1, n, 1, p, 1, 0, p, None), "spike_readout_bwd_weight", "too many neurons")
