"""Arguments of the readout operations that are not what they look like, refused before anything is asked of a device."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from bmtk_amd import readout


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
