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
