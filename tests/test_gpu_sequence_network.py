"""A network that is simulated, its sequence readout's loss, and the gradients of the readout and of the network's synapses."""
import pytest
import torch

from bmtk_amd import ops, synthetic, training
from bmtk_amd.simulator import Glif3Simulator
from test_gpu_readout import U
from test_gpu_sequence_loss import PARAMETERS, case, on_device, reference, run

pytestmark = pytest.mark.gpu


def test_sequence_loss_trains_a_network_down_to_its_spikes():
    """The readout's gradients against float64 autograd of the definition, the synapses' as what Glif3Bptt makes of that dl_dz."""
    n, batch, steps, channels, states, groups, vocab = 96, 4, 120, 24, 8, 2, 30
    cfg = synthetic.small_glif3_network(n=n, n_in=200, steps=steps, seed=3, in_w_scale=4.0)
    sim = Glif3Simulator(n, cfg["par"], 1.0, batch=batch, rec=cfg["rec_src"], inp=cfg["inp_src"], ring_slots=cfg["L"])
    in_ptr, in_events = ops.poisson_events(200, 60.0, 1.0, steps, batch=batch, seed=5)
    sim.set_input_events(in_ptr, in_events)
    fwd = sim.run(steps, save_state=True)
    z = sim.raster(fwd["bits"]).cpu().view(steps, n * batch).bool()
    assert z.sum() > 100
    c = dict(case(steps, batch, n, channels, states, groups, vocab, torch.float32), z=z)
    loss, dl_dz, grads, answer, _ = run(dict(on_device(c), bits=fwd["bits"]))
    want_loss, want_logp, want, _ = reference(c)
    # everything is of order one: as many roundings as the longest sums one behind the other have terms, forward and back, of terms up to some four times the largest result
    tolerance = 4 * 2 * (steps + batch + n + channels * states + vocab) * U
    assert (loss.double().cpu() - want_loss).abs() <= tolerance * (1 + want_loss)
    assert (answer.logp.double().cpu() - want_logp).abs().max() <= tolerance * (1 + want_logp.abs().max())
    for name in PARAMETERS:
        assert (grads[name].double().cpu() - want[name]).abs().max() <= tolerance * want[name].abs().max(), name
    by_spike = want["z"].reshape(steps, n * batch)
    assert dl_dz.any() and (dl_dz.double().cpu() - by_spike).abs().max() <= tolerance * by_spike.abs().max()
    bptt, other = training.Glif3Bptt(sim), training.Glif3Bptt(sim)
    bptt.backward(fwd, dl_dz=dl_dz)
    other.backward(fwd, dl_dz=by_spike.float().cuda())
    assert torch.isfinite(bptt.d_rec_w).all() and bptt.d_rec_w.abs().sum() > 0
    # (the same pass, which is linear, of a dl_dz that is off by `tolerance` of its largest entry at most; entries that are off alike add up where a synapse's own do not: ten times that)
    assert (bptt.d_rec_w - other.d_rec_w).abs().max() <= 10 * tolerance * other.d_rec_w.abs().max()
