"""Balance loss of a gate: calls that once went wrong (a trainer's counts after replays)."""
import pytest
import torch

import mdnvae_amd as M

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def mixture(n=68):
    torch.manual_seed(7)
    model = M.MDNGateVAE(R=3, n_nodes=n, k=6, n_layers=2, latent_dim=12, n_traits=4, symmetric_input=True).to(DEV)
    gen = torch.Generator().manual_seed(1)
    adjacency = [[int(v) for v in torch.randperm(n, generator=gen)[:6]] for _ in range(n)]
    x = M.data.synthetic_sc(48, n, seed=3, device=DEV)
    return model, adjacency, x, torch.randn(48, 4, generator=gen).to(DEV), torch.randn(48, 12, generator=gen).to(DEV)


@pytest.mark.parametrize("optimizer", ["adam", "muon"])
@pytest.mark.parametrize("fused", [True, False])
def test_gate_counts_are_the_last_steps_eager_or_replayed(fused, optimizer):
    model, adjacency, x, traits, eps = mixture()
    trainer = M.Trainer(model, "mdn", gate_balance=0.1, gate_top_k=1, fused_loss=fused, optimizer=optimizer)

    def counts_of(rows):
        z = model.gate(traits[rows]).detach().cpu()
        return torch.bincount(z.argmax(dim=1), minlength=3).to(torch.int32)

    def run(step, rows):
        want = counts_of(rows)                               # of the parameters that the step starts from
        step((x[rows], adjacency, traits[rows]), x[rows], eps[rows])
        torch.cuda.synchronize()
        assert torch.equal(trainer.gate_counts.cpu(), want), (step.__name__, rows)

    a, b, ragged = slice(0, 20), slice(20, 40), slice(40, 47)
    trainer.capture((x[a], adjacency, traits[a]), x[a], eps[a])
    assert trainer.gate_counts is None                       # no step yet
    for rows in (a, b):
        run(trainer.replay, rows)
    run(trainer.step, ragged)                                # the last batch of an epoch
    for rows in (b, a):
        run(trainer.replay, rows)
    run(trainer.step, a)
    held = trainer.gate_counts
    trainer.capture((x[b], adjacency, traits[b]), x[b], eps[b])
    assert trainer.gate_counts is held                       # capturing is no step
    run(trainer.replay, b)
