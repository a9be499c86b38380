"""Balance loss of a gate: calls that once went wrong (a trainer's counts after replays, means over very many rows)."""
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


# probabilities carry about eight fp32 roundings, and their sum eight more: sixteen halves of a step, whatever the number of rows
@pytest.mark.parametrize("T,E,dtype", [(1 << 27, 5, torch.float32), (1 << 26, 5, torch.float32), (1 << 25, 60, torch.bfloat16),
                                       (1 << 23, 160, torch.bfloat16), (1 << 21, 1000, torch.bfloat16), (1 << 21, 500, torch.float32)])
def test_means_over_many_equal_rows(T, E, dtype):
    """Every row rounds the same way: 128 to 512 rows of a lane in one fp32 sum were off by up to 6e-6."""
    loss, counts, mean = M.gate_balance_loss(torch.zeros(T, E, dtype=dtype, device=DEV), 1)
    assert int(counts[0]) == T and int(counts.sum()) == T
    assert float((mean.double() * E - 1.0).abs().max()) <= 16 * 2.0 ** -24
    assert abs(float(loss) - 1.0) <= 2 * 16 * 2.0 ** -24


def test_rows_of_a_lane_on_both_sides_of_a_flush():
    """1024 workgroups of 4 waves: one row per lane and 4096, 8192, ... rows more; padding in between."""
    E = 513                                                   # a row per wave
    for rows in (31, 32, 33, 64, 70):
        T = 4096 * (rows - 1) + 5
        z = torch.randn(T, E, generator=torch.Generator(device=DEV).manual_seed(rows), device=DEV)
        valid = torch.rand(T, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) < 0.9
        loss, counts, mean = M.gate_balance_loss(z, 1, valid)
        n = int(valid.sum())
        want = torch.zeros(E, dtype=torch.float64, device=DEV)
        for lo in range(0, T, 1 << 16):
            want += (torch.softmax(z[lo:lo + (1 << 16)].double(), dim=1) * valid[lo:lo + (1 << 16), None]).sum(dim=0)
        assert torch.equal(counts.long(), torch.bincount(z[valid].argmax(dim=1), minlength=E))
        assert float((mean.double() * n / want - 1.0).abs().max()) <= 16 * 2.0 ** -24, rows
        want_loss = float(E / n * (counts.double() * want / n).sum())
        assert abs(float(loss) - want_loss) <= 2 * 16 * 2.0 ** -24 * want_loss
