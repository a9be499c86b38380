"""Orthogonalised updates with two data-parallel ranks on one GPU (gloo through host memory, as in test_zgloo2_gpu.py): gradients
are summed first, symmetric first layers' folded and early from backward, late, or between two captured graphs; every rank then
takes the same step, which has to be the one of a single process on the whole batch.

Tolerance.  The two sum the same products in another order, so gradients differ by a share r of their norm (measured here, with a
bar of 64 roundings of 2^-22).  Where u is small the iteration is a = 3.4445 times u per step, and nowhere is it steeper, so an update
moves by at most a^5 r = 485 r, beside the 60 * 2^-22 of its norm that each of the two is off by itself and the parameter's rounding."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from conftest import load_fixture, fixture_params
import mdnvae_amd as M

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B, LR = 48, 0.02


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _train(lo, hi, seed, graph=False, **trainer_kw):
    """One step on subjects [lo, hi): (gradients, parameters before and after, momenta) by name, and the trainer."""
    fix = load_fixture("mm_gate")
    adjacency = [list(map(int, r)) for r in fix["adjacency"]]
    torch.manual_seed(seed)                                   # the gate layer is not in the fixture
    model = M.MDNGateVAE(R=5, n_nodes=68, k=32, n_layers=3, latent_dim=68, n_traits=4, symmetric_input=True)
    model.load_state_dict(fixture_params(fix), strict=False)
    with torch.no_grad():
        model.log_sigma.fill_(1.0)
    model = model.to(DEV)
    x = M.data.synthetic_sc(B, 68, seed=77, device=DEV)[lo:hi]
    g = torch.Generator().manual_seed(9)
    eps, traits = torch.randn(B, 68, generator=g).to(DEV)[lo:hi], torch.randn(B, 4, generator=g).to(DEV)[lo:hi]
    trainer = M.Trainer(model, "mdn", optimizer="muon", muon_lr=LR, muon_weight_decay=0.1, **trainer_kw)
    before = {k: v.detach().cpu().clone() for k, v in model.named_parameters()}
    if graph:
        trainer.capture((x, adjacency, traits), x, eps)
    (trainer.replay if graph else trainer.step)((x, adjacency, traits), x, eps)
    torch.cuda.synchronize()
    after = {k: v.detach().cpu().clone() for k, v in model.named_parameters()}
    grads = {k: v.grad.detach().cpu().clone() for k, v in model.named_parameters()}
    return grads, before, after, trainer.muon_buf.cpu(), trainer


def _worker(rank, world, port, overlap, graph, out):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    torch.cuda.set_device(0)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    lo, hi = M.data.shard_range(B, rank, world)
    grads, before, after, momenta, trainer = _train(lo, hi, 5 + 100 * rank, graph, **({} if overlap else {"overlap_floats": 0}))
    assert (trainer._graph_adam is not None) if graph else True
    assert bool(trainer._hook_of) == overlap
    out[rank] = (grads, before, after, momenta)
    dist.destroy_process_group()


@pytest.mark.parametrize("overlap,graph", [(True, False), (False, False), (True, True)])
def test_two_ranks_take_the_single_process_orthogonalised_step(overlap, graph):
    out = mp.Manager().dict()
    mp.spawn(_worker, args=(2, _free_port(), overlap, graph, out), nprocs=2, join=True)
    (g0, b0, a0, m0), (g1, b1, a1, m1) = out[0], out[1]
    assert torch.equal(m0, m1)
    grads, before, after, _, _ = _train(0, B, 5)
    for k, p in after.items():
        assert torch.equal(b0[k], b1[k]) and torch.equal(b0[k], before[k]), k          # rank 0's were broadcast
        assert torch.equal(a0[k], a1[k]) and torch.equal(g0[k], g1[k]), k              # replicas stay identical
        if p.dim() < 2:
            continue
        r = float((g0[k].double() - grads[k].double()).norm() / grads[k].double().norm())
        assert r <= 64 * 2.0 ** -22, (k, r)
        rows, cols = p.shape[0], p[0].numel()
        update = (p.double() - before[k].double() * (1 - LR * 0.1)).norm()
        scale = LR * max(1.0, rows / cols) ** 0.5
        bound = scale * 3.4445 ** 5 * r + 2 * 60 * 2.0 ** -22 * float(update) + 2.0 ** -22 * float(p.double().norm())
        assert float((a0[k].double() - p.double()).norm()) <= bound, k
        assert float(update) > 0
