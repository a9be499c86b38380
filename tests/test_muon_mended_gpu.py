"""Orthogonalised updates: calls that once went wrong (batches of more matrices than one launch's extent holds,
bf16 results with products of fewer bits than asked for, small matrices whose arithmetic their neighbours decided,
coefficients that shrink the iterates below what fp16 parts held, masked weights)."""
import math

import pytest
import torch

import mdnvae_amd as M
from mdnvae_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL32 = 60 * 2.0 ** -22      # five steps of three products, each rounding to 2^-22 of its size, times four


def gaussian(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def exact(g, steps=5, coefficients=ops.NS_COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = g.double().cpu()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if tall else x
    x = x / torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True).clamp(min=eps)
    for _ in range(steps):
        s = x @ x.transpose(-1, -2)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(-1, -2) if tall else x


# 2^24 workgroups of 256 threads are one launch too many; so are 2^22 of 1024 (17 blocks of 32 x 32: one workgroup each only
# in a batch of 256 and more, which the ten left over for the last pass are not by themselves)
@pytest.mark.parametrize("count,rows,cols,dtype", [((1 << 24) + 3, 1, 1, torch.float32), ((1 << 22) + 9, 1, 520, torch.bfloat16)],
                         ids=["256 threads", "1024 threads"])
def test_more_small_matrices_than_a_launch_holds(count, rows, cols, dtype):
    one = torch.stack([gaussian(rows, cols, seed=i, dtype=dtype) for i in range(8)])
    x = one.to(DEV).repeat((count + 7) // 8, 1, 1)[:count].contiguous()
    y = ops.orthogonalize(x, out=torch.full_like(x, 7.0))
    want = ops.orthogonalize(one.to(DEV).repeat(40, 1, 1))[:8]
    half = 0.0 if dtype == torch.float32 else 2.0 ** -8
    for k in range(8):
        e = exact(one[k])
        assert float((want[k].double().cpu() - e).norm()) <= (half + TOL32) * float(e.norm())
        assert bool((y[k::8] == want[k]).all()), k


# both tiles, shares of X X^T, one workgroup, a batch
@pytest.mark.parametrize("shape", [(68, 68), (64, 512), (129, 129), (192, 1728), (1024, 640), (640, 1024), (1000, 4624), (16, 160, 161)], ids=str)
def test_bf16_result_is_the_fp32_one_rounded_once(shape):
    x = gaussian(*shape, seed=1, dtype=torch.bfloat16).to(DEV)
    wide = ops.orthogonalize(x.float())
    assert torch.equal(ops.orthogonalize(x), wide.bfloat16())
    # and so is as near to the definition as its rounding lets it be: |got - e| <= |rounded(e) - e| + 2 |fp32 result - e|
    e = exact(x)
    own = float((e.bfloat16().double() - e).norm())
    assert float((ops.orthogonalize(x).double().cpu() - e).norm()) <= own + 2 * TOL32 * float(e.norm())


def test_bf16_step_is_the_fp32_one_rounded_once():
    shapes = [(48, 1, 7, 7), (96, 48, 3, 3), (192, 96, 3, 3), (192, 192, 3, 3), (68, 768), (5, 4)]
    p, g = ([gaussian(*s, seed=k + i, dtype=torch.bfloat16).to(DEV) for i, s in enumerate(shapes)] for k in (0, 50))
    m = [gaussian(*s, seed=90 + i).to(DEV) for i, s in enumerate(shapes)]
    wide = [[t.float() for t in ts] for ts in (p, g)] + [[t.clone() for t in m]]
    ops.muon_step(p, g, m, lr=0.5, weight_decay=0.1)
    ops.muon_step(*wide, lr=0.5, weight_decay=0.1)
    assert all(torch.equal(a, b.bfloat16()) for a, b in zip(p, wide[0]))
    assert all(torch.equal(a, b) for a, b in zip(m, wide[2]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("arithmetic", ["f16", "f16x2"])
def test_a_small_matrix_keeps_its_arithmetic_in_any_company(arithmetic, dtype):
    """The large ones take 64 x 64 tiles: the list that the small ones would join."""
    shapes = [(68, 68), (48, 49), (128, 128), (1, 9), (192, 1728), (192, 1728), (192, 900)]
    make = lambda k, n: [gaussian(*s, seed=k + i, dtype=dtype).to(DEV) for i, s in enumerate(shapes[:n])]  # noqa: E731
    zeros = lambda n: [torch.zeros(s, device=DEV) for s in shapes[:n]]  # noqa: E731
    p = [torch.zeros_like(t) for t in make(0, 7)]
    alone = [t.clone() for t in p[:4]]
    ops.muon_step(p, make(50, 7), zeros(7), lr=1.0, scale=None, arithmetic=arithmetic)
    ops.muon_step(alone, make(50, 4), zeros(4), lr=1.0, scale=None, arithmetic=arithmetic)
    half = 0.0 if dtype == torch.float32 else 2.0 ** -8
    for a, b, g in zip(p, alone, make(50, 4)):
        e = exact(g)                                                     # u = g + 0.95 g: a multiple
        assert float((a.double().cpu() + e).norm()) <= (half + TOL32) * float(e.norm())
        if arithmetic == "f16":
            assert torch.equal(a, b)


# one block of X per wave (kept in fp32 registers), two and three blocks, tiled
@pytest.mark.parametrize("shape", [(40, 70), (256, 60, 500), (256, 30, 1180), (150, 260), (1000, 1000)], ids=str)
@pytest.mark.parametrize("coefficients,steps", [((0.1, 0.0, 0.0), 16), ((0.2, 0.1, 0.0), 16), ((0.05, 0.3, -0.2), 12), ((0.01, 0.0, 0.0), 16),
                                                ((0.5, 0.0, 0.0), 3), ((0.0, 0.0, 0.0), 2)], ids=str)
def test_coefficients_that_shrink_the_iterates(shape, coefficients, steps):
    x = gaussian(*shape, seed=4).to(DEV)
    got, want = ops.orthogonalize(x, steps=steps, coefficients=coefficients), exact(x[:2] if len(shape) == 3 else x, steps, coefficients)
    got = (got[:2] if len(shape) == 3 else got).double().cpu()
    # three roundings a step, as everywhere: nothing here is amplified
    assert float((got - want).norm()) <= 12 * steps * 2.0 ** -22 * float(want.norm())


@pytest.mark.parametrize("graph", [False, True])
def test_masked_weights_stay_zero(graph):
    """A masked layer's gradient is zero where its mask is, its orthogonalised update is not."""
    torch.manual_seed(3)
    n, B = 68, 4
    model = M.ConvVAE(decoder="gcn", intercept="diag", final="none", n_nodes=n, latent_dim=68).to(DEV)
    x, eps = M.data.synthetic_sc(B, n, seed=4, device=DEV), torch.randn(B, 68, device=DEV)
    trainer = M.Trainer(model, "poisson_log", optimizer="muon", muon_lr=0.01)
    mask = (torch.rand(n, n) < 0.5).float().fill_diagonal_(1.0)
    model.set_mask([mask] * 5)
    names = [f"fc{i}.weight" for i in range(4, 9)]
    before = {k: v.detach().clone() for k, v in model.named_parameters() if k in names}
    if graph:
        trainer.capture((x,), x, eps)
    for _ in range(2):
        (trainer.replay if graph else trainer.step)((x,), x, eps)
    torch.cuda.synchronize()
    got = dict(model.named_parameters())
    assert len(before) == 5
    for k, p0 in before.items():
        off_mask = mask.to(DEV) == 0
        assert bool((got[k][off_mask] == 0).all()), k
        assert bool((got[k][~off_mask] != p0[~off_mask]).float().mean() > 0.9), k


@pytest.mark.parametrize("shape", [(68, 68), (200, 300)], ids=str)
@pytest.mark.parametrize("below", [1e-2, 1e-4, 1e-6])
def test_norm_far_below_eps(shape, below):
    """X_0 is exact to 2^-40 in each entry, and the iterates that grow from it to half of that again."""
    x, eps = gaussian(*shape, seed=8), 1e-3
    x = x * (below * eps / float(x.norm()))
    got, want = ops.orthogonalize(x.to(DEV), eps=eps).double().cpu(), exact(x, eps=eps)
    share = 2 * math.sqrt(x.numel()) * 2.0 ** -40 * eps / float(x.double().norm())
    assert float((got - want).norm()) <= (TOL32 + share) * float(want.norm())
