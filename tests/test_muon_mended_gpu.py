"""Orthogonalised updates: calls that once went wrong (batches of more matrices than one launch's extent holds)."""
import pytest
import torch

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
