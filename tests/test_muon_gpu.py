"""Orthogonalised updates (ops.orthogonalize, ops.muon_step, Trainer(optimizer="muon")) against the definition in float64.

Tolerances.  fp32: a step rounds X, B and their product to about 2^-22 of their size (two fp16 parts each, fp32 sums); five
steps of three such roundings, times four for spectra whose small directions grow faster than the norm: 60 * 2^-22 =
1.5e-5 of the result's norm.  bf16: the result's rounding, 2^-8, and for matrices that take the tiled kernels products of
operands rounded to 11 bits - three operands in each of the three steps in which B is not small against a, 2^-11 /
sqrt(3) each: 2^-8 + 9 * 2^-11 / sqrt(3) = 6.4e-3."""
import math

import pytest
import torch

import mdnvae_amd as M
from mdnvae_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = {torch.float32: 60 * 2.0 ** -22, torch.bfloat16: 2.0 ** -8 + 9 * 2.0 ** -11 / math.sqrt(3)}


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


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def gaussian(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# one workgroup (its limits: 128 x 128, 32 x 1184, 64 x 512), just over it, tiles that end inside, tall and wide, batches
SHAPES = [(1, 1), (1, 7), (9, 1), (5, 4), (31, 33), (68, 68), (87, 32), (68, 128), (128, 128), (32, 1184), (64, 512), (3, 64, 500),
          (129, 128), (129, 129), (33, 1200), (130, 200), (2, 200, 130), (192, 1728), (300, 40), (5, 2, 160, 161), (512, 512),
          (520, 1030), (1024, 640)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize_matches_float64(shape, dtype):
    x = gaussian(*shape, seed=sum(shape), dtype=dtype)
    y = ops.orthogonalize(x.to(DEV))
    assert y.shape == x.shape and y.dtype == dtype
    assert off(y, exact(x)) <= TOL[dtype]


# what the cost of a launch decides: both tiles for each product, X X^T in one piece, in a few and in many (the shares of
# (129, 20000) number 32, the last of them shorter), a batch that fills the chip
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(160, 1000), (129, 20000), (700, 5000), (1000, 4624), (1500, 1501), (1990, 2000), (4, 1000, 2048)], ids=str)
def test_large_matrices(shape, dtype):
    x = gaussian(*shape, seed=sum(shape), dtype=dtype).to(DEV)
    y = ops.orthogonalize(x, steps=3)
    a, b, c = ops.NS_COEFFICIENTS
    want = x.double()
    want = want / torch.linalg.vector_norm(want, dim=(-2, -1), keepdim=True)
    for _ in range(3):
        s = want @ want.transpose(-1, -2).contiguous()
        want = a * want + (b * s + c * (s @ s)) @ want
    assert float((y.double() - want).norm() / want.norm()) <= TOL[dtype]


# matrices of two and three blocks per wave go to one workgroup each from 256 of them on; the same ones alone do not
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(256, 60, 500), (259, 30, 1180), (256, 1180, 30)], ids=str)
def test_large_batches_of_middling_matrices(shape, dtype):
    x = gaussian(*shape, seed=3, dtype=dtype)
    y = ops.orthogonalize(x.to(DEV))
    some = [0, 17, shape[0] - 1]
    want = exact(x[some])
    for i, k in enumerate(some):
        assert off(y[k], want[i]) <= TOL[dtype]
        assert off(ops.orthogonalize(x[k].to(DEV)), want[i]) <= TOL[dtype]
    assert bool(torch.isfinite(y).all())


@pytest.mark.parametrize("steps", [1, 2, 3, 9, 16])
@pytest.mark.parametrize("shape", [(40, 70), (150, 260)], ids=str)
def test_number_of_steps(shape, steps):
    x = gaussian(*shape, seed=steps)
    # every step adds its three roundings; fewer steps, fewer of them
    assert off(ops.orthogonalize(x.to(DEV), steps=steps), exact(x, steps)) <= 12 * steps * 2.0 ** -22


@pytest.mark.parametrize("coefficients", [(1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.0, 0.0, 0.0), (0.0, 0.0, 0.0)], ids=str)
@pytest.mark.parametrize("shape", [(40, 70), (150, 260)], ids=str)
def test_other_coefficients(shape, coefficients):
    x = gaussian(*shape, seed=3)
    got, want = ops.orthogonalize(x.to(DEV), coefficients=coefficients), exact(x, 5, coefficients)
    assert float((got.double().cpu() - want).norm()) <= TOL[torch.float32] * max(float(want.norm()), 1e-30)


@pytest.mark.parametrize("shape", [(96, 128), (256, 400)], ids=str)
def test_falling_spectrum_is_as_exact_as_plain_fp32(shape):
    """Singular values 1, 2^-1.5, 3^-1.5, ...: the small directions are amplified a hundredfold, with all noise in them."""
    m, n = shape
    u, v = torch.linalg.qr(gaussian(m, m, seed=1).double())[0], torch.linalg.qr(gaussian(n, m, seed=2).double())[0]
    x = ((u * torch.arange(1, m + 1).double().pow(-1.5)) @ v.t()).float()
    want = exact(x)
    a, b, c = ops.NS_COEFFICIENTS
    plain = x / x.norm()
    for _ in range(5):
        s = plain @ plain.t()
        plain = a * plain + (b * s + c * (s @ s)) @ plain
    # 22-bit operands against 24-bit ones, but a X apart from B X: no worse than twice the plain iteration
    assert off(ops.orthogonalize(x.to(DEV)), want) <= 2 * off(plain, want) + 2.0 ** -22


@pytest.mark.parametrize("shape", [(68, 68), (200, 300)], ids=str)
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e20, 3e38], ids=str)
def test_scale_of_the_input(shape, scale):
    x = (gaussian(*shape, seed=5).clamp(-1, 1) * scale)
    got, want = ops.orthogonalize(x.to(DEV)).double().cpu(), exact(x)
    assert torch.isfinite(got).all()
    # below eps the result is small itself: fp16 parts hold X down to 2^-38
    assert float((got - want).norm()) <= TOL[torch.float32] * float(want.norm()) + 2.0 ** -38 * 500 * math.sqrt(x.numel())


@pytest.mark.parametrize("shape", [(4, 40, 60), (4, 140, 200)], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
def test_non_finite_and_zero_matrices_stay_by_themselves(shape, bad):
    x = gaussian(*shape, seed=6)
    want = exact(x)
    x[1, 3, 5] = bad
    x[2] = 0.0
    y = ops.orthogonalize(x.to(DEV)).cpu()
    assert torch.isnan(y[1]).all() and bool((y[2] == 0).all())
    for i in (0, 3):
        assert off(y[i], want[i]) <= TOL[torch.float32]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(41, 67), (133, 257), (257, 133)], ids=str)
def test_unaligned_storage_and_in_place(shape, dtype):
    n = shape[0] * shape[1]
    buf = torch.full((n + 8,), 7.0, dtype=dtype, device=DEV)
    x = gaussian(*shape, seed=7, dtype=dtype)
    view = buf[1:1 + n].view(shape)
    view.copy_(x)
    want = ops.orthogonalize(x.to(DEV))
    assert ops.orthogonalize(view, out=view) is not None
    assert torch.equal(view, want)
    assert bool((buf[0] == 7) & (buf[1 + n:] == 7).all())


def test_empty_matrices():
    for shape in [(0, 5), (5, 0), (0, 3, 3)]:
        assert ops.orthogonalize(torch.empty(shape, device=DEV)).shape == shape
    ops.muon_step([], [], [], lr=0.1)
    p = torch.empty(0, 4, device=DEV)
    ops.muon_step([p], [p.clone()], [p.clone()], lr=0.1)


def test_many_small_matrices_past_32_bit_offsets():
    n = (1 << 31) // (68 * 68) + 40
    x = torch.empty(n, 68, 68, dtype=torch.bfloat16, device=DEV)
    x[:] = gaussian(68, 68, seed=8).to(DEV)
    x[-1] = gaussian(68, 68, seed=9).to(DEV)
    y = ops.orthogonalize(x, out=x)
    assert off(y[-1], exact(gaussian(68, 68, seed=9, dtype=torch.bfloat16))) <= TOL[torch.bfloat16]
    assert torch.equal(y[0], y[-2]) and off(y[0], exact(gaussian(68, 68, seed=8, dtype=torch.bfloat16))) <= TOL[torch.bfloat16]


def test_batch_in_several_passes():
    """More matrices than one pass's workspace holds (1 GiB): the passes differ in size, the results do not."""
    one = gaussian(300, 900, seed=10)
    per = M._lib.load().mdnvae_orthogonalize_workspace_bytes(1, 300, 900)
    n = (1 << 30) // per * 2 + 3
    x = one.to(DEV).expand(n, 300, 900).contiguous()
    y = ops.orthogonalize(x)
    want = exact(one)
    for i in (0, n // 2, n - 1):
        assert off(y[i], want) <= TOL[torch.float32]


def test_same_call_same_bits():
    for shape in [(68, 68), (192, 900)]:
        x = gaussian(*shape, seed=11).to(DEV)
        assert torch.equal(ops.orthogonalize(x), ops.orthogonalize(x))


# ---- the step ---------------------------------------------------------------------------------------------------------
def step64(p, g, m, lr, momentum, nesterov, decay, scale):
    p, g, m = p.double(), g.double(), m.double()
    m = momentum * m + g
    o = exact((g + momentum * m if nesterov else m).reshape(p.shape[0], -1))
    rows, cols = o.shape
    s = {"shape": max(1.0, rows / cols) ** 0.5, "rms": 0.2 * max(rows, cols) ** 0.5, None: 1.0}[scale]
    return (1 - lr * decay) * p - lr * s * o.reshape(p.shape), m, lr * s * float(o.norm())


MIXED = [(68, 68), (87, 32), (5, 4), (1, 9), (128, 1024), (48, 1, 7, 7), (96, 48, 3, 3), (200, 150), (68, 128), (300, 10)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("nesterov,scale,decay", [(True, "shape", 0.1), (False, "rms", 0.0), (True, None, 0.01)])
def test_step_over_mixed_shapes(dtype, nesterov, scale, decay):
    lr, mu = 0.03, 0.9
    p = [gaussian(*s, seed=i, dtype=dtype) for i, s in enumerate(MIXED)]
    g = [gaussian(*s, seed=50 + i, dtype=dtype) for i, s in enumerate(MIXED)]
    m = [2 * gaussian(*s, seed=90 + i) for i, s in enumerate(MIXED)]
    dp, dg, dm = ([t.to(DEV) for t in ts] for ts in (p, g, m))
    for _ in range(2):                                     # the second step starts from the first one's momentum
        before = [(a.cpu(), b.cpu()) for a, b in zip(dp, dm)]
        ops.muon_step(dp, dg, dm, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay, scale=scale)
        for i, (p0, m0) in enumerate(before):
            want_p, want_m, size = step64(p0, g[i], m0, lr, mu, nesterov, decay, scale)
            # momentum: one product and one sum in fp32
            bound = 2.0 ** -23 * (mu * m0.double().abs() + g[i].double().abs())
            assert bool(((dm[i].double().cpu() - want_m).abs() <= bound).all()), MIXED[i]
            half = 2.0 ** -23 if dtype == torch.float32 else 2.0 ** -8
            err = float((dp[i].double().cpu() - want_p).norm())
            # the products' error is a share of the update alone; the rounding a share of the parameter
            assert err <= half * float(want_p.norm()) + TOL[dtype] * size, MIXED[i]
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dg, g))


def test_more_matrices_than_a_launch_holds():
    shapes = [(20 + i % 7, 30) for i in range(40)] + [(140, 40 + i) for i in range(36)]
    p = [gaussian(*s, seed=i).to(DEV) for i, s in enumerate(shapes)]
    g = [gaussian(*s, seed=200 + i).to(DEV) for i, s in enumerate(shapes)]
    m = [torch.zeros(s, device=DEV) for s in shapes]
    ops.muon_step(p, g, m, lr=0.1, momentum=0.5)
    for i, s in enumerate(shapes):
        want, _, size = step64(gaussian(*s, seed=i), g[i].cpu(), torch.zeros(s), 0.1, 0.5, True, 0.0, "shape")
        assert float((p[i].double().cpu() - want).norm()) <= 2.0 ** -23 * float(want.norm()) + TOL[torch.float32] * size, (i, s)


def test_single_product_arithmetic_and_its_name():
    x = gaussian(300, 500, seed=12)
    assert off(ops.orthogonalize(x.to(DEV), arithmetic="f16"), exact(x)) <= 9 * 2.0 ** -11 / math.sqrt(3)
    b = gaussian(300, 500, seed=12, dtype=torch.bfloat16)
    assert off(ops.orthogonalize(b.to(DEV), arithmetic="f16x2"), exact(b)) <= 2.0 ** -8 + TOL[torch.float32]


# ---- streams, graphs --------------------------------------------------------------------------------------------------
def test_on_another_stream():
    x, big = gaussian(500, 700, seed=13).to(DEV), gaussian(70, 70, seed=14).to(DEV)
    want = [ops.orthogonalize(x), ops.orthogonalize(big)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [ops.orthogonalize(x), ops.orthogonalize(big)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_calls_at_once_do_not_share_scratch():
    xs = [gaussian(400, 900, seed=15 + i).to(DEV) for i in range(2)]
    want = [ops.orthogonalize(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = ops.orthogonalize(xs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_step_replays():
    shapes = [(68, 68), (150, 300), (5, 4)]
    make = lambda seed: [gaussian(*s, seed=seed + i).to(DEV) for i, s in enumerate(shapes)]  # noqa: E731
    p, g, m = make(0), make(10), [torch.zeros(s, device=DEV) for s in shapes]
    args = dict(lr=0.05, weight_decay=0.1)
    ops.muon_step(make(0), g, [t.clone() for t in m], **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_step(p, g, m, **args)
    ep, em = [t.clone() for t in p], [t.clone() for t in m]
    for k in range(4):
        new = make(20 + 10 * k)
        for a, b in zip(g, new):
            a.copy_(b)
        graph.replay()
        ops.muon_step(ep, new, em, **args)                  # the program's own work in between
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(p + m, ep + em)), k


# ---- the trainer ------------------------------------------------------------------------------------------------------
def mixture(symmetric=True, n=68):
    torch.manual_seed(7)
    model = M.MDNGateVAE(R=3, n_nodes=n, k=6, n_layers=2, latent_dim=12, n_traits=4, symmetric_input=symmetric).to(DEV)
    gen = torch.Generator().manual_seed(1)
    adjacency = [[int(v) for v in torch.randperm(n, generator=gen)[:6]] for _ in range(n)]
    x = M.data.synthetic_sc(24, n, seed=3, device=DEV)
    traits = torch.randn(24, 4, generator=gen).to(DEV)
    eps = torch.randn(24, 12, generator=gen).to(DEV)
    return model, (x, adjacency, traits), x, eps


@pytest.mark.parametrize("symmetric", [True, False])
def test_trainer_step_is_backward_then_muon_and_adam(symmetric):
    model, inputs, x, eps = mixture(symmetric)
    trainer = M.Trainer(model, "mdn", optimizer="muon", muon_lr=0.01, muon_weight_decay=0.1)
    before = {k: v.detach().clone() for k, v in model.named_parameters()}
    trainer.step(inputs, x, eps=eps)
    grads = {k: v.grad.detach().cpu() for k, v in model.named_parameters()}
    for k, v in model.named_parameters():
        if v.dim() >= 2:
            want, _, size = step64(before[k].cpu(), grads[k], torch.zeros(v.shape), 0.01, 0.95, True, 0.1, "shape")
            assert float((v.detach().double().cpu() - want).norm()) <= 2.0 ** -23 * float(want.norm()) + TOL[torch.float32] * size, k
        else:
            # Adam's first step: lr g / (|g| + eps)
            g = grads[k].double()
            want = before[k].double().cpu() - 1e-3 * g / (g.abs() + 1e-8)
            assert float((v.detach().double().cpu() - want).abs().max()) <= 1e-3 * 2.0 ** -20 + 2.0 ** -23 * float(want.abs().max()), k


def test_trainer_captured_muon_steps_equal_eager_ones():
    model, inputs, x, eps = mixture()
    other, _, _, _ = mixture()
    eager = M.Trainer(other, "mdn", optimizer="muon", gate_balance=0.1)
    graph = M.Trainer(model, "mdn", optimizer="muon", gate_balance=0.1)
    graph.capture(inputs, x, eps)
    for k in range(3):
        e = eps + 0.1 * k
        a, b = float(graph.replay(inputs, x, e)), float(eager.step(inputs, x, eps=e))
        assert a == pytest.approx(b, rel=1e-6)
        torch.cuda.synchronize()
        # sums of gradients through atomics aside the two run the same kernels
        assert float((graph.buf.flat_p - eager.buf.flat_p).norm()) <= 1e-5 * float(eager.buf.flat_p.norm())


def test_trainer_refuses_what_it_does_not_know():
    model, _, _, _ = mixture()
    with pytest.raises(ValueError, match="optimizer"):
        M.Trainer(model, "mdn", optimizer="sgd")
    with pytest.raises(ValueError, match="gate_balance"):
        M.Trainer(model, "mse", gate_balance=0.1)
    with pytest.raises(ValueError, match="fewer than two"):
        M.Trainer(model, "mdn", optimizer="muon", muon_params=lambda name, p: True)


def test_trainer_leaves_chosen_parameters_to_adam():
    model, inputs, x, eps = mixture()
    trainer = M.Trainer(model, "mdn", optimizer="muon", muon_params=lambda name, p: name == "fc111.weight")
    trainer.step(inputs, x, eps=eps)
    assert trainer.muon_buf.numel() == model.fc111.weight.numel() and float(trainer.muon_buf.norm()) > 0
    assert float(trainer.exp_avg[:trainer.muon_buf.numel()].norm()) == 0


def test_refusals():
    x = torch.zeros(6, 8, device=DEV)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.orthogonalize(x.t())
    with pytest.raises(RuntimeError, match="two dimensions"):
        ops.orthogonalize(x[0])
    with pytest.raises(RuntimeError, match="dtype"):
        ops.orthogonalize(x.half())
    with pytest.raises(RuntimeError, match="out"):
        ops.orthogonalize(x, out=torch.zeros(8, 6, device=DEV))
    with pytest.raises(RuntimeError, match="dtype"):
        ops.orthogonalize(x, out=x.bfloat16())
    with pytest.raises(RuntimeError, match="steps"):
        ops.orthogonalize(x, steps=0)
    with pytest.raises(RuntimeError, match="eps"):
        ops.orthogonalize(x, eps=0.0)
    with pytest.raises(RuntimeError, match="leave"):
        ops.orthogonalize(x, coefficients=(30.0, 0.0, 0.0))
    with pytest.raises(ValueError, match="arithmetic"):
        ops.orthogonalize(x, arithmetic="bf16")
    p, g, m = (torch.zeros(4, 6, device=DEV) for _ in range(3))
    for bad, match in [(([p], [g], []), "momenta"), (([p, p], [g, g], [m, m.clone()]), "overlaps"), (([p], [p], [m]), "overlaps"),
                       (([p], [g], [p]), "overlaps"), (([p], [None], [m]), "missing"), (([p], [g.t()], [m]), "contiguous"),
                       (([p], [g[:2]], [m]), "shape"), (([p[0]], [g[0]], [m[0]]), "two dimensions"),
                       (([p], [g.bfloat16()], [m]), "dtype"), (([p], [g], [m.bfloat16()]), "dtype"), (([p], [g.cpu()], [m]), "cpu")]:
        with pytest.raises((RuntimeError, TypeError), match=match):
            ops.muon_step(*bad, lr=0.1)
    with pytest.raises(RuntimeError, match="momentum"):
        ops.muon_step([p], [g], [m], lr=0.1, momentum=1.0)
    with pytest.raises(RuntimeError, match="finite"):
        ops.muon_step([p], [g], [m], lr=math.nan)
    with pytest.raises(ValueError, match="scale"):
        ops.muon_step([p], [g], [m], lr=0.1, scale="l2")
    flat = torch.zeros(60, device=DEV)
    with pytest.raises(RuntimeError, match="overlaps"):     # views that share their middle
        ops.muon_step([flat[:24].view(4, 6), flat[20:44].view(4, 6)], [g, g], [m, torch.zeros(4, 6, device=DEV)], lr=0.1)
    assert bool((p == 0).all()) and bool((m == 0).all())


def test_out_that_overlaps_x_is_refused():
    buf = gaussian(3, 150, 150).to(DEV)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.orthogonalize(buf[:2], out=buf[1:])
    want = ops.orthogonalize(buf[:1])
    assert torch.equal(ops.orthogonalize(buf[:1], out=buf[1:2]), want)


def test_step_between_forward_and_backward_is_noticed():
    p, m = gaussian(40, 30).to(DEV).requires_grad_(True), torch.zeros(40, 30, device=DEV)
    loss = (p * p).sum()
    ops.muon_step([p], [torch.ones_like(p)], [m], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_result_over_a_saved_tensor_is_noticed():
    x = gaussian(40, 30).to(DEV).requires_grad_(True)
    y = x * 2.0
    loss = (y * y).sum()
    ops.orthogonalize(y, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
