"""Balance loss of a gate (ops.gate_balance_loss*, Trainer(gate_balance=...)) against the definition in float64.

Tolerances.  Probabilities carry about eight fp32 roundings (difference, exponential, sum, quotient), their means as many
again spread over the rows, so 16 * 2^-24 = 1e-6 relative to the largest; the loss is one sum of those.  The gradient
p (w - sum p w) adds the cancellation of w against its mean, at most sum |p w| <= max |w|: 16 * 2^-24 of max |w|, plus the
rounding of its type (half a step: 2^-8 of the value in bf16)."""
import math

import pytest
import torch

import mdnvae_amd as M
from mdnvae_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 16 * 2.0 ** -24


def definition(logits, top_k, valid=None, g_loss=1.0, g_mean=None):
    """(loss, counts, mean_probs, grad, max |w|) in float64 on the CPU."""
    z = logits.double().cpu()
    T, E = z.shape
    rows = torch.ones(T, dtype=torch.bool) if valid is None else valid.cpu()
    rows = rows & ~(z == -math.inf).all(dim=1)
    z = z[rows]
    n = z.shape[0]
    if n == 0:
        return 0.0, torch.zeros(E, dtype=torch.int32), torch.zeros(E).double(), torch.zeros(T, E).double(), 0.0
    p = torch.softmax(z, dim=1)
    order = torch.sort(torch.where(torch.isnan(z), torch.full_like(z, math.inf), z), dim=1, descending=True, stable=True).indices[:, :top_k]
    if torch.isnan(z).any():                                # NaN counts as the largest number
        key = torch.where(torch.isnan(z), torch.tensor(2.0), torch.where(z == math.inf, torch.tensor(1.0), torch.tensor(0.0)))
        order = torch.stack([torch.tensor(sorted(range(E), key=lambda e: (-float(key[t, e]), -float(z[t, e]) if key[t, e] == 0 else 0.0, e))[:top_k])
                             for t in range(n)])
    taken = torch.zeros(n, E, dtype=torch.bool).scatter_(1, order, True) & (z != -math.inf)
    counts = taken.sum(dim=0)
    mean = p.sum(dim=0) / n
    w = g_loss * E / (top_k * n * n) * counts.double()
    w = w - w.mean() + (0.0 if g_mean is None else g_mean.double().cpu() / n)
    grad = torch.zeros(T, E).double()
    grad[rows] = p * (w - (p * w).sum(dim=1, keepdim=True))
    loss = float(E / (top_k * n) * (counts.double() * mean).sum())
    return loss, counts.to(torch.int32), mean, grad, float(w.abs().max())


def check(logits, top_k, valid=None):
    loss, counts, mean, grad = ops.gate_balance_loss_and_grads(logits, top_k, valid)
    want_loss, want_counts, want_mean, want_grad, w = definition(logits, top_k, valid)
    assert loss.dtype == mean.dtype == torch.float32 and counts.dtype == torch.int32 and grad.dtype == logits.dtype
    assert torch.equal(counts.cpu(), want_counts)
    assert float((mean.double().cpu() - want_mean).abs().max()) <= EPS * max(float(want_mean.max()), 1e-30)
    assert abs(float(loss) - want_loss) <= 2 * EPS * abs(want_loss)
    half = 0.0 if logits.dtype == torch.float32 else 2.0 ** -8
    # below bf16's (and fp32's) smallest normal number a value may vanish
    assert bool(((grad.double().cpu() - want_grad).abs() <= half * want_grad.abs() + EPS * w + 2.0 ** -126).all())
    return loss, counts, mean, grad


def logits_of(T, E, dtype=torch.float32, seed=0, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(T, E, generator=g) + torch.randn(E, generator=g)).to(dtype).to(DEV)


# rows and experts on both sides of every lane layout, of the one-workgroup limit and of the fused sum
CASES = [(1, 1, 1), (1, 5, 2), (3, 2, 2), (7, 8, 3), (64, 9, 1), (65, 16, 16), (256, 5, 1), (300, 17, 4), (1000, 32, 5), (777, 33, 2),
         (513, 64, 6), (400, 65, 6), (500, 127, 7), (600, 128, 9), (100, 129, 3), (511, 256, 8), (520, 257, 10), (130, 511, 2),
         (140, 513, 20), (90, 1000, 1), (64, 1024, 64), (8192, 5, 1), (8193, 5, 2), (16384, 5, 1), (9001, 60, 6), (20000, 200, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,E,k", CASES)
def test_against_the_definition(T, E, k, dtype):
    check(logits_of(T, E, dtype, seed=T + E), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,E,k", [(1, 3, 1), (300, 17, 4), (9001, 60, 6), (12000, 5, 1), (700, 256, 8)])
def test_padded_rows(T, E, k, dtype):
    z = logits_of(T, E, dtype, seed=1)
    valid = torch.rand(T, generator=torch.Generator().manual_seed(2)) < 0.7
    valid[T - T // 5:] = False
    valid = valid.to(DEV)
    clean = check(z, k, valid)
    for junk in (math.nan, math.inf, -math.inf, 3e38):       # what padding holds is never looked at
        dirty = z.clone()
        dirty[~valid] = junk
        got = ops.gate_balance_loss_and_grads(dirty, k, valid)
        assert all(torch.equal(a, b) for a, b in zip(got, clean))
    assert bool((clean[3][~valid] == 0).all())


@pytest.mark.parametrize("T", [1, 50, 30000])
def test_no_valid_row(T):
    z = logits_of(T, 6)
    for got in (ops.gate_balance_loss_and_grads(z, 2, torch.zeros(T, dtype=torch.bool, device=DEV)),
                ops.gate_balance_loss_and_grads(torch.full_like(z, -math.inf), 2)):
        assert all(bool((t == 0).all()) for t in got)


def test_no_rows():
    loss, counts, mean, grad = ops.gate_balance_loss_and_grads(torch.empty(0, 7, device=DEV), 2)
    assert float(loss) == 0 and int(counts.sum()) == 0 and float(mean.sum()) == 0 and grad.shape == (0, 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,E,k", [(200, 5, 3), (300, 60, 6), (200, 250, 8), (12000, 12, 4)])
def test_masked_experts(T, E, k, dtype):
    """-inf takes an expert out of a row: never counted, even where fewer than top_k are left; the type's lowest number is a
    number like any other."""
    z = logits_of(T, E, dtype, seed=3)
    g = torch.Generator().manual_seed(4)
    drop = torch.rand(T, E, generator=g) < 0.6
    drop[0] = True
    drop[0, E - 1] = False                                   # one left
    drop[1] = True                                           # none left: the row is not valid
    out = z.masked_fill(drop.to(DEV), -math.inf)
    _, counts, _, grad = check(out, k)
    assert bool((grad[drop.to(DEV)] == 0).all())
    assert int(counts.sum()) == int((~drop).sum(dim=1).clamp(max=k).sum())
    low = z.masked_fill(drop.to(DEV), torch.finfo(dtype).min)
    _, counts, _, _ = check(low, k)
    assert int(counts.sum()) == T * k


@pytest.mark.parametrize("E,k", [(5, 1), (5, 3), (8, 8), (60, 6), (64, 7), (256, 8), (256, 1), (1024, 12)])
def test_ties_go_to_the_lowest_index(E, k):
    g = torch.Generator().manual_seed(5)
    z = torch.randint(0, 3, (400, E), generator=g).float()
    z[0] = 1.0
    z[1] = -0.0
    z[1, ::2] = 0.0                                          # -0 and +0 are the same number
    for dtype in (torch.float32, torch.bfloat16):
        check(z.to(dtype).to(DEV), k)


@pytest.mark.parametrize("scale", [0.0, 1e-3, 50.0, 1e4, 1e30])
def test_range_of_the_logits(scale):
    check(logits_of(500, 40, seed=6, scale=scale), 4)
    check(logits_of(500, 5, seed=6, scale=scale), 1)


@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=str)
@pytest.mark.parametrize("T", [40, 20000])
def test_nan_and_infinity_show_and_stay_in_their_row(bad, T):
    z = logits_of(T, 6, seed=7)
    z[5, 2] = bad
    if math.isnan(bad):
        z[6] = torch.tensor([math.nan, 1.0, -math.nan, 9.0, math.inf, 2.0], device=DEV)
    loss, counts, mean, grad = ops.gate_balance_loss_and_grads(z, 2)
    bad_rows = [5, 6] if math.isnan(bad) else [5]
    assert math.isnan(float(loss)) and bool(torch.isnan(mean).all())
    assert bool(torch.isnan(grad[bad_rows]).all())
    rest = torch.ones(T, dtype=torch.bool, device=DEV)
    rest[bad_rows] = False
    assert bool(torch.isfinite(grad[rest]).all())
    assert torch.equal(counts.cpu(), definition(z, 2)[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,E", [(100, 60), (9000, 60), (300, 256)])
def test_unaligned_storage(T, E, dtype):
    z = logits_of(T, E, dtype, seed=8)
    buf = torch.zeros(T * E + 9, dtype=dtype, device=DEV)
    view = buf[1:1 + T * E].view(T, E)
    view.copy_(z)
    _, counts, mean, grad = check(view, 5)
    _, counts2, mean2, grad2 = check(z, 5)
    assert torch.equal(counts, counts2)                      # the lanes hold other experts: sums of p may round otherwise


def test_same_call_same_bits():
    z = logits_of(50000, 60, seed=9)
    a, b = ops.gate_balance_loss_and_grads(z, 6), ops.gate_balance_loss_and_grads(z, 6)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_rows_past_32_bit_offsets():
    E, T = 256, (1 << 31) // 256 + 1000
    z = torch.zeros(T, E, dtype=torch.bfloat16, device=DEV)
    tail = logits_of(1000, E, torch.bfloat16, seed=10)
    z[-1000:] = tail
    valid = torch.zeros(T, dtype=torch.bool, device=DEV)
    valid[-1000:] = True
    loss, counts, mean, grad = ops.gate_balance_loss_and_grads(z, 8, valid)
    want_loss, want_counts, want_mean, want_grad, w = definition(tail, 8)
    assert torch.equal(counts.cpu(), want_counts) and abs(float(loss) - want_loss) <= 2 * EPS * want_loss
    assert bool(((grad[-1000:].double().cpu() - want_grad).abs() <= 2.0 ** -8 * want_grad.abs() + EPS * w).all())
    assert bool((grad[:1000] == 0).all())


# ---- autograd ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,E,k", [(40, 5, 1), (12000, 5, 2), (700, 60, 6), (300, 256, 8)])
def test_backward_with_upstream_gradients(T, E, k, dtype):
    z = logits_of(T, E, dtype, seed=11).requires_grad_(True)
    valid = (torch.rand(T, generator=torch.Generator().manual_seed(12)) < 0.8).to(DEV)
    g_mean = torch.randn(E, generator=torch.Generator().manual_seed(13))
    half = 0.0 if dtype == torch.float32 else 2.0 ** -8
    for a, b in ((1.0, 0.0), (2.5, 1.0), (0.0, 1.0)):
        loss, counts, mean = ops.gate_balance_loss(z, k, valid)
        assert not counts.requires_grad
        total = (a * loss if a else 0.0) + (b * (mean * g_mean.to(DEV)).sum() if b else 0.0)
        (got,) = torch.autograd.grad(total, z)
        _, _, _, want, w = definition(z.detach(), k, valid, a, b * g_mean if b else None)
        assert bool(((got.double().cpu() - want).abs() <= half * want.abs() + 2 * EPS * w + 2.0 ** -126).all()), (a, b)


def test_gradient_against_differences():
    """Central differences of the kernel's own loss, logits far enough apart that no selection changes within h."""
    T, E, k, h = 6, 5, 2, 2.0 ** -5
    z = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t)).float() * 0.5 for t in range(T)]).to(DEV)
    _, _, _, grad = ops.gate_balance_loss_and_grads(z, k)
    worst = 0.0
    for t in range(T):
        for e in range(E):
            up, down = z.clone(), z.clone()
            up[t, e] += h
            down[t, e] -= h
            d = (float(ops.gate_balance_loss(up, k)[0]) - float(ops.gate_balance_loss(down, k)[0])) / (2 * h)
            worst = max(worst, abs(d - float(grad[t, e])))
    # a third derivative of at most max |w| (the loss is a sum of p w) times h^2 / 6, and two fp32 losses of about one over 2 h
    w = E / (k * T * T) * T
    assert worst <= w * h * h / 6 + 2 * 2.0 ** -23 / (2 * h)


def test_captured_forward_and_backward_replay_beside_eager_work():
    for T, E, k in ((200, 5, 1), (20000, 12, 3), (3000, 60, 6)):
        z = logits_of(T, E, seed=14)
        out = ops.gate_balance_loss_and_grads(z, k)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.gate_balance_loss_and_grads(z, k)
        for r in range(4):
            z.copy_(logits_of(T, E, seed=20 + r))
            graph.replay()
            want = ops.gate_balance_loss_and_grads(z.clone(), k)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), (T, r)


def test_on_another_stream():
    z = logits_of(30000, 60, seed=15)
    want = ops.gate_balance_loss_and_grads(z, 6)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.gate_balance_loss_and_grads(z, 6)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- the mixture model and its trainer ------------------------------------------------------------------------------------
def mixture():
    torch.manual_seed(7)
    n = 68
    model = M.MDNGateVAE(R=3, n_nodes=n, k=6, n_layers=2, latent_dim=12, n_traits=4, symmetric_input=True).to(DEV)
    gen = torch.Generator().manual_seed(1)
    adjacency = [[int(v) for v in torch.randperm(n, generator=gen)[:6]] for _ in range(n)]
    x = M.data.synthetic_sc(24, n, seed=3, device=DEV)
    return model, (x, adjacency, torch.randn(24, 4, generator=gen).to(DEV)), x, torch.randn(24, 12, generator=gen).to(DEV)


@pytest.mark.parametrize("fused", [True, False])
def test_trainer_adds_the_balance_term(fused):
    grads, losses = [], []
    for weight in (0.0, 0.5):
        model, inputs, x, eps = mixture()
        trainer = M.Trainer(model, "mdn", gate_balance=weight, gate_top_k=2, fused_loss=fused)
        losses.append(float(trainer.forward_backward(inputs, x, eps)))
        grads.append(model.gate.weight.grad.double().cpu())
    logits = model.gate(inputs[2]).detach()
    want_loss, counts, _, want_grad, _ = definition(logits, 2)
    assert torch.equal(trainer.gate_counts.cpu(), counts)
    weight = 0.5 * 24
    assert abs(losses[1] - losses[0] - weight * want_loss) <= 1e-6 * abs(losses[0])           # fp32 losses of that size
    want = weight * want_grad.t() @ inputs[2].double().cpu()
    # the difference of two fp32 gradients of the gate's weight
    assert float((grads[1] - grads[0] - want).abs().max()) <= 1e-5 * float(grads[0].abs().max()) + 1e-5 * float(want.abs().max())


def test_model_method():
    model, inputs, _, _ = mixture()
    loss, counts, mean = model.gate_balance(model.gate(inputs[2]), top_k=1)
    loss.backward()
    assert int(counts.sum()) == 24 and float(mean.sum()) == pytest.approx(1.0, abs=1e-5)
    assert model.gate.weight.grad is not None and bool(torch.isfinite(model.gate.weight.grad).all())


def test_refusals():
    z = logits_of(8, 6)
    for bad, match in [((z.t(),), "contiguous"), ((z[0],), "rows, experts"), ((z.double(),), "dtype"), ((z, 0), "top_k"), ((z, 7), "top_k"),
                       ((z, 1, torch.ones(7, dtype=torch.bool, device=DEV)), "valid"), ((z, 1, torch.ones(8, device=DEV)), "dtype"),
                       ((z, 1, torch.ones(8, dtype=torch.bool)), "valid"), ((torch.zeros(4, 1025, device=DEV),), "experts"),
                       ((torch.zeros(4, 0, device=DEV),), "experts")]:
        for f in (ops.gate_balance_loss, ops.gate_balance_loss_and_grads):
            with pytest.raises(RuntimeError, match=match):
                f(*bad)


def test_second_derivatives_are_refused():
    x = torch.randn(40, 6, device=DEV, requires_grad=True)
    loss, _, _ = ops.gate_balance_loss(x, 2)
    (g,) = torch.autograd.grad(loss, x, create_graph=True)
    assert torch.equal(g.detach(), ops.gate_balance_loss_and_grads(x, 2)[3])
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(g.square().sum(), x)
