"""CPU checks of the orthogonalised updates' and the gate balance loss's boundary: what they refuse, they refuse before
anything touches a device, and the C entry points check their arguments themselves."""
import ctypes

import pytest
import torch

import mdnvae_amd as M
from mdnvae_amd import _lib, ops

COEF = (3.4445, -4.775, 2.0315)


def ortho(lib, x=1, out=1, batch=1, rows=4, cols=4, dtype=0, steps=5, coef=COEF, eps=1e-7, terms=3, ws=None, size=0):
    return lib.mdnvae_orthogonalize(x, out, batch, rows, cols, dtype, steps, *coef, eps, terms, ws, size, None)


def test_orthogonalize_arguments_need_no_gpu():
    lib = _lib.load()
    for kw, text in [(dict(dtype=2), b"element type"), (dict(steps=0), b"steps"), (dict(steps=17), b"steps"), (dict(eps=0.0), b"eps"),
                     (dict(eps=float("nan")), b"eps"), (dict(terms=2), b"terms"), (dict(coef=(float("inf"), 0, 0)), b"finite"),
                     (dict(coef=(300.0, 0.0, 0.0)), b"leave"), (dict(coef=(5.0, 5.0, 5.0)), b"leave"), (dict(rows=-1), b"negative"),
                     (dict(x=None), b"null"), (dict(out=None), b"null"), (dict(rows=70000, cols=70000), b"larger"),
                     (dict(rows=1, cols=1 << 25), b"larger"), (dict(rows=300, cols=300), b"workspace"),
                     (dict(rows=300, cols=300, ws=8, size=1 << 40), b"aligned")]:
        assert ortho(lib, **kw) < 0, kw
        assert text in lib.mdnvae_last_error(), (kw, lib.mdnvae_last_error())
    for kw in (dict(batch=0), dict(rows=0), dict(cols=0)):
        assert ortho(lib, **kw) == 0


def test_orthogonalize_refuses_an_output_that_overlaps_its_input():
    lib = _lib.load()
    # a batch of two: the first result would land on the second matrix before that is read
    for x, out in [(4096, 4100), (4096, 4096 + 64), (4100, 4096), (4096, 4096 + 127)]:
        assert ortho(lib, x=x, out=out, batch=2) < 0
        assert b"overlaps" in lib.mdnvae_last_error()
    # apart, and the same memory: the next check's turn
    for x, out in [(4096, 4096 + 2 * 300 * 300 * 4), (4096, 4096)]:
        assert ortho(lib, x=x, out=out, batch=2, rows=300, cols=300) < 0
        assert b"workspace" in lib.mdnvae_last_error()


def test_workspace_of_small_matrices_is_none_and_of_batches_bounded():
    lib = _lib.load()
    for rows, cols in [(1, 1), (128, 128), (128, 68), (1184, 32), (64, 512)]:
        assert lib.mdnvae_orthogonalize_workspace_bytes(10000, rows, cols) == 0
    one = lib.mdnvae_orthogonalize_workspace_bytes(1, 512, 512)
    assert one >= 8 * 512 * 512 * 2
    assert lib.mdnvae_orthogonalize_workspace_bytes(100000, 512, 512) <= 3 << 30
    assert lib.mdnvae_orthogonalize_workspace_bytes(1, 70000, 70000) == 0
    rows, cols = (ctypes.c_long * 3)(68, 1024, 4), (ctypes.c_long * 3)(68, 7569, 5)
    assert lib.mdnvae_muon_workspace_bytes(rows, cols, 3) >= 8 * 1024 * 7569
    assert lib.mdnvae_muon_workspace_bytes(rows, cols, 1) == 0


def muon(lib, n=1, rows=4, cols=4, params=(4096,), grads=(8192,), momenta=(16384,), lr=0.1, momentum=0.9, decay=0.0, scale=1, dtype=0):
    arr = lambda v: (ctypes.c_void_p * max(len(v), 1))(*v)  # noqa: E731
    r, c = (ctypes.c_long * max(n, 1))(*[rows] * n), (ctypes.c_long * max(n, 1))(*[cols] * n)
    return lib.mdnvae_muon_step(arr(params), arr(grads), arr(momenta), r, c, n, dtype, lr, momentum, 1, decay, scale, 5, *COEF, 1e-7, 3, None,
                                0, None)


def test_muon_step_arguments_need_no_gpu():
    lib = _lib.load()
    nan = float("nan")
    for kw, text in [(dict(n=-1), b"count"), (dict(lr=nan), b"finite"), (dict(decay=nan), b"finite"), (dict(momentum=1.0), b"momentum"),
                     (dict(momentum=-0.1), b"momentum"), (dict(momentum=nan), b"momentum"), (dict(scale=3), b"scale"), (dict(dtype=5), b"element"),
                     (dict(rows=-4), b"negative"), (dict(params=(None,)), b"null"), (dict(grads=(None,)), b"null"),
                     (dict(momenta=(None,)), b"null"), (dict(grads=(4096,)), b"overlaps"), (dict(momenta=(4100,)), b"overlaps"),
                     (dict(n=2, params=(4096, 4096 + 60), grads=(8192, 8192), momenta=(16384, 32768)), b"overlaps"),
                     (dict(rows=300, cols=300, params=(1 << 20,), grads=(2 << 20,), momenta=(4 << 20,)), b"workspace")]:
        assert muon(lib, **kw) < 0, kw
        assert text in lib.mdnvae_last_error(), (kw, lib.mdnvae_last_error())
    assert muon(lib, n=0) == 0 and muon(lib, rows=0) == 0


def test_gate_balance_arguments_need_no_gpu():
    lib = _lib.load()

    def gate(logits=1, T=4, E=5, k=1, dtype=0, ws=None, size=0, loss=1, counts=1, mean=1):
        return lib.mdnvae_gate_balance(logits, None, T, E, k, dtype, ws, size, loss, counts, mean, None, None, None)

    for kw, text in [(dict(dtype=3), b"element"), (dict(T=-1), b"rows"), (dict(T=1 << 31), b"rows"), (dict(E=0), b"experts"),
                     (dict(E=1025), b"experts"), (dict(k=0), b"top_k"), (dict(k=6), b"top_k"), (dict(logits=None), b"null"),
                     (dict(loss=None), b"null"), (dict(counts=None), b"null"), (dict(mean=None), b"null"), (dict(T=100000), b"workspace"),
                     (dict(T=100000, ws=2, size=1 << 30), b"aligned")]:
        assert gate(**kw) < 0, kw
        assert text in lib.mdnvae_last_error(), (kw, lib.mdnvae_last_error())
    assert lib.mdnvae_gate_balance_bwd(1, None, 4, 5, 1, 0, None, 1, 1, None, None, 1, None) < 0 and b"null" in lib.mdnvae_last_error()
    assert lib.mdnvae_gate_balance_bwd(1, None, 4, 5, 9, 0, 1, 1, 1, None, None, 1, None) < 0 and b"top_k" in lib.mdnvae_last_error()
    assert lib.mdnvae_gate_balance_workspace_bytes(256, 5) == 0
    assert lib.mdnvae_gate_balance_workspace_bytes(1 << 20, 1024) <= 16 << 20


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        M.orthogonalize(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        M.muon_step([x], [x.clone()], [x.clone()], lr=0.1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        M.gate_balance_loss(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        M.gate_balance_loss_and_grads(x)


def test_wrappers_check_types_and_names():
    x = torch.zeros(4, 4)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.orthogonalize([[1.0]])
    with pytest.raises(RuntimeError, match="dtype"):
        ops.orthogonalize(x.half())
    with pytest.raises(ValueError, match="scale"):
        ops.muon_step([x], [x], [x], lr=0.1, scale="norm")
    with pytest.raises(RuntimeError, match="gradients"):
        ops.muon_step([x], [], [x], lr=0.1)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.gate_balance_loss_and_grads(None)
    with pytest.raises(RuntimeError, match="rows, experts"):
        ops.gate_balance_loss(torch.zeros(3))
