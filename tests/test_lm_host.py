"""Refusals of layer norm, lookup and distillation, and what their ops say of shapes (no GPU)."""
import ctypes

import pytest
import torch

import flexsae_amd as flex
from flexsae_amd import _lib

FAKE = 0x10000  # never dereferenced: validation fails first


def _norm(rows=4, cols=8, x_stride=8, dy_stride=8, eps=1e-5, dtype=0, weight_dtype=0, bias_dtype=0):
    return ctypes.byref(_lib.Norm(rows, cols, x_stride, dy_stride, eps, dtype, weight_dtype, bias_dtype))


def _lookup(n=4, vocab=10, cols=8, weight_stride=8, dout_stride=8, factor=1.0, dtype=0, scale_dtype=0):
    return ctypes.byref(_lib.Lookup(n, vocab, cols, weight_stride, dout_stride, factor, dtype, scale_dtype))


def _distill(rows=4, vocab=10, k=3, logits_stride=10, temperature=1.0, dtype=0, top_dtype=0, flags=0):
    return ctypes.byref(_lib.Distill(rows, vocab, k, logits_stride, temperature, dtype, top_dtype, flags))


BAD = _lib.ERR_INVALID_ARGUMENT
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), BAD), (dict(cols=0), BAD), (dict(eps=-1.0), BAD), (dict(eps=NAN), BAD), (dict(eps=INF), BAD), (dict(dtype=3), BAD),
    (dict(weight_dtype=-1), BAD), (dict(x_stride=-1), BAD), (dict(rows=1 << 33), _lib.ERR_UNSUPPORTED), (dict(cols=1 << 30), _lib.ERR_UNSUPPORTED)])
def test_norm_refuses(change, status):
    lib = _lib.load()
    assert lib.flexsae_layer_norm_fwd(_norm(**change), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == status
    assert lib.flexsae_layer_norm_bwd(_norm(**change), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None) == status
    assert lib.flexsae_layer_norm_bwd_workspace_bytes(_norm(**change)) == 0


def test_norm_refuses_pointers():
    lib = _lib.load()
    assert lib.flexsae_layer_norm_fwd(None, FAKE, None, None, FAKE, None, None, None) == BAD
    for i in (0, 3):
        p = [FAKE] * 6
        p[i] = None
        assert lib.flexsae_layer_norm_fwd(_norm(), *p, None) == BAD
    for i in range(6):
        p = [FAKE] * 6
        p[i] = FAKE + 1
        assert lib.flexsae_layer_norm_fwd(_norm(), *p, None) == _lib.ERR_ALIGNMENT
    for i in (0, 1, 3, 4):
        p = [FAKE] * 8
        p[i] = None
        assert lib.flexsae_layer_norm_bwd(_norm(), *p, FAKE, 1 << 30, None) == BAD
    for i in range(8):
        p = [FAKE] * 8
        p[i] = FAKE + 1
        assert lib.flexsae_layer_norm_bwd(_norm(), *p, FAKE, 1 << 30, None) == _lib.ERR_ALIGNMENT
    for ws, n in ((None, 1 << 30), (FAKE + 16, 1 << 30), (FAKE, 8)):
        assert lib.flexsae_layer_norm_bwd(_norm(), *[FAKE] * 8, ws, n, None) == _lib.ERR_WORKSPACE
    # nothing to do
    assert lib.flexsae_layer_norm_fwd(_norm(rows=0), None, None, None, None, None, None, None) == _lib.OK
    assert lib.flexsae_layer_norm_bwd(_norm(), *[FAKE] * 5, None, None, None, None, 0, None) == _lib.OK


@pytest.mark.parametrize("change,status", [
    (dict(n=-1), BAD), (dict(vocab=0), BAD), (dict(cols=0), BAD), (dict(factor=NAN), BAD), (dict(factor=INF), BAD), (dict(dtype=7), BAD),
    (dict(scale_dtype=7), BAD), (dict(weight_stride=-1), BAD), (dict(dout_stride=-8), BAD), (dict(n=1 << 32), _lib.ERR_UNSUPPORTED),
    (dict(vocab=1 << 31), _lib.ERR_UNSUPPORTED), (dict(cols=1 << 29), _lib.ERR_UNSUPPORTED)])
def test_lookup_refuses(change, status):
    lib = _lib.load()
    assert lib.flexsae_lookup_fwd(_lookup(**change), FAKE, FAKE, FAKE, FAKE, None, None) == status
    assert lib.flexsae_lookup_bwd(_lookup(**change), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None) == status
    assert lib.flexsae_lookup_bwd_workspace_bytes(_lookup(**change)) == 0


def test_lookup_refuses_pointers():
    lib = _lib.load()
    for i in (0, 1, 3):
        p = [FAKE] * 4
        p[i] = None
        assert lib.flexsae_lookup_fwd(_lookup(), *p, None, None) == BAD
    for i in range(4):
        p = [FAKE] * 4
        p[i] = FAKE + 1
        assert lib.flexsae_lookup_fwd(_lookup(), *p, None, None) == _lib.ERR_ALIGNMENT
    for i in range(4):  # (weight and scale are needed for dscale)
        p = [FAKE] * 6
        p[i] = None
        assert lib.flexsae_lookup_bwd(_lookup(), *p, FAKE, 1 << 30, None) == BAD
    for i in range(6):
        p = [FAKE] * 6
        p[i] = FAKE + 1
        assert lib.flexsae_lookup_bwd(_lookup(), *p, FAKE, 1 << 30, None) == _lib.ERR_ALIGNMENT
    for ws, n in ((None, 1 << 30), (FAKE + 16, 1 << 30), (FAKE, 8)):
        assert lib.flexsae_lookup_bwd(_lookup(), *[FAKE] * 6, ws, n, None) == _lib.ERR_WORKSPACE
    assert lib.flexsae_lookup_fwd(_lookup(n=0), None, None, None, None, None, None) == _lib.OK
    assert lib.flexsae_lookup_bwd(_lookup(), *[FAKE] * 4, None, None, None, 0, None) == _lib.OK


@pytest.mark.parametrize("change,status", [
    (dict(rows=0), BAD), (dict(vocab=0), BAD), (dict(k=0), BAD), (dict(temperature=0.0), BAD), (dict(temperature=-1.0), BAD),
    (dict(temperature=NAN), BAD), (dict(temperature=INF), BAD), (dict(temperature=1e-39), BAD), (dict(temperature=1e30), BAD),
    (dict(dtype=9), BAD), (dict(top_dtype=9), BAD), (dict(flags=2), BAD), (dict(logits_stride=-1), BAD),
    (dict(rows=1 << 31), _lib.ERR_UNSUPPORTED), (dict(vocab=1 << 31), _lib.ERR_UNSUPPORTED)])
def test_distill_refuses(change, status):
    lib = _lib.load()
    assert lib.flexsae_distill_fwd(_distill(**change), *[FAKE] * 7, FAKE, 1 << 40, None, None) == status
    assert lib.flexsae_distill_bwd(_distill(**change), *[FAKE] * 6, 0, FAKE, None) == status
    assert lib.flexsae_distill_workspace_bytes(_distill(**change)) == 0


def test_distill_refuses_pointers():
    lib = _lib.load()
    for i in (0, 1, 2, 4, 5):
        p = [FAKE] * 7
        p[i] = None
        assert lib.flexsae_distill_fwd(_distill(), *p, FAKE, 1 << 30, None, None) == BAD
    for i in range(7):
        p = [FAKE] * 7
        p[i] = FAKE + 1
        assert lib.flexsae_distill_fwd(_distill(), *p, FAKE, 1 << 30, None, None) == _lib.ERR_ALIGNMENT
    for ws, n in ((None, 1 << 30), (FAKE + 16, 1 << 30), (FAKE, 8)):
        assert lib.flexsae_distill_fwd(_distill(), *[FAKE] * 7, ws, n, None, None) == _lib.ERR_WORKSPACE
    for i in (0, 1, 2, 4, 5):
        p = [FAKE] * 6
        p[i] = None
        assert lib.flexsae_distill_bwd(_distill(), *p, 0, FAKE, None) == BAD
    assert lib.flexsae_distill_bwd(_distill(), *[FAKE] * 6, 0, None, None) == BAD
    assert lib.flexsae_distill_bwd(_distill(flags=_lib.DISTILL_BY_ROW), *[FAKE] * 6, 1, FAKE, None) == BAD
    assert lib.flexsae_distill_bwd(_distill(), *[FAKE] * 6, 0, FAKE + 2, None) == _lib.ERR_ALIGNMENT


# ---- the public functions ------------------------------------------------------------------

X = torch.zeros(4, 8)


@pytest.mark.parametrize("call,error", [
    (lambda: flex.layer_norm(X), RuntimeError),
    (lambda: flex.layer_norm(X.double()), TypeError),
    (lambda: flex.layer_norm(torch.tensor(1.0)), ValueError),
    (lambda: flex.layer_norm(torch.zeros(4, 0)), ValueError),
    (lambda: flex.layer_norm(X, torch.ones(7)), ValueError),
    (lambda: flex.layer_norm(X, torch.ones(1, 8)), ValueError),
    (lambda: flex.layer_norm(X, torch.ones(8), torch.ones(8, dtype=torch.int32)), TypeError),
    (lambda: flex.layer_norm(X, eps=-1e-5), ValueError),
    (lambda: flex.layer_norm(X, eps=NAN), ValueError),
    (lambda: flex.layer_norm_stats(X), RuntimeError),
    (lambda: flex.embedding_lookup(torch.zeros(3, dtype=torch.int64), X), RuntimeError),
    (lambda: flex.embedding_lookup(torch.zeros(3), X), TypeError),
    (lambda: flex.embedding_lookup(torch.zeros(3, dtype=torch.int16), X), TypeError),
    (lambda: flex.embedding_lookup(torch.zeros(3, dtype=torch.int64), X.double()), TypeError),
    (lambda: flex.embedding_lookup(torch.zeros(3, dtype=torch.int64), X[0]), ValueError),
    (lambda: flex.embedding_lookup(torch.zeros(3, dtype=torch.int64), X[:0]), ValueError),
    (lambda: flex.embedding_lookup(torch.zeros(3, dtype=torch.int64), X, torch.ones(2)), RuntimeError),
    (lambda: flex.embedding_lookup(torch.zeros(3, dtype=torch.int64), X, torch.ones(3, dtype=torch.int64)), TypeError),
    (lambda: flex.embedding_lookup(torch.zeros(3, dtype=torch.int64), X, INF), ValueError),
    (lambda: flex.distillation_loss(X, X[:, :2], torch.zeros(4, 2, dtype=torch.int64)), RuntimeError),
    (lambda: flex.distillation_loss(X, X[:, :2], torch.zeros(4, 2)), TypeError),
    (lambda: flex.distillation_loss(X.double(), X[:, :2], torch.zeros(4, 2, dtype=torch.int64)), TypeError),
    (lambda: flex.distillation_loss(X, X[:, :2].long(), torch.zeros(4, 2, dtype=torch.int64)), TypeError),
    (lambda: flex.distillation_loss(X, X[:, :3], torch.zeros(4, 2, dtype=torch.int64)), ValueError),
    (lambda: flex.distillation_loss(X, X[:3, :2], torch.zeros(3, 2, dtype=torch.int64)), ValueError),
    (lambda: flex.distillation_loss(X, X[:, :0], torch.zeros(4, 0, dtype=torch.int64)), ValueError),
    (lambda: flex.distillation_loss(X[:0], X[:0, :2], torch.zeros(0, 2, dtype=torch.int64)), ValueError),
    (lambda: flex.distillation_loss(X, X[:, :2], torch.zeros(4, 2, dtype=torch.int64), temperature=0.0), ValueError),
    (lambda: flex.distillation_loss(X, X[:, :2], torch.zeros(4, 2, dtype=torch.int64), temperature=NAN), ValueError),
    (lambda: flex.distillation_loss(X, X[:, :2], torch.zeros(4, 2, dtype=torch.int64), row_weights=torch.ones(3)), ValueError),
    (lambda: flex.distillation_loss(X, X[:, :2], torch.zeros(4, 2, dtype=torch.int64), row_weights=torch.ones(4, dtype=torch.int64)), TypeError),
    (lambda: flex.distillation_loss(X, X[:, :2], torch.zeros(4, 2, dtype=torch.int64), reduction="sum"), ValueError),
])
def test_functions_refuse(call, error):
    with pytest.raises(error):
        call()


def test_ops_say_shapes_without_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.flexsae_amd
    with FakeTensorMode():
        x = torch.empty(3, 5, 16, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(16, device="cuda")
        y, mean, rstd = flex.layer_norm_stats(x, w)
        assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == rstd.shape == (3, 5) and mean.dtype == torch.float32
        dx, dw, db = ops.layer_norm_bwd(y, x, w, None, mean, rstd, True, True, False)
        assert dx.shape == x.shape and dx.dtype == x.dtype and dw.shape == (16,) and dw.dtype == torch.float32 and db.numel() == 0
        table = torch.empty(50, 16, dtype=torch.bfloat16, device="cuda")
        gates, tokens = torch.empty(3, 5, device="cuda"), torch.empty(3, 5, dtype=torch.int64, device="cuda")
        out = flex.embedding_lookup(tokens.int(), table, gates)
        assert out.shape == (3, 5, 16) and out.dtype == torch.bfloat16
        dt, dg = ops.lookup_bwd(out, tokens, table, gates, 1.0, True, True)
        assert dt.shape == table.shape and dt.dtype == table.dtype and dg.shape == (3, 5) and dg.dtype == torch.float32
        z = torch.empty(3, 5, 50, dtype=torch.float16, device="cuda")
        top, index = torch.empty(3, 5, 4, device="cuda"), torch.empty(3, 5, 4, dtype=torch.int64, device="cuda")
        mask = torch.empty(3, 5, dtype=torch.bool, device="cuda")
        for reduction, shape in (("mean", ()), ("none", (3, 5))):
            loss = flex.distillation_loss(z, top, index, row_weights=mask, reduction=reduction)
            assert loss.shape == shape and loss.dtype == torch.float32
        _, stats = ops.distill_fwd(z, top, index, mask.float(), 1.0, True)
        assert stats.shape == (16, 4)
        dz = ops.distill_bwd(loss, z, top, index, mask.float(), stats, 1.0, True)
        assert dz.shape == z.shape and dz.dtype == torch.float16
