"""CPU: what the training-step operators refuse before anything is launched, at the C entries (codes, never an abort) and in Python."""
import struct

import pytest
import torch

from openpcdet_amd import _lib, optim, scatter
from openpcdet_amd.spconv import pytorch as spconv
from openpcdet_amd.spconv.pytorch import norm

INVALID, WORKSPACE, RANGE = -1, -2, -4
P = 4096          # stands for a device address: refused calls never follow it


def fwd(**kw):
    a = dict(x=P, n=10, c=8, dtype=0, samples=2, offsets=P, order=None, groups=2, weight=P, bias=P, pd=0, eps=1e-5, residual=None, act=1, y=P,
             mean=P, rstd=P, ws=P, size=0)
    a.update(kw)
    return _lib.lib().pvx_group_norm_act_fwd(*[a[k] for k in ("x", "n", "c", "dtype", "samples", "offsets", "order", "groups", "weight", "bias",
                                                             "pd", "eps", "residual", "act", "y", "mean", "rstd", "ws", "size")], None)


def bwd(**kw):
    a = dict(dy=P, x=P, residual=None, n=10, c=8, dtype=0, samples=2, offsets=P, order=None, groups=2, weight=P, bias=P, pd=0, mean=P, rstd=P,
             act=1, dx=P, dres=None, dw=P, db=P, ws=P, size=0)
    a.update(kw)
    return _lib.lib().pvx_group_norm_act_bwd(*[a[k] for k in ("dy", "x", "residual", "n", "c", "dtype", "samples", "offsets", "order", "groups",
                                                             "weight", "bias", "pd", "mean", "rstd", "act", "dx", "dres", "dw", "db", "ws",
                                                             "size")], None)


def test_group_norm_codes():
    for call in (fwd, bwd):
        for kw in (dict(n=-1), dict(c=0), dict(c=-8), dict(samples=0), dict(groups=0), dict(groups=3), dict(dtype=3), dict(dtype=-1), dict(pd=7),
                   dict(act=4), dict(act=-1), dict(x=None), dict(mean=None), dict(rstd=None), dict(offsets=None, samples=3)):
            assert call(**kw) == INVALID, kw
        assert call() == WORKSPACE and call(ws=None, size=1 << 30) == WORKSPACE
        assert call(n=0x7fffffff) == RANGE and call(c=1 << 21, groups=1) == RANGE and call(samples=0x7fffffff, groups=2) == RANGE
    assert fwd(y=None) == INVALID and fwd(eps=-1.0) == INVALID and fwd(eps=float("nan")) == INVALID
    assert bwd(dy=None) == INVALID and bwd(dx=None) == INVALID
    assert fwd(n=0) == 0 and bwd(n=0, dw=None, db=None) == 0
    L = _lib.lib()
    small, large = L.pvx_group_norm_act_workspace_bytes(1000, 16, 2, 1, 4), L.pvx_group_norm_act_workspace_bytes(10 ** 6, 64, 5000, 1, 8)
    assert 256 < small < large and L.pvx_group_norm_act_workspace_bytes(0, 16, 2, 1, 4) == 256
    assert fwd(ws=P, size=L.pvx_group_norm_act_workspace_bytes(10, 8, 2, 1, 2) - 256) == WORKSPACE


def test_lookup_codes():
    L = _lib.lib()
    look = lambda table=P, dtype=0, index=P, wide=0, n=5, m=4, w=8, out=P: L.pvx_lookup_rows(table, dtype, index, wide, n, m, w, 1.0, out, None)  # noqa: E731
    for kw in (dict(n=-1), dict(m=-1), dict(w=-1), dict(dtype=3), dict(dtype=-1), dict(table=None), dict(index=None), dict(out=None)):
        assert look(**kw) == INVALID, kw
    assert look(n=0) == 0 and look(w=0) == 0 and look(n=0x7fffffff) == RANGE and look(m=0x7fffffff) == RANGE and look(w=1 << 25) == RANGE
    sort = lambda index=P, n=5, m=4, order=P, keys=P, offsets=P, ws=P, size=0: L.pvx_sort_index(index, 1, n, m, order, keys, offsets, ws, size, None)  # noqa: E731
    for kw in (dict(n=-1), dict(m=0), dict(m=-2), dict(index=None), dict(order=None), dict(keys=None)):
        assert sort(**kw) == INVALID, kw
    assert sort(n=0x7fffffff) == RANGE and sort(m=0x7fffffff) == RANGE
    assert sort(n=100000, m=50) == WORKSPACE and sort(n=100000, ws=None, size=1 << 30) == WORKSPACE
    assert L.pvx_sort_index_workspace_bytes(100000) > 3 * 4 * 100000 and L.pvx_sort_index_workspace_bytes(0) == 256
    grad = lambda dout=P, dtype=0, index=P, order=P, keys=P, n=5000, m=4, w=8, out=P, ws=P, size=0: L.pvx_lookup_rows_grad(  # noqa: E731
        dout, dtype, index, 0, order, keys, n, m, w, 1.0, out, ws, size, None)
    for kw in (dict(n=-1), dict(m=-1), dict(w=-1), dict(dtype=9), dict(dout=None), dict(order=None), dict(keys=None), dict(out=None),
               dict(index=None, order=None, keys=None)):
        assert grad(**kw) == INVALID, kw
    assert grad(m=0) == 0 and grad(w=0) == 0 and grad() == WORKSPACE and grad(order=None, keys=None) == WORKSPACE and grad(n=0x7fffffff) == RANGE
    sorted_bytes = L.pvx_lookup_rows_grad_workspace_bytes(5000, 8, 1)
    assert sorted_bytes > 5000 // 64 * 8 * 4 and L.pvx_lookup_rows_grad_workspace_bytes(5000, 8, 0) > sorted_bytes + 2 * 4 * 5000
    assert grad(order=None, keys=None, size=sorted_bytes) == WORKSPACE


def test_python_refuses_cpu_tensors():
    x = torch.zeros(6, 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        norm.group_norm_act(x, 2)
    with pytest.raises(RuntimeError, match="GPU only"):
        scatter.lookup_rows(x, torch.zeros(3, dtype=torch.long))
    with pytest.raises(RuntimeError, match="GPU only"):
        scatter.sort_index(torch.zeros(3, dtype=torch.long), 4)


def test_modules_refuse():
    with pytest.raises(ValueError):
        spconv.SparseGroupNorm(3, 16)
    with pytest.raises(ValueError):
        spconv.SparseGroupNorm(0, 16)
    gn = spconv.SparseGroupNorm(4, 16, affine=False)
    assert list(gn.parameters()) == [] and "4, 16" in repr(gn)
    assert norm.act_name(torch.nn.GELU("tanh")) is None and norm.act_name(torch.nn.GELU()) == "gelu" and norm.act_name(torch.nn.ReLU6()) is None


@pytest.mark.parametrize("co, steps, holds", [
    (optim.COEFFICIENTS, 5, 1), (optim.COEFFICIENTS, 64, 1), ((1.5, -0.5, 0.0), 64, 1), ((1.875, -1.25, 0.375), 64, 1), ((2.0, -1.5, 0.5), 64, 1),
    ((4.0, 0.0, 0.0), 6, 1), ((4.0, 0.0, 0.0), 16, 0), ((0.5, 0.0, 0.0), 64, 1), ((0.0, 0.0, 0.0), 3, 1), ((3.0, -2.0, 0.0), 0, 1),
    ((3.0, -2.0, 0.0), 6, 0), ((0.5, 1.0, 0.0), 4, 0), ((1.0, -1.0, 0.0), 1, 0), (optim.COEFFICIENTS, 65, 0), (optim.COEFFICIENTS, -1, 0)])
def test_orthogonalize_coefficients(co, steps, holds):
    """4^16 > 1e9; 3 x - 2 x^3 and x - x^3 have a root in (0, 1.01 ..]; x / 2 + x^3 leaves 0.7 to either side."""
    assert _lib.lib().pvx_orthogonalize_holds(steps, *co) == holds
    if not holds and 0 <= steps <= optim.MAX_STEPS:
        assert _lib.lib().pvx_orthogonalize(None, 0, 0, steps, *co, 1e-7, None, 0, None) == RANGE
        with pytest.raises(ValueError, match="bounds"):
            optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))], steps=steps, coefficients=co)


def test_orthogonalize_codes():
    L = _lib.lib()
    call = lambda mats, count=None, dtype=0, steps=5, eps=1e-7, ws=P, size=0: L.pvx_orthogonalize(  # noqa: E731
        struct.pack("QQii" * len(mats), *[v for m in mats for v in m]) if mats else None, len(mats) if count is None else count, dtype, steps,
        3.4445, -4.775, 2.0315, eps, ws, size, None)
    good = (P, P, 64, 432)
    for args in (dict(mats=[good], count=-1), dict(mats=[], count=2), dict(mats=[good], dtype=3), dict(mats=[good], steps=-1), dict(mats=[good], eps=-1.0),
                 dict(mats=[good], eps=float("nan")), dict(mats=[good, (P, P, 0, 4)]), dict(mats=[(P, P, 4, -1)]), dict(mats=[(0, P, 4, 4)]),
                 dict(mats=[good, (P, 0, 4, 4)])):
        assert call(**args) == INVALID, args
    assert call([good] * 65) == RANGE and call([(P, P, 4, (1 << 20) + 1)]) == RANGE
    assert call([]) == 0 and call([good]) == WORKSPACE and call([good], ws=None, size=1 << 30) == WORKSPACE
    need = L.pvx_orthogonalize_workspace_bytes(struct.pack("QQii", *good), 1, 0)
    assert need > 4 * 64 * 432 and call([good], size=need - 1) == WORKSPACE and call([good], ws=P + 16, size=need) == WORKSPACE
    assert L.pvx_orthogonalize_workspace_bytes(None, 0, 0) == 0
    assert L.pvx_orthogonalize_workspace_bytes(struct.pack("QQii", P, P, 16, 432), 1, 0) == 0     # one workgroup, no workspace


def test_optimiser_refuses():
    w = torch.nn.Parameter(torch.zeros(4, 4))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(steps=-1), dict(eps=-1.0), dict(coefficients=(1.0,))):
        with pytest.raises(ValueError):
            optim.Muon([w], **kw)
    with pytest.raises(ValueError, match="two and more"):
        optim.Muon([w, torch.nn.Parameter(torch.zeros(4))])
    w.grad = torch.ones(4, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        optim.Muon([w]).step()
    with pytest.raises(RuntimeError, match="GPU only"):
        optim.orthogonalize(torch.zeros(4, 4))
    assert optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))]).step() is None      # nothing has a gradient
