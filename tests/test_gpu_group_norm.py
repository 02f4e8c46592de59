"""Group norm (+ residual) + activation over rows (csrc/group_norm.hip; spconv.pytorch.norm.group_norm_act, SparseGroupNorm) against its
definition in float64, forward and backward.

Tolerances, element by element, from the arithmetic: the statistics are exact to binary32 (sums in binary64), so
z = (x - mu) rs w + b + r carries at most 2^-24 (2 |mu| rs |w| + 6 |xhat w| + 2 |b| + 2 |r| + 2 |z|); an activation's slope is below 1.2
and its exponential adds (4 + |z|) 2^-24 relative; the result is rounded once to its type (eps / 2).  The backward's terms likewise."""
import numpy as np
import pytest
import torch

from openpcdet_amd import backbones, engine
from openpcdet_amd.spconv import pytorch as spconv
from openpcdet_amd.spconv.pytorch import norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def act64(z, act):
    """-> value, slope"""
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(z / 2 ** 0.5))
        return z * p, p + z * torch.exp(-z * z / 2) / (2 * np.pi) ** 0.5
    return z, torch.ones_like(z)


def reference(x, groups, w, b, eps, act, res, sample, samples, dy=None):
    """float64; sample[row] = its sample, -1 for none -> dict of values and of their tolerances (before the rounding to a type)"""
    n, c = x.shape
    x, cpg = x.double(), c // groups
    w = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if b is None else b.double()
    r = torch.zeros_like(x) if res is None else res.double()
    out = {k: torch.zeros_like(x) for k in ("y", "dx", "dres")}
    tol = {k: torch.zeros_like(x) for k in out}
    out["dw"], out["db"] = torch.zeros_like(w), torch.zeros_like(w)
    tol["dw"], tol["db"] = torch.zeros_like(w), torch.zeros_like(w)
    z_all, ez_all = torch.full_like(x, 1e9), torch.zeros_like(x)
    for s in range(samples):
        rows = torch.nonzero(sample == s).flatten()
        k = rows.numel()
        if k == 0:
            continue
        v = x[rows].view(k, groups, cpg)
        mu = v.mean((0, 2), keepdim=True)
        rs = 1.0 / torch.sqrt(((v - mu) ** 2).mean((0, 2), keepdim=True) + eps)
        mu, rs = mu.expand_as(v).reshape(k, c), rs.expand_as(v).reshape(k, c)
        xh = (x[rows] - mu) * rs
        z = xh * w + b + r[rows]
        ez = U * (2 * mu.abs() * rs * w.abs() + 6 * (xh * w).abs() + 2 * b.abs() + 2 * r[rows].abs() + 2 * z.abs())
        val, slope = act64(z, act)
        out["y"][rows] = val
        tol["y"][rows] = 1.2 * ez + U * (4 + z.abs()) * val.abs() + 2.0 ** -40
        z_all[rows], ez_all[rows] = z, ez
        if dy is None:
            continue
        d = dy[rows].double()
        gz = d * slope
        egz = d.abs() * (ez * (0 if act in (None, "relu") else 1.0) + U * (8 + z.abs()))
        exh = U * (2 * mu.abs() * rs + 4 * xh.abs())
        gx = gz * w
        mean = lambda t: t.view(k, groups, cpg).mean((0, 2), keepdim=True).expand(k, groups, cpg).reshape(k, c)  # noqa: E731
        a, q = mean(gx), mean(gx * xh)
        out["dx"][rows] = rs * (gx - a - xh * q)
        out["dres"][rows] = gz
        out["db"] += gz.sum(0)
        out["dw"] += (gz * xh).sum(0)
        tol["dres"][rows] = egz
        tol["db"] += egz.sum(0)
        tol["dw"] += (egz * xh.abs() + gz.abs() * exh).sum(0)
        ea, eq = mean(egz * w.abs()), mean(egz * (w * xh).abs() + gx.abs() * exh)
        tol["dx"][rows] = rs * (egz * w.abs() + ea + xh.abs() * eq + exh * q.abs() + 8 * U * (gx.abs() + a.abs() + (xh * q).abs()))
    return out, tol, z_all, ez_all


def close(got, want, tol, what):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    bound = tol + half * (want.abs() + tol) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    bad = err > bound
    assert not bool(bad.any()), "%s: %d of %d outside; worst %.3g against %.3g" % (
        what, int(bad.sum()), bad.numel(), float(err[bad].max()), float(bound[bad].max()))


def check(dev, n, c, groups, cuts=None, dtype=torch.float32, act=None, res=False, affine=True, pdtype=torch.float32, mixed=False, equal=None,
          shift=0.0, eps=1e-5, seed=0, misalign=False):
    """cuts: ascending offsets of ragged samples; equal: number of equal samples instead"""
    g = torch.Generator(device=dev).manual_seed(seed + n + 7 * c)
    x = torch.randn(n, c, device=dev, generator=g) * (torch.rand(c, device=dev, generator=g) + 0.5) + torch.randn(c, device=dev, generator=g) + shift
    x = x.to(dtype)
    if misalign:                                     # contiguous, but off the 16-byte grid
        x = torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(n, c)
        assert x.data_ptr() % 16 != 0
    w = (torch.rand(c, device=dev, generator=g) + 0.5).to(pdtype) if affine else None
    b = (torch.randn(c, device=dev, generator=g) * 0.3).to(pdtype) if affine else None
    r = torch.randn(n, c, device=dev, generator=g).to(dtype) if res else None
    dy = torch.randn(n, c, device=dev, generator=g).to(dtype)
    offsets = order = None
    if equal is not None:
        sample = torch.arange(equal, device=dev).repeat_interleave(n // equal)
        samples = equal
    else:
        cuts = [0, n] if cuts is None else cuts
        samples = len(cuts) - 1
        sample = torch.full((n,), -1, dtype=torch.long, device=dev)
        for s in range(samples):
            sample[cuts[s]:cuts[s + 1]] = s
        offsets = torch.tensor(cuts, dtype=torch.int32, device=dev)
        if mixed:
            order = torch.randperm(n, device=dev, generator=g)
            by_row = torch.empty_like(sample)
            by_row[order] = sample                   # position p is row order[p]
            sample, order = by_row, order.int()
    _, _, z, ez = reference(x, groups, w, b, eps, act, r, sample, samples)
    if act == "relu":                                # where 32 bits do not decide the side of the step, nothing flows back
        dy = torch.where(z.abs() <= 2 * ez, torch.zeros_like(dy), dy)
    want, tol, _, _ = reference(x, groups, w, b, eps, act, r, sample, samples, dy)
    leaves = [t.clone().requires_grad_(True) if t is not None and not (misalign and t is x) else (t.requires_grad_(True) if t is not None else None)
              for t in (x, w, b, r)]
    shape = (equal, n // equal, c) if equal is not None else (n, c)
    y = norm.group_norm_act(leaves[0].view(shape) if equal is not None else leaves[0], groups, leaves[1], leaves[2], eps=eps, act=act,
                            residual=(leaves[3].view(shape) if equal is not None else leaves[3]) if res else None, offsets=offsets,
                            order=order).view(n, c)
    assert y.dtype == dtype
    close(y.detach(), want["y"], tol["y"], "y")
    with torch.no_grad():                            # the form without a graph gives the same bits
        y2 = norm.group_norm_act(x.view(shape), groups, w, b, eps=eps, act=act, residual=r.view(shape) if res else None, offsets=offsets, order=order)
    assert torch.equal(y2.view(n, c), y.detach())
    names = [k for k, t in zip(("dx", "dw", "db", "dres"), leaves) if t is not None]
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy, retain_graph=True)
    for k, got in zip(names, grads):
        close(got, want[k], tol[k], k)
    again = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,res", [(None, False), ("relu", True), ("silu", False), ("gelu", True)])
def test_few_and_many_rows(cuda_device, dtype, act, res):
    check(cuda_device, 300, 16, 4, dtype=dtype, act=act, res=res)                                        # one workgroup
    check(cuda_device, 20011, 64, 8, cuts=[0, 7000, 7000, 7001, 20011], dtype=dtype, act=act, res=res)   # an empty sample, one of one row
    check(cuda_device, 5003, 24, 8, cuts=[0, 2500, 5003], dtype=dtype, act=act, res=res, mixed=True)


@pytest.mark.parametrize("n,c,groups,cuts", [
    (1, 1, 1, None), (1, 8, 8, None), (2, 37, 37, None), (7, 37, 1, [0, 3, 7]), (4099, 37, 1, [0, 1, 4099]), (3001, 130, 5, [0, 3001]),
    (257, 100, 25, [0, 0, 257, 257]), (40, 2056, 2, [0, 11, 40]), (9, 4100, 4, [0, 2, 9]), (600, 3, 3, [0, 600])])
def test_odd_shapes(cuda_device, n, c, groups, cuts):
    for dtype in (torch.float32, torch.bfloat16):
        check(cuda_device, n, c, groups, cuts=cuts, dtype=dtype, act="silu", eps=1e-3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,c,groups", [(41000, 96, 8), (41001, 104, 52), (270000, 128, 16), (270001, 128, 32), (34000, 1000, 8)])
def test_chunks_of_two_and_four_channels(cuda_device, dtype, n, c, groups):
    """past 2^22 and past 2^25 elements; few enough groups for the applying kernels to finish the statistics, and too many"""
    check(cuda_device, n, c, groups, cuts=[0, 17, 17, n // 3, n - 100], dtype=dtype, act="silu", res=True, mixed=True)


def test_chunks_that_an_address_narrows(cuda_device):
    check(cuda_device, 270000, 128, 8, cuts=[0, 100000, 270000], dtype=torch.bfloat16, misalign=True)


def test_offsets_past_32_bits(cuda_device):
    rows, c = 2 ** 25 + 4000, 64                              # 2^31 elements end inside the second sample
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x = torch.randn(rows, c, device=cuda_device, dtype=torch.bfloat16, generator=g).requires_grad_(True)
    up = torch.randn(rows, c, device=cuda_device, dtype=torch.bfloat16, generator=g)
    w = (torch.rand(c, device=cuda_device, generator=g) + 0.5).requires_grad_(True)
    cut = 2 ** 25 - 3000
    off = torch.tensor([0, cut, rows], dtype=torch.int32, device=cuda_device)
    y = norm.group_norm_act(x, 8, w, None, act="silu", offsets=off)
    dx, dw = torch.autograd.grad(y, [x, w], up)
    for lo, hi, a, b in ((0, 2000, 0, cut), (cut, rows, cut, rows)):      # rows lo .. hi of the sample a .. b
        mean = torch.zeros(8, dtype=torch.float64, device=cuda_device)
        square = torch.zeros_like(mean)
        for k in range(a, b, 2 ** 22):
            part = x.detach()[k:min(b, k + 2 ** 22)].double().view(-1, 8, 8)
            mean += part.sum((0, 2))
            square += part.square().sum((0, 2))
        count = (b - a) * 8
        mean, rstd = mean / count, 1 / (square / count - (mean / count).square() + 1e-5).sqrt()
        rep = lambda v: v.repeat_interleave(8)  # noqa: E731
        xh = (x.detach()[lo:hi].double() - rep(mean)) * rep(rstd)
        z = xh * w.detach().double()
        want = z * torch.sigmoid(z)
        # z is off by at most 8 roundings of values up to 2 |z| + 1, SiLU's slope is below 1.1, and the result is rounded once: bfloat16 has
        # steps of 2^-7 in [1, 2), so half a step is at most eps / 2 = 2^-8 of the value
        half = torch.finfo(torch.bfloat16).eps / 2
        assert bool(((y.detach()[lo:hi].double() - want).abs() <= half * want.abs() + 16 * U * (2 * z.abs() + 1)).all())
    # the gradient of the second sample alone, from the same rows in a tensor of their own: the same formula from other pieces
    tail = x.detach()[cut:].clone().requires_grad_(True)
    wt = w.detach().clone().requires_grad_(True)
    dt, = torch.autograd.grad(norm.group_norm_act(tail, 8, wt, None, act="silu", offsets=off[1:] - cut), [tail], up[cut:])
    # means agree to 2^-23 of the values (at most 3 here), so dx to a few of those before its rounding, where the two may fall to either
    # side: half a step each, 2 (eps / 2) = 2^-7 of the value
    assert bool(((dt.double() - dx[cut:].double()).abs() <= 2 * half * dt.double().abs() + 64 * U).all())
    assert bool(torch.isfinite(dw).all())


def test_many_groups_and_samples(cuda_device):
    check(cuda_device, 20000, 2048, 2048, cuts=[0, 20000], act="silu")                   # a group a channel: the widest workgroup's LDS
    check(cuda_device, 20000, 2048, 1, cuts=[0, 9000, 20000], act="silu")
    check(cuda_device, 3000, 1024, 1024, cuts=[0, 3000], dtype=torch.bfloat16)
    check(cuda_device, 60000, 4, 4, cuts=[0] + sorted(torch.randint(0, 60000, (2999,), generator=torch.Generator().manual_seed(1)).tolist()) + [60000], eps=1e-2)      # 3000 frames


def test_rows_of_no_sample(cuda_device):
    check(cuda_device, 120, 16, 2, cuts=[10, 50, 100], act="gelu", res=True)              # one launch
    check(cuda_device, 9000, 16, 2, cuts=[100, 5000, 8000], act="gelu", res=True)
    check(cuda_device, 9000, 16, 2, cuts=[100, 5000, 8000], act="silu", mixed=True)
    check(cuda_device, 50, 16, 2, cuts=[0, 0, 0])                                         # all samples empty


def test_equal_samples_and_parameter_types(cuda_device):
    check(cuda_device, 3 * 4000, 32, 4, equal=3, act="relu", dtype=torch.bfloat16, pdtype=torch.bfloat16)
    check(cuda_device, 3 * 40, 32, 4, equal=3, act="silu", dtype=torch.float16, pdtype=torch.float16)
    check(cuda_device, 5000, 8, 2, equal=5000, act="silu", eps=1e-2)                      # a sample a row, more samples than workgroups
    check(cuda_device, 3 * 4100, 8, 4, equal=4100, act=None, eps=1e-2)
    check(cuda_device, 700, 16, 16, affine=False, act="gelu")


def test_far_mean_flat_groups_and_alignment(cuda_device):
    check(cuda_device, 8192, 16, 2, shift=1000.0)                                         # mean >> spread: the sums keep their digits
    check(cuda_device, 8192, 16, 2, shift=1000.0, dtype=torch.bfloat16)
    check(cuda_device, 2000, 32, 4, misalign=True, act="silu", dtype=torch.bfloat16)
    check(cuda_device, 20000, 32, 4, misalign=True, act="silu")
    x = torch.full((500, 8), 3.25, device=cuda_device)
    assert torch.equal(norm.group_norm_act(x, 2, offsets=torch.tensor([0, 500], dtype=torch.int32, device=cuda_device)), torch.zeros_like(x))


def test_nan_and_infinity_stay_in_their_group(cuda_device):
    for n in (200, 20000):
        x = torch.randn(n, 16, device=cuda_device)
        off = torch.tensor([0, n // 2, n], dtype=torch.int32, device=cuda_device)
        clean = norm.group_norm_act(x, 4, act="relu", offsets=off)
        x[3, 5], x[n - 1, 15] = float("nan"), float("inf")
        y = norm.group_norm_act(x, 4, act="relu", offsets=off)
        bad = torch.zeros(n, 16, dtype=torch.bool, device=cuda_device)
        bad[:n // 2, 4:8] = True
        bad[n // 2:, 12:16] = True
        assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], clean[~bad])


def test_strides_broadcasts_and_shared_leaves(cuda_device):
    torch.manual_seed(0)
    base = torch.randn(2, 16, 9, 11, device=cuda_device, requires_grad=True)              # [B, C, H, W]: channels are moved last by a view
    w = torch.rand(16, device=cuda_device, requires_grad=True)
    y = norm.group_norm_act(base.permute(0, 2, 3, 1), 4, w, None, act="silu")
    y.sum().backward()                                                                    # a gradient of stride 0
    b64, w64 = base.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    want = torch.nn.functional.silu(torch.nn.functional.group_norm(b64, 4, w64))
    want.sum().backward()
    assert torch.allclose(y.detach().permute(0, 3, 1, 2).double(), want.detach(), atol=2e-6)
    assert torch.allclose(base.grad.double(), b64.grad, atol=1e-5) and torch.allclose(w.grad.double(), w64.grad, rtol=1e-5, atol=1e-3)
    x = torch.randn(1, 8, device=cuda_device, requires_grad=True)                         # a broadcast input, and the same tensor as residual
    z = x.expand(64, 8)
    off = torch.tensor([0, 64], dtype=torch.int32, device=cuda_device)
    out = norm.group_norm_act(z, 1, residual=z, offsets=off)
    up = torch.randn(64, 8, device=cuda_device)
    (out * up).sum().backward()
    x64 = x.detach().double().requires_grad_(True)
    z64 = x64.expand(64, 8)
    mu, var = z64.mean(), z64.var(unbiased=False)
    (((z64 - mu) / torch.sqrt(var + 1e-5) + z64) * up.double()).sum().backward()
    assert torch.allclose(x.grad.double(), x64.grad, atol=1e-4)


def test_gradient_against_differences(cuda_device):
    torch.manual_seed(4)
    x = torch.randn(12, 8, device=cuda_device)
    w, b = torch.rand(8, device=cuda_device) + 0.5, torch.randn(8, device=cuda_device)
    off = torch.tensor([0, 5, 12], dtype=torch.int32, device=cuda_device)
    up = torch.randn(12, 8, device=cuda_device)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    value = lambda ts: (norm.group_norm_act(ts[0], 2, ts[1], ts[2], act="gelu", offsets=off).double() * up.double()).sum()  # noqa: E731
    grads = torch.autograd.grad(value(leaves), leaves)
    h = 2.0 ** -6
    for k, t in enumerate((x, w, b)):
        d = torch.randn_like(t)
        d /= d.norm()
        plus, minus = [v.clone() for v in (x, w, b)], [v.clone() for v in (x, w, b)]
        plus[k] += h * d
        minus[k] -= h * d
        with torch.no_grad():
            slope = float(value(plus) - value(minus)) / (2 * h)
        # central differences: third derivatives times h^2 / 6 (values here are of order 10), rounding 96 * 4 U / h
        assert abs(slope - float((grads[k] * d).sum())) <= 10 * h * h + 96 * 8 * U / h


def test_streams_and_graph(cuda_device):
    torch.manual_seed(2)
    for n in (200, 30000):                                    # one launch, three launches
        off = torch.tensor([0, n // 3, n], dtype=torch.int32, device=cuda_device)
        data = [torch.randn(n, 32, device=cuda_device) for _ in range(3)]
        ups = [torch.randn(n, 32, device=cuda_device) for _ in range(3)]
        w = torch.rand(32, device=cuda_device)

        def step(x, up):
            x = x.detach().requires_grad_(True)
            wl = w.detach().requires_grad_(True)
            y = norm.group_norm_act(x, 8, wl, None, act="silu", offsets=off)
            return (y.detach(),) + torch.autograd.grad(y, [x, wl], up)

        want = [step(x, up) for x, up in zip(data, ups)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(data[1], ups[1])
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want[1]))
        xs, us = data[0].clone(), ups[0].clone()
        graphs = []
        for _ in range(2):                                    # two graphs, replayed in turn
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                out = step(xs, us)
            graphs.append((gr, out))
        for k in (1, 2, 0, 1):
            xs.copy_(data[k])
            us.copy_(ups[k])
            for gr, out in graphs:
                gr.replay()
            step(data[2], ups[2])                             # eager work between the replays
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(p, q) for p, q in zip(out, want[k]))


def _sites(dev, c, mixed=False, batch=3, seed=1):
    r = np.random.default_rng(seed)
    coords = np.unique(np.stack([r.integers(0, batch, 2500), r.integers(0, 8, 2500), r.integers(0, 20, 2500), r.integers(0, 20, 2500)], 1), axis=0)
    coords = coords[coords[:, 0] != 1]                        # a frame without sites
    if mixed:
        coords = coords[r.permutation(len(coords))]
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(len(coords), c, device=dev, generator=g), torch.from_numpy(coords.astype(np.int32)).to(dev))


def test_sparse_module_and_sequential(cuda_device):
    feats, idx = _sites(cuda_device, 16, mixed=True)
    gn = spconv.SparseGroupNorm(4, 32).to(cuda_device)
    assert sorted(gn.state_dict()) == ["bias", "weight"]
    with torch.no_grad():
        gn.weight.uniform_(0.5, 1.5)
        gn.bias.normal_()
    for act_module, act in ((torch.nn.ReLU(), "relu"), (torch.nn.SiLU(), "silu"), (torch.nn.GELU(), "gelu"), (torch.nn.Tanh(), None)):
        seq = spconv.SparseSequential(spconv.SubMConv3d(16, 32, 3, padding=1, bias=False, indice_key="k"), gn, act_module).to(cuda_device)
        f = feats.clone().requires_grad_(True)
        x = spconv.SparseConvTensor(f, idx, [8, 20, 20], 3)
        out = seq(x)
        conv = seq[0](x).features.detach()
        want, tol, _, _ = reference(conv, 4, gn.weight.detach(), gn.bias.detach(), gn.eps, act, None, idx[:, 0].long(), 3)
        if act is None:
            want["y"], tol["y"] = torch.tanh(want["y"]), tol["y"] + 8 * U
        close(out.features.detach(), want["y"], tol["y"], "sequential")
        gn.zero_grad()
        out.features.square().sum().backward()
        assert float(f.grad.abs().sum()) > 0 and gn.weight.grad is not None
        assert torch.equal(seq.eval()(x).features, out.features)          # nothing depends on the mode
    none = spconv.SparseConvTensor(feats[:0].requires_grad_(True), idx[:0], [8, 20, 20], 3)
    assert spconv.SparseSequential(spconv.SparseGroupNorm(4, 16).to(cuda_device), torch.nn.ReLU())(none).features.shape == (0, 16)
    assert x._sample_rows()[0].tolist()[1] == x._sample_rows()[0].tolist()[2]
    first = x._sample_rows()
    assert x._sample_rows()[0] is first[0] and x.replace_feature(f)._sample_rows()[0] is first[0]
    x.indices[:, 0] = 0                                       # written to: the rows are listed anew
    assert x._sample_rows()[0].tolist() == [0, len(idx), len(idx), len(idx)]


def test_hooks_of_an_activation_are_called(cuda_device):
    feats, idx = _sites(cuda_device, 16)
    seen, relu = [], torch.nn.ReLU()
    seq = spconv.SparseSequential(spconv.SparseGroupNorm(4, 16).to(cuda_device), relu)
    want = seq(spconv.SparseConvTensor(feats, idx, [8, 20, 20], 3)).features
    relu.register_forward_hook(lambda m, i, o: seen.append(i[0]))
    got = seq(spconv.SparseConvTensor(feats, idx, [8, 20, 20], 3)).features
    assert len(seen) == 1 and float(seen[0].min()) < 0 and torch.equal(got, want)      # the clamp of the same fp32 values


def test_sample_rows_follow_stream_and_capture(cuda_device):
    feats, idx = _sites(cuda_device, 16, mixed=True)
    gn = spconv.SparseGroupNorm(4, 16).to(cuda_device)
    fresh = lambda i: gn(spconv.SparseConvTensor(feats, i, [8, 20, 20], 3)).features.detach()  # noqa: E731
    x = spconv.SparseConvTensor(feats, idx.clone(), [8, 20, 20], 3)
    want = [fresh(idx)]
    swapped = idx.clone()
    swapped[:, 0] = 2 - swapped[:, 0] + (swapped[:, 1] == 0).int()        # other frames, some rows in none
    want.append(fresh(swapped))
    first = x._sample_rows()[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert x._sample_rows()[0] is not first                           # this stream has not waited for that sort
        other = gn(x).features.detach()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want[0])
    for known in (False, True):                                           # captured before and after an eager call has listed the rows
        x = spconv.SparseConvTensor(feats, idx.clone(), [8, 20, 20], 3)
        if known:
            gn(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = gn(x).features.detach()
        assert torch.equal(gn(x).features.detach(), want[0])              # eager, before any replay
        for k, indices in ((0, idx), (1, swapped), (0, idx), (1, swapped)):
            x.indices.copy_(indices)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[k])
            assert torch.equal(gn(x).features.detach(), want[k])


def test_backbone_with_group_norm(cuda_device):
    torch.manual_seed(0)
    feats, idx = _sites(cuda_device, 5, batch=2)
    idx[:, 0] = (idx[:, 0] > 0).int()
    idx = torch.unique(idx, dim=0).contiguous()
    feats = torch.randn(len(idx), 5, device=cuda_device)
    net = backbones.VoxelResBackBone8x(input_channels=5, grid_size=np.array([64, 64, 40]), model_cfg={"NORM_GROUPS": 4}).to(cuda_device)
    assert not any(isinstance(m, torch.nn.BatchNorm1d) for m in net.modules())
    run = lambda f, i: net({"voxel_features": f, "voxel_coords": i.float(), "batch_size": 2})["encoded_spconv_tensor"]  # noqa: E731
    out = run(feats, idx)
    out.features.square().sum().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in net.parameters())
    # a frame's result does not depend on its neighbours in the batch
    one = idx[idx[:, 0] == 1].clone()
    one[:, 0] = 0
    alone = net({"voxel_features": feats[idx[:, 0] == 1], "voxel_coords": one.float(), "batch_size": 1})["encoded_spconv_tensor"]
    both = out.features[out.indices[:, 0] == 1]
    assert torch.allclose(alone.features, both, rtol=1e-4, atol=1e-5)
    with pytest.raises(TypeError, match="group norm"):
        engine.HotPathEngine(net.eval(), 1, [0, 0, 0, 6.4, 6.4, 4], [0.1, 0.1, 0.1], 5, 1000, 5, 1000, device=cuda_device)


def test_no_rows(cuda_device):
    for shape, off in (((0, 16), [0, 0]), ((0, 16), [0, 0, 0, 0]), ((0, 4, 16), None), ((3, 0, 16), None)):
        x = torch.zeros(shape, device=cuda_device, requires_grad=True)
        w = torch.ones(16, device=cuda_device, requires_grad=True)
        o = torch.tensor(off, dtype=torch.int32, device=cuda_device) if off else None
        y = norm.group_norm_act(x, 4, w, None, act="relu", offsets=o)
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape and torch.equal(w.grad, torch.zeros_like(w))


def test_refusals_on_the_device(cuda_device):
    x = torch.zeros(6, 8, device=cuda_device)
    off = torch.tensor([0, 6], dtype=torch.int32, device=cuda_device)
    bad = [dict(num_groups=3), dict(num_groups=0), dict(act="tanh"), dict(eps=-1.0), dict(eps=float("nan")), dict(order=off),
           dict(weight=torch.zeros(7, device=cuda_device)), dict(weight=torch.zeros(8)), dict(residual=torch.zeros(6, 4, device=cuda_device)),
           dict(offsets=off.long()), dict(offsets=off[:1]), dict(offsets=off, order=off), dict(offsets=off.cpu())]
    for kw in bad:
        args = dict(num_groups=2)
        args.update(kw)
        with pytest.raises(ValueError):
            norm.group_norm_act(x, **args)
    with pytest.raises(ValueError):
        norm.group_norm_act(x.view(2, 3, 8), 2, offsets=off)
    for kw in (dict(weight=torch.zeros(8, device=cuda_device, dtype=torch.float64)),
               dict(weight=torch.zeros(8, device=cuda_device), bias=torch.zeros(8, device=cuda_device).half())):
        with pytest.raises(TypeError):
            norm.group_norm_act(x, 2, **kw)
    with pytest.raises(TypeError):
        norm.group_norm_act(x.double(), 2)
    y = norm.group_norm_act(x.requires_grad_(True), 2, offsets=off)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):                         # no second derivative
        g.sum().backward()
