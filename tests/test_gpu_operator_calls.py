"""Calls of the training-step operators (csrc/group_norm.hip, csrc/lookup.hip, csrc/orthogonalize.hip and their Python entries) that the
tests by operator leave out: other derivatives, sizes past 32 bits, special values, hooks, caches, optimiser options and states."""
import copy

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from openpcdet_amd import backbones, optim, scatter, vfe
from openpcdet_amd.spconv import pytorch as spconv
from openpcdet_amd.spconv.pytorch import norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# ---- sizes past 32 bits ----------------------------------------------------------------------------------------------------
def test_lookup_refuses_counts_past_32_bits(cuda_device):
    """2^32 + 5 is 5 in 32 bits.  The tensors are expanded from one element: refused before anything of that size is made"""
    big = 2 ** 32 + 5
    one, zero = torch.zeros(1, 1, dtype=torch.bfloat16, device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for call in (lambda: scatter.lookup_rows(one.expand(big, 1), zero), lambda: scatter.lookup_rows(one, zero.expand(big)),
                 lambda: scatter.lookup_rows(one.expand(2, big), zero), lambda: scatter.sort_index(zero, big),
                 lambda: scatter.sort_index(zero.expand(big), 4)):
        with pytest.raises(ValueError, match="32 bits"):
            call()


def test_group_norm_refuses_counts_past_32_bits(cuda_device):
    big = 2 ** 32 + 5
    one, off = torch.zeros(1, 1, dtype=torch.bfloat16, device=cuda_device), torch.zeros(2, dtype=torch.int32, device=cuda_device)
    for call in (lambda: norm.group_norm_act(one.expand(big, 1), 1, offsets=off), lambda: norm.group_norm_act(one.expand(big, 1), 1),
                 lambda: norm.group_norm_act(one.expand(1, big), 1), lambda: norm.group_norm_act(one.unsqueeze(0).expand(1, big, 1), 1),
                 lambda: norm.group_norm_act(one, 1, offsets=off[:1].expand(big))):
        with pytest.raises(ValueError, match="32 bits"):
            call()


# ---- forward-mode derivatives ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(cuda_device, grad):
    """no forward-mode derivative is defined: refused, not taken for zero"""
    x, w, r = (torch.randn(s, device=cuda_device) for s in ((6, 8), (8,), (6, 8)))
    index = torch.tensor([0, 5, 2], device=cuda_device)
    plain = norm.group_norm_act(x, 2, w, act="relu", residual=r), scatter.lookup_rows(x, index)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: norm.group_norm_act(dual(x), 2, w), lambda: norm.group_norm_act(x, 2, dual(w)),
                     lambda: norm.group_norm_act(x, 2, w, dual(w)), lambda: norm.group_norm_act(x, 2, residual=dual(r)),
                     lambda: scatter.lookup_rows(dual(x), index)):
            with pytest.raises(RuntimeError):
                call()
        assert torch.equal(norm.group_norm_act(x, 2, w, act="relu", residual=r), plain[0])      # nothing dual: as ever
        assert torch.equal(scatter.lookup_rows(x, index), plain[1])
    with torch.set_grad_enabled(grad):
        for f in (lambda t: norm.group_norm_act(t, 2, w), lambda t: scatter.lookup_rows(t, index)):
            with pytest.raises(RuntimeError):
                torch.func.jvp(f, (x,), (torch.ones_like(x),))
            with pytest.raises(RuntimeError):
                torch.func.vmap(f)(x.expand(3, 6, 8))


# ---- the largest sizes of the norm -----------------------------------------------------------------------------------------
def test_norm_of_more_than_2_30_samples(cuda_device):
    """the rows are those of the last sample: the search for it adds up sample numbers past 2^31"""
    samples, n = 2 ** 30 + 1000, 700
    off = torch.zeros(samples + 1, dtype=torch.int32, device=cuda_device)
    off[-1] = n
    x = torch.randn(n, 1, device=cuda_device)
    y = norm.group_norm_act(x, 1, offsets=off)
    want = norm.group_norm_act(x, 1, offsets=torch.tensor([0, n], dtype=torch.int32, device=cuda_device))
    assert float((y - want).abs().max()) <= 8 * U * float(want.abs().max() + 1)


def test_norm_of_nearly_2_31_rows(cuda_device):
    """one channel, rows up to the largest count that is taken: the last workgroup's range ends past 2^31"""
    n = 2 ** 31 - 2 ** 20 - 1
    g = torch.Generator(device=cuda_device).manual_seed(6)
    x = torch.empty(n, 1, dtype=torch.float16, device=cuda_device)
    x.normal_(generator=g)
    cut = n - 5000000                                          # the last sample lies in the last two ranges
    off = torch.tensor([0, cut, n], dtype=torch.int32, device=cuda_device)
    up = torch.empty_like(x)
    up.normal_(generator=g)
    y = norm.group_norm_act(x.requires_grad_(True), 1, offsets=off)
    dx, = torch.autograd.grad(y, x, up)
    x, y = x.detach(), y.detach()
    for lo, hi, a, b in ((0, 1000, 0, cut), (cut - 1000, cut, 0, cut), (cut, n, cut, n)):
        mean = square = 0.0
        for k in range(a, b, 2 ** 28):
            part = x[k:min(b, k + 2 ** 28)].double()
            mean, square = mean + float(part.sum()), square + float(part.square().sum())
        mean, square = mean / (b - a), square / (b - a)
        want = (x[lo:hi].double() - mean) / (square - mean * mean + 1e-5) ** 0.5
        # five roundings of 32 bits and one of 16
        tol = 8 * U * (want.abs() + 1) + 2.0 ** -25
        assert bool(((y[lo:hi].double() - want).abs() <= tol + 2.0 ** -11 * (want.abs() + tol)).all())
    # of the last sample, whole: xhat is `want`, and dx = (dy - mean dy - xhat mean(dy xhat)) / sqrt(var + eps), a dozen roundings of terms
    # no larger than |dy| + |mean| + |xhat mean|
    d = up[cut:].double()
    m0, m1 = d.mean(), (d * want).mean()
    terms = (d.abs() + m0.abs() + (want * m1).abs() + 1) / (square - mean * mean + 1e-5) ** 0.5
    slope = (d - m0 - want * m1) / (square - mean * mean + 1e-5) ** 0.5
    assert bool(((dx[cut:].double() - slope).abs() <= 16 * U * terms + 2.0 ** -25 + 2.0 ** -11 * slope.abs() * (1 + 2.0 ** -10)).all())


# ---- hooks and subclasses --------------------------------------------------------------------------------------------------
def _sites(dev, c, batch=3, seed=1):
    r = np.random.default_rng(seed)
    coords = np.unique(np.stack([r.integers(0, batch, 2500), r.integers(0, 8, 2500), r.integers(0, 20, 2500), r.integers(0, 20, 2500)], 1), axis=0)
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(len(coords), c, device=dev, generator=g), torch.from_numpy(coords.astype(np.int32)).to(dev)


# ---- the list of each frame's rows -----------------------------------------------------------------------------------------
def test_sample_rows_follow_the_batch_size(cuda_device):
    feats, idx = _sites(cuda_device, 16)
    gn = spconv.SparseGroupNorm(4, 16).to(cuda_device)
    want = gn(spconv.SparseConvTensor(feats, idx, [8, 20, 20], 3)).features
    x = spconv.SparseConvTensor(feats, idx, [8, 20, 20], 2)
    assert float(gn(x).features[idx[:, 0] == 2].abs().max()) == 0      # rows of no frame
    x.batch_size = 3
    assert torch.equal(gn(x).features, want)


def test_sample_rows_of_inference_mode(cuda_device):
    feats, idx = _sites(cuda_device, 16)
    gn = spconv.SparseGroupNorm(4, 16).to(cuda_device)
    want = gn(spconv.SparseConvTensor(feats, idx, [8, 20, 20], 3)).features.detach()
    x = spconv.SparseConvTensor(feats, idx, [8, 20, 20], 3)
    with torch.inference_mode():
        assert torch.equal(gn(x).features, want)
        inside = spconv.SparseConvTensor(feats.clone(), idx.clone(), [8, 20, 20], 3)      # tensors of inference mode: no version counter
        assert torch.equal(gn(inside).features, want)
    f = feats.clone().requires_grad_(True)
    y = gn(x.replace_feature(f)).features                      # a training call on the same sites
    assert torch.equal(y.detach(), want)
    y.square().sum().backward()
    assert f.grad is not None and gn.weight.grad is not None


# ---- special values --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [200, 20000])
def test_relu_passes_the_gradient_of_nan(cuda_device, n, dtype):
    """relu's slope is 0 only where z <= 0: a NaN keeps the gradient that came in, so a loss that has gone wrong shows"""
    g = torch.Generator(device=cuda_device).manual_seed(n)
    x = torch.randn(n, 16, device=cuda_device, generator=g).to(dtype)
    x[3, 5] = float("nan")
    res = torch.randn(n, 16, device=cuda_device, generator=g).to(dtype).requires_grad_(True)
    b = torch.randn(16, device=cuda_device, generator=g).requires_grad_(True)
    up = torch.randn(n, 16, device=cuda_device, generator=g).to(dtype)
    off = torch.tensor([0, n // 2, n], dtype=torch.int32, device=cuda_device)
    y = norm.group_norm_act(x, 4, None, b, act="relu", residual=res, offsets=off)
    dres, db = torch.autograd.grad(y, [res, b], up)
    # torch's own rule on the same outputs
    assert torch.equal(dres, torch.where(y <= 0, torch.zeros_like(up), up))
    assert bool(torch.isnan(y[:n // 2, 4:8]).all())
    want = torch.where(y <= 0, torch.zeros_like(up), up).double().sum(0)
    assert bool(((db.double() - want).abs() <= U * want.abs() + 1e-30).all())        # sums in 64 bits, rounded once


# ---- second derivatives and indices from the end through the voxel encoders ------------------------------------------------
def _encoder_layer(dev):
    """a PFNLayerV2, its input, indices that count from the end among them, and what x_max[unq_inv] makes of it"""
    torch.manual_seed(3)
    layer = vfe.PFNLayerV2(10, 32, use_norm=False).to(dev)
    inv = torch.randint(-500, 500, (4000,), device=dev, dtype=torch.int32)

    def plain(a):
        h = layer.relu(layer.linear(a))
        return torch.cat([h, scatter.scatter_max(h, inv, dim=0, dim_size=500)[0][inv.long(), :]], dim=1)

    return layer, torch.randn(4000, 10, device=dev), inv, plain


def test_voxel_encoder_layer_counts_from_the_end(cuda_device):
    layer, x, inv, plain = _encoder_layer(cuda_device)
    results = []
    for f in (lambda a: layer(a, inv, 500), lambda a: layer(a, inv.long(), 500), plain):
        a = x.clone().requires_grad_(True)
        out = f(a)
        results.append((out.detach(), torch.autograd.grad((out ** 2).sum(), a)[0]))
    for got in results[:2]:
        assert torch.equal(got[0], results[2][0])
        assert float((got[1] - results[2][1]).norm()) <= 1e-5 * float(results[2][1].norm())      # sums of some 20 terms, in another order


def test_voxel_encoders_take_the_lookup(cuda_device, monkeypatch):
    calls = []
    real = vfe.lookup_rows
    monkeypatch.setattr(vfe, "lookup_rows", lambda t, i, **kw: calls.append(int(i.min())) or real(t, i, **kw))
    enc = vfe.DynamicVoxelVFE(dict(USE_NORM=True, WITH_DISTANCE=False, USE_ABSLOTE_XYZ=True, NUM_FILTERS=[32, 16]), 4, [0.25, 0.25, 0.1], [64, 64, 40],
                              [0.0, -8.0, -2.0, 16.0, 8.0, 2.0]).to(cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    pts = torch.rand(3000, 5, device=cuda_device, generator=g) * torch.tensor([0.0, 20.0, 16.0, 4.0, 1.0], device=cuda_device) \
        - torch.tensor([0.0, 0.0, 8.0, 2.0, 0.0], device=cuda_device)
    enc({"points": pts, "batch_size": 1})                                  # a fifth of the points lies outside
    assert len(calls) == 1 and calls[0] >= 0


def test_lookup_differentiates_again(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(1)
    for n, m in ((300, 40), (20000, 700)):
        table = torch.randn(m, 24, device=cuda_device, generator=g).requires_grad_(True)
        index = torch.randint(-3, m + 3, (n,), device=cuda_device, generator=g)
        v = torch.randn(m, 24, device=cuda_device, generator=g)
        for sort in (None, scatter.sort_index(index, m)):
            out = scatter.lookup_rows(table, index, scale=0.5, sort=sort)
            first, = torch.autograd.grad((out ** 3).sum(), table, create_graph=True)
            second, = torch.autograd.grad((first * v).sum(), table)
            # L = sum (s T)^3 over the entries inside: dL = 3 s^3 T^2, times v, again: 6 s^3 T v, once an entry
            count = torch.bincount(index[(index >= 0) & (index < m)], minlength=m).double().unsqueeze(1)
            t64 = table.detach().double()
            want = count * 6 * 0.125 * t64 * v.double()
            assert torch.allclose(first.detach().double(), count * 3 * 0.125 * t64 ** 2, rtol=0, atol=float(count.max()) * 40 * U * float((t64 ** 2).max()))
            assert bool(((second.double() - want).abs() <= (count + 12) * U * want.abs()).all())


def test_voxel_encoder_layer_differentiates_again(cuda_device):
    layer, x, inv, plain = _encoder_layer(cuda_device)
    results = []
    for f in (lambda a: layer(a, inv, 500), plain):
        a = x.clone().requires_grad_(True)
        first, = torch.autograd.grad((f(a) ** 2).sum(), a, create_graph=True)
        results.append((first.detach(),) + torch.autograd.grad((first ** 2).sum(), [a, layer.linear.weight]))
    for got, want in zip(*results):
        assert float((got - want).norm()) <= 1e-5 * float(want.norm())        # sums of some 20 terms, in another order


# ---- the optimiser ---------------------------------------------------------------------------------------------------------
def test_muon_refuses_in_any_group_before_it_changes_anything(cuda_device):
    def setup(bad_shape=(4, 4), dtype=torch.float32, device=cuda_device):
        good, bad = torch.nn.Parameter(torch.ones(4, 4, device=cuda_device)), torch.nn.Parameter(torch.ones(bad_shape, device=device, dtype=dtype))
        good.grad, bad.grad = torch.ones_like(good), torch.ones_like(bad)
        return good, bad, optim.Muon([dict(params=[good]), dict(params=[bad])])

    def untouched(good, opt):
        return float((good - 1).abs().max()) == 0 and not opt.state

    for kw, error in ((dict(dtype=torch.float64), TypeError), (dict(device="cpu"), RuntimeError), (dict(bad_shape=(1, 2 ** 20 + 1)), ValueError),
                      (dict(bad_shape=(2 ** 20 + 1, 1)), ValueError)):
        good, bad, opt = setup(**kw)
        with pytest.raises(error):
            opt.step()
        assert untouched(good, opt), kw
    good, bad, opt = setup()
    bad.grad = bad.grad.to_sparse()
    with pytest.raises(RuntimeError):
        opt.step()
    assert untouched(good, opt)
    for kw in (dict(steps=65), dict(steps=-1), dict(coefficients=(3.0, -2.0, 0.0)), dict(coefficients=(1.0, 2.0)), dict(eps=-1.0), dict(momentum=-3.0),
               dict(momentum=1.0), dict(weight_decay=-1.0), dict(lr=-1.0), dict(lr=float("nan"))):
        good, bad, opt = setup()
        opt.param_groups[1].update(kw)                         # as a scheduler or a loaded state may
        with pytest.raises(ValueError):
            opt.step()
        assert untouched(good, opt), kw


def reference(m, steps=5, eps=1e-7, coefficients=optim.COEFFICIENTS):
    a, b, c = coefficients
    x = m.double()
    tall = x.shape[0] > x.shape[1]
    x = (x.t() if tall else x).contiguous()
    x = x / (x.square().sum().sqrt() + eps)
    for _ in range(steps):
        g = x @ x.t().contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if tall else x


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1.0), (torch.float16, 1.0), (torch.float16, 2.0 ** -22), (torch.float32, 1.0)])
def test_muon_keeps_its_momentum_in_32_bits(cuda_device, dtype, size, nesterov):
    """Against the recurrence in 64 bits on the same gradients (2^-22: a few steps above the least of float16).  The momentum takes two
    roundings a step of sums no larger than sum |grad|; a weight takes one of its type on (1 - lr decay) p - lr scale o, where o is within
    3800 2^-24 of its own norm (the five steps of the polynomial on the halves of its operands) and four roundings of 32 bits come to it."""
    g = torch.Generator(device=cuda_device).manual_seed(9)
    lr, decay, mom = 0.05, 0.1, 0.9
    shapes = [(16, 3, 3, 3, 5), (90, 16), (4, 4)]
    params = [torch.nn.Parameter(torch.randn(s, device=cuda_device, generator=g).to(dtype)) for s in shapes]
    opt = optim.Muon(params, lr=lr, momentum=mom, nesterov=nesterov, weight_decay=decay)
    bufs = [torch.zeros(s, dtype=torch.float64, device=cuda_device) for s in shapes]
    mags = [torch.zeros_like(b) for b in bufs]
    for step in range(6):
        before = [p.detach().double().clone() for p in params]
        want = []
        for k, p in enumerate(params):
            p.grad = (torch.randn(p.shape, device=cuda_device, generator=g) * size + (size if step < 3 else 0.0)).to(dtype)
            bufs[k] = mom * bufs[k] + p.grad.double()
            mags[k] = mom * mags[k] + p.grad.double().abs()
            u = p.grad.double() + mom * bufs[k] if nesterov else bufs[k]
            o = reference(u.view(u.shape[0], -1))
            scale = max(1.0, o.shape[0] / o.shape[1]) ** 0.5
            want.append((before[k] * (1 - lr * decay) - lr * scale * o.view(u.shape), lr * scale * float(o.norm())))
        opt.step()
        for p, buf, mag, q, (w, o) in zip(params, bufs, mags, before, want):
            got = opt.state[p]["momentum_buffer"]
            assert got.dtype == torch.float32
            assert bool(((got.double() - buf).abs() <= 2 * (step + 1) * U * mag).all())
            tol = 3800 * U * o + 4 * U * (q.abs() + o)
            tol = tol + torch.finfo(dtype).eps / 2 * (w.abs() + tol)
            assert bool(((p.detach().double() - w).abs() <= tol).all()), "step %d, %s" % (step, tuple(p.shape))
    again = optim.Muon([torch.nn.Parameter(p.detach().clone()) for p in params], lr=lr, momentum=mom, nesterov=nesterov, weight_decay=decay)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    for p, q in zip(params, again.param_groups[0]["params"]):
        assert torch.equal(opt.state[p]["momentum_buffer"], again.state[q]["momentum_buffer"])      # the type and the bits survive loading
        p.grad = torch.randn(p.shape, device=cuda_device, generator=g).to(dtype)
        q.grad = p.grad.clone()
    opt.step()
    again.step()
    assert all(torch.equal(p, q) for p, q in zip(params, again.param_groups[0]["params"]))


class OldNorm(spconv.SparseGroupNorm):
    def forward(self, input):                                  # the signature of any sparse module
        return super().forward(input)


def test_hooks_of_a_group_norm_see_the_norm(cuda_device):
    feats, idx = _sites(cuda_device, 16)
    make = lambda: spconv.SparseConvTensor(feats, idx, [8, 20, 20], 3)  # noqa: E731
    gn = spconv.SparseGroupNorm(4, 16).to(cuda_device)
    seq = spconv.SparseSequential(gn, torch.nn.ReLU())
    want, alone = seq(make()).features, gn(make()).features
    seen = []
    handle = gn.register_forward_hook(lambda m, i, o: seen.append(o.features))
    got = seq(make()).features
    assert len(seen) == 1 and torch.equal(seen[0], alone) and torch.equal(got, want)      # the clamp of the same fp32 values
    handle.remove()
    assert torch.equal(spconv.SparseSequential(OldNorm(4, 16).to(cuda_device), torch.nn.ReLU())(make()).features, want)
    called = []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, i, o: called.append(type(m).__name__))
    try:
        assert torch.equal(seq(make()).features, want)
    finally:
        handle.remove()
    assert called == ["SparseGroupNorm", "ReLU", "SparseSequential"]


def test_hooks_of_a_residual_block_see_the_norm(cuda_device):
    feats, idx = _sites(cuda_device, 16)
    make = lambda: spconv.SparseConvTensor(feats, idx, [8, 20, 20], 3)  # noqa: E731
    torch.manual_seed(0)
    block = backbones.SparseBasicBlock(16, 16, norm_fn=lambda c: spconv.SparseGroupNorm(4, c), indice_key="k").to(cuda_device)
    want = block(make()).features
    seen = []
    handles = [m.register_forward_hook(lambda m, i, o: seen.append(o.features)) for m in (block.bn1, block.bn2)]
    got = block(make()).features
    [h.remove() for h in handles]
    assert len(seen) == 2 and all(float(s.min()) < 0 for s in seen)
    assert torch.equal(got, want)                              # fp32: norm, + residual and clamp round as the fused form does
    old = backbones.SparseBasicBlock(16, 16, norm_fn=lambda c: OldNorm(4, c), indice_key="k").to(cuda_device)
    old.load_state_dict(block.state_dict())
    assert torch.equal(old(make()).features, want)


# ---- orthogonalisation -----------------------------------------------------------------------------------------------------
def test_many_equal_singular_values(cuda_device):
    """16384 orthogonal rows: every singular value is 1 / 128 of the norm, and the result is a multiple of the matrix that the polynomial
    on one number gives.  A step adds up to three roundings of 2.7 2^-24 and the sums' sqrt(6 k / 16), here over k = 16384 three times."""
    h = torch.ones(1, 1, device=cuda_device)
    while h.shape[0] < 16384:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    g = torch.Generator(device=cuda_device).manual_seed(4)
    h = h * (2.0 * torch.randint(0, 2, (16384,), device=cuda_device, generator=g) - 1)      # other signs for the columns
    got = optim.orthogonalize(h)
    a, b, c = optim.COEFFICIENTS
    t = 1.0 / 128
    for _ in range(5):
        t = a * t + b * t ** 3 + c * t ** 5
    want = t / 128                                             # the entries of h / |h| times the ratio of t to 1 / 128
    err = (got.double() - want * h.double()).norm() / (want * 16384)
    assert float(err) <= (40 + 5 * 3 * (6 * 16384 / 16) ** 0.5) * U


def test_lists_and_views_as_near_as_single_matrices(cuda_device):
    """matrices at least twice as wide as high, so that no direction is amplified beyond the result itself: three roundings a step of up to
    2.7 2^-24 each over five steps make 40, and the sums over k in steps of 16 add sqrt(6 k / 16) of one rounding each, one over n and two
    over m a step"""
    g = torch.Generator(device=cuda_device).manual_seed(7)
    shapes = [(16, 135)] + [(16, 432)] * 4 + [(432, 16), (128, 384), (64, 864), (256, 2304), (300, 7)]
    mats = [torch.randn(s, device=cuda_device, generator=g) for s in shapes]
    base = torch.randn(60, 400, device=cuda_device, generator=g)
    mats += [base[:, ::2], base[1::3], base.t(), base.t()[::2]]
    batch = torch.randn(3, 20, 50, device=cuda_device, generator=g)
    outs = list(optim.orthogonalize(mats)) + list(optim.orthogonalize(batch).unbind(0)) + list(optim.orthogonalize([m.bfloat16() for m in mats]))
    for o, m in zip(outs, mats + list(batch.unbind(0)) + [m.bfloat16() for m in mats]):
        want, k = reference(m), (min(m.shape), max(m.shape))
        sums = 5 * ((6 * k[1] / 16) ** 0.5 + 2 * (6 * k[0] / 16) ** 0.5)
        rel = float((o.double() - want).norm() / want.norm())
        assert rel <= (40 + sums) * U + torch.finfo(m.dtype).eps / 2, (tuple(m.shape), rel)


# ---- the longest list of a lookup ------------------------------------------------------------------------------------------
def test_lookup_of_nearly_2_31_entries(cuda_device):
    n, m = 2 ** 31 - 2 ** 20 - 1, 3
    g = torch.Generator(device=cuda_device).manual_seed(8)
    index = torch.randint(-1, m + 1, (n,), device=cuda_device, dtype=torch.int32, generator=g)
    table = torch.tensor([[1.0], [2.0], [4.0]], device=cuda_device, requires_grad=True)
    out = scatter.lookup_rows(table, index)
    parts = [slice(k, min(n, k + 2 ** 27)) for k in range(0, n, 2 ** 27)]
    values = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.0], device=cuda_device)
    assert all(torch.equal(out.detach()[p, 0], values[index[p].long() + 1]) for p in parts)
    up = torch.empty(n, 1, device=cuda_device)
    up.normal_(generator=g)
    got, = torch.autograd.grad(out, table, up)
    del out
    for v in range(m):
        total = size = count = 0.0
        for p in parts:
            d = up[p, 0].double() * (index[p] == v)
            total, size, count = total + float(d.sum()), size + float(d.abs().sum()), count + float((index[p] == v).sum())
        # blocks of 64 on four levels: 3 (64 - 1) blocks and as many additions within the ends, and the last level's count / 64^4
        assert abs(float(got[v]) - total) <= (4 * 64 + 6 * 63 + count / 64 ** 4 + 2) * U * size


# ---- runs of empty samples -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("samples", [60, 1000, 2 ** 25])
def test_norm_with_runs_of_empty_samples(cuda_device, samples):
    """as without them; in no more time than the search takes (a step for each of 2^25 would be 18 s a pass)"""
    n = 9000
    rows = torch.zeros(samples, dtype=torch.int32, device=cuda_device)
    rows[[0, samples // 3, samples // 3 + 1, samples - 2]] = torch.tensor([1200, 1, 3799, 4000], dtype=torch.int32, device=cuda_device)
    off = torch.cat([rows.new_zeros(1), rows.cumsum(0, dtype=torch.int32)])
    x = torch.randn(n, 16, device=cuda_device)
    up = torch.randn(n, 16, device=cuda_device)
    w = torch.rand(16, device=cuda_device) + 0.5
    results = []
    for o in (off, torch.unique(off).int()):
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        y = norm.group_norm_act(leaves[0], 4, leaves[1], act="silu", offsets=o)
        torch.cuda.synchronize()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        y = norm.group_norm_act(leaves[0], 4, leaves[1], act="silu", offsets=o)
        grads = torch.autograd.grad(y, leaves, up)
        end.record()
        end.synchronize()
        results.append((y.detach(),) + grads)
        assert start.elapsed_time(end) < 5000
    for got, want in zip(*results):
        assert float((got - want).abs().max()) <= 64 * U * float(want.abs().max())      # the same pieces, summed in another order in 64 bits
