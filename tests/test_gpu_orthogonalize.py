"""Newton-Schulz orthogonalisation (csrc/orthogonalize.hip; optim.orthogonalize, optim.Muon) against the iteration in float64.

Tolerance.  A step is X <- p(X X^T) X with |p| <= a + |b| + |c| on [0, 1.3].  Let d be the relative error of a product's operands
(two f16 halves hold 22 bits and the sign of the second one: at most 2^-22, 2^-24 in the root mean square, the dropped product of the
second halves included, whatever the matrices' dtype): it enters X at most three times a step (A, A A, B X), scaled by at most a + 2 |b| + 3 |c| = 19 of
the value it enters, and the later steps carry it with a gain of at most a = 3.4445 each (the polynomial's slope at 0 is its largest on
the range).  Over five steps that is at most 19 (1 + .. + 3.4445^4) d = 19 * 198 d <= 3800 d relative to the result: `bound(.., tight=False)`,
for any spectrum.  Where no direction is amplified by more than the result itself (random matrices at least twice as wide as high: all
singular values within a factor of six), an error stays the share of the result that it was, and three roundings a step of up to
2.7 d each (19 / 7, the mean of the scaling over the range) over five steps make 40 d.  The sums add to it: a product over k is
6 k / 16 additions of one rounding (2^-24 of a running sum no larger than the result) each, of either sign, sqrt(6 k / 16) of them
together; a step has one such sum over n and two over m, and five steps add up linearly at worst.  Results are rounded once (eps / 2)."""
import copy

import numpy as np
import pytest
import torch

from openpcdet_amd import backbones, optim

pytestmark = pytest.mark.gpu
A, B, C = optim.COEFFICIENTS


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


def rel(got, want):
    return float((got.double() - want).norm() / want.norm().clamp(min=1e-300))


def bound(dtype, tight, shape=(1, 1)):
    d, m, n = 2.0 ** -24, min(shape), max(shape)
    sums = 5 * ((6 * n / 16) ** 0.5 + 2 * (6 * m / 16) ** 0.5) * 2.0 ** -24
    return (40 if tight else 3800) * d + sums + torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("r,c", [(1, 1), (1, 7), (9, 1), (2, 2), (3, 5), (16, 135), (16, 432), (31, 33), (64, 64), (65, 129), (128, 1152), (333, 77),
                                 (300, 301), (512, 512), (1000, 130), (130, 5001)])
def test_matrix(cuda_device, dtype, r, c):
    g = torch.Generator(device=cuda_device).manual_seed(r * 1000 + c)
    m = (torch.randn(r, c, device=cuda_device, generator=g) * 1e-3).to(dtype)
    got = optim.orthogonalize(m)
    assert got.shape == m.shape and got.dtype == dtype
    assert rel(got, reference(m)) <= bound(dtype, min(r, c) * 2 <= max(r, c), (r, c))
    assert torch.equal(got, optim.orthogonalize(m))                      # the same bits again


def test_large_tiles(cuda_device):
    for dtype, r, c in ((torch.float32, 1100, 2300), (torch.bfloat16, 2050, 2300), (torch.float16, 5000, 900)):
        g = torch.Generator(device=cuda_device).manual_seed(r)
        m = torch.randn(r, c, device=cuda_device, generator=g).to(dtype)
        assert rel(optim.orthogonalize(m), reference(m)) <= bound(dtype, 2 * min(r, c) <= max(r, c), (r, c))


def test_spectrum(cuda_device):
    """a chosen spectrum: the polynomial acts on each singular value, the vectors stay"""
    g = torch.Generator(device=cuda_device).manual_seed(5)
    u = torch.linalg.qr(torch.randn(96, 96, device=cuda_device, generator=g, dtype=torch.float64))[0]
    v = torch.linalg.qr(torch.randn(400, 96, device=cuda_device, generator=g, dtype=torch.float64))[0]
    s = torch.logspace(0, -3, 96, dtype=torch.float64, device=cuda_device)
    m = ((u * s) @ v.t().contiguous()).float()
    got = optim.orthogonalize(m).double()
    t = s / (s.square().sum().sqrt() + 1e-7)
    for _ in range(5):
        t = A * t + B * t ** 3 + C * t ** 5
    # the input's own rounding to float32 (2^-24 of the largest entry) is amplified like everything else
    assert rel(got, (u * t) @ v.t().contiguous()) <= 2 * bound(torch.float32, False)


def test_steps_and_scale(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(6)
    m = torch.randn(40, 90, device=cuda_device, generator=g)
    for steps in (0, 1, 2, 3, 8):
        assert rel(optim.orthogonalize(m, steps=steps), reference(m, steps)) <= 3800 * 2.0 ** -24 * 3.4445 ** max(0, steps - 5)
        assert rel(optim.orthogonalize(m.t(), steps=steps), reference(m, steps).t()) <= 3800 * 2.0 ** -24 * 3.4445 ** max(0, steps - 5)
    other = (2.0, -1.5, 0.5)
    assert rel(optim.orthogonalize(m, steps=10, coefficients=other), reference(m, 10, coefficients=other)) <= 40 * 2.0 ** -24 * 10
    for scale in (1e-30, 1e-6, 1e30):                                    # squares beyond binary32, and the eps that matters
        assert rel(optim.orthogonalize(m * scale), reference(m * scale)) <= 3800 * 2.0 ** -24
    assert float(optim.orthogonalize(torch.zeros(5, 9, device=cuda_device)).abs().max()) == 0.0
    assert bool(torch.isnan(optim.orthogonalize(torch.zeros(5, 9, device=cuda_device), eps=0.0)).all())
    m[3, 4] = float("nan")
    both = optim.orthogonalize([m, m[:, 10:]])
    assert bool(torch.isnan(both[0]).all()) and bool(torch.isfinite(both[1]).all())
    big = torch.randn(70, 300, device=cuda_device)
    big[3, 4] = float("inf")
    assert bool(torch.isnan(optim.orthogonalize(big)).all())
    for grow in ((4.0, 0.0, 0.0), (0.5, 0.0, 0.0)):                      # coefficients that let the values grow or fall: the scales follow
        assert rel(optim.orthogonalize(big[10:], steps=6, coefficients=grow), reference(big[10:], 6, coefficients=grow)) <= 100 * 2.0 ** -24
    # 3 x - 2 x^3 keeps [0, sqrt(2)], but its slope at that end is 3 - 6 * 2 = -9: with 1 % to spare a step the bound of the values goes
    # 1.43, 1.56, 2.9, 39, 1.2e5, 3.7e15 while they stay below 1.42, and words kept against it hold nothing.  Refused, not computed wrongly.
    with pytest.raises(ValueError, match="bounds"):
        optim.orthogonalize(big[10:], steps=6, coefficients=(3.0, -2.0, 0.0))


def test_lists_batches_and_strides(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(7)
    shapes = [(16, 135)] + [(16, 432)] * 4 + [(432, 16), (1, 1), (128, 384), (0, 5), (70, 64), (3, 0)]
    mats = [torch.randn(s, device=cuda_device, generator=g) for s in shapes]
    mats += [m.to(torch.bfloat16) for m in mats[:3]]
    outs = optim.orthogonalize(tuple(mats))
    assert isinstance(outs, tuple) and all(o.shape == m.shape and o.dtype == m.dtype for o, m in zip(outs, mats))
    for o, m in zip(outs, mats):
        if m.numel():
            assert rel(o, reference(m)) <= bound(m.dtype, False)
    many = [torch.randn(8, 24, device=cuda_device, generator=g) for _ in range(150)]          # more than one call takes
    for o, m in zip(optim.orthogonalize(many), many):
        assert rel(o, reference(m)) <= bound(torch.float32, False)
    batch = torch.randn(3, 20, 50, device=cuda_device, generator=g)
    ob = optim.orthogonalize(batch)
    assert ob.shape == batch.shape and torch.equal(ob[1], optim.orthogonalize([batch[0], batch[1], batch[2]])[1])
    wide = torch.randn(50, 80, device=cuda_device, generator=g)
    for view in (wide[:, ::2], wide.t(), wide[1::3]):
        assert rel(optim.orthogonalize(view), reference(view)) <= bound(torch.float32, False)
    assert optim.orthogonalize([]) == [] and optim.orthogonalize(torch.zeros(0, 4, 4, device=cuda_device)).shape == (0, 4, 4)
    same = optim.orthogonalize([wide, wide])                             # the same matrix twice
    assert torch.equal(same[0], same[1])


def test_streams_and_graph(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(8)
    data = [[torch.randn(s, device=cuda_device, generator=g) for s in ((64, 300), (200, 90))] for _ in range(3)]
    want = [optim.orthogonalize(d) for d in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = optim.orthogonalize(data[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want[1]))
    static = [t.clone() for t in data[0]]
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = optim.orthogonalize(static)
        graphs.append((gr, out))
    for k in (1, 2, 0, 1):
        for s, t in zip(static, data[k]):
            s.copy_(t)
        for gr, _ in graphs:
            gr.replay()
        optim.orthogonalize(data[2])
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, want[k]))


@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (False, 0.1)])
def test_muon_step(cuda_device, nesterov, decay):
    g = torch.Generator(device=cuda_device).manual_seed(9)
    shapes = [(16, 3, 3, 3, 5), (32, 3, 3, 3, 16), (90, 16), (4, 4)]
    params = [torch.nn.Parameter(torch.randn(s, device=cuda_device, generator=g)) for s in shapes] + [torch.nn.Parameter(torch.zeros(3, 3, device=cuda_device))]
    opt = optim.Muon(params, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=decay)
    p64 = [p.detach().double().clone() for p in params]
    bufs = [torch.zeros_like(p) for p in p64]
    for _ in range(3):
        for k, p in enumerate(params[:-1]):                              # the last one never has a gradient
            p.grad = torch.randn(p.shape, device=cuda_device, generator=g)
            bufs[k] = 0.9 * bufs[k] + p.grad.double()
            u = p.grad.double() + 0.9 * bufs[k] if nesterov else bufs[k]
            o = reference(u.view(u.shape[0], -1))
            p64[k] = p64[k] * (1 - 0.05 * decay) - 0.05 * max(1.0, o.shape[0] / o.shape[1]) ** 0.5 * o.view(u.shape)
        opt.step()
    for p, q in zip(params, p64):
        assert float((p.detach().double() - q).norm()) <= 3 * 0.05 * 2.4 * 3800 * 2.0 ** -24 * max(p.shape) ** 0.5 + 8 * 2.0 ** -24 * float(q.norm())
    state = copy.deepcopy(opt.state_dict())                              # a loaded state shares its tensors with the source
    again = optim.Muon([torch.nn.Parameter(p.detach().clone()) for p in params], lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=decay)
    again.load_state_dict(state)
    for p, q in zip(params, again.param_groups[0]["params"]):
        if p.grad is not None:
            q.grad = p.grad.clone()
    opt.step()
    again.step()
    assert all(torch.equal(p, q) for p, q in zip(params, again.param_groups[0]["params"]))


def test_refusals_on_the_device(cuda_device):
    m = torch.zeros(4, 4, device=cuda_device)
    for bad in (m[0], m.view(1, 2, 2, 4), [m, m[0]], [m, None]):
        with pytest.raises(ValueError):
            optim.orthogonalize(bad)
    for kw in (dict(steps=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(coefficients=(1.0, 2.0))):
        with pytest.raises(ValueError):
            optim.orthogonalize(m, **kw)
    for bad in (m.double(), [m, m.long()]):
        with pytest.raises(TypeError):
            optim.orthogonalize(bad)
    with pytest.raises(RuntimeError):
        optim.orthogonalize([m, m.cpu()])


def test_offsets_past_32_bits(cuda_device):
    m, n = 2112, 2 ** 20                                                 # 2.2e9 elements
    a, b, c = optim.COEFFICIENTS
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x = torch.randn(m, n, device=cuda_device, dtype=torch.bfloat16, generator=g)
    got = optim.orthogonalize(x, steps=2)
    gram = torch.zeros(m, m, dtype=torch.float64, device=cuda_device)
    for k in range(0, n, 2 ** 16):
        part = x[:, k:k + 2 ** 16].double()
        gram += part @ part.t().contiguous()
    norm = float(gram.diagonal().sum().sqrt()) + 1e-7
    gram /= norm * norm
    eye = torch.eye(m, dtype=torch.float64, device=cuda_device)
    total = eye
    for _ in range(2):                                                   # the products with X come to one matrix: A follows from A
        step = a * eye + b * gram + c * (gram @ gram)
        total, gram = step @ total, step @ gram @ step
    for k in (0, n // 2 - 1000, n - 4096):
        assert rel(got[:, k:k + 4096], total @ (x[:, k:k + 4096].double() / norm)) <= bound(torch.bfloat16, True, (m, n))


def test_muon_refuses_before_it_changes_anything(cuda_device):
    ok, bad = torch.nn.Parameter(torch.ones(4, 4, device=cuda_device)), torch.nn.Parameter(torch.ones(4, 4, device=cuda_device, dtype=torch.float64))
    opt = optim.Muon([ok, bad])
    ok.grad, bad.grad = torch.ones_like(ok), torch.ones_like(bad)
    with pytest.raises(TypeError, match="float64"):
        opt.step()
    assert float((ok - 1).abs().max()) == 0 and not opt.state


def test_training_step_with_all_of_them(cuda_device):
    """points -> dynamic voxel encoder (rows looked up) -> residual backbone with group norm -> dense -> backward -> Muon on the
    convolutions, AdamW on the rest: every parameter moves, the same way twice"""
    from openpcdet_amd import vfe
    rng, vs, grid = [0.0, -8.0, -2.0, 16.0, 8.0, 2.0], [0.25, 0.25, 0.1], [64, 64, 40]

    def build():
        torch.manual_seed(11)
        enc = vfe.DynamicVoxelVFE(dict(USE_NORM=True, WITH_DISTANCE=False, USE_ABSLOTE_XYZ=True, NUM_FILTERS=[32, 16]), 4, vs, grid, rng)
        net = backbones.VoxelResBackBone8x(input_channels=16, grid_size=np.array(grid), model_cfg={"NORM_GROUPS": 4})
        model = torch.nn.ModuleList([enc, net]).to(cuda_device).train()
        convs = [p for p in net.parameters() if p.dim() >= 2]
        rest = [p for p in model.parameters() if not any(p is q for q in convs)]
        return model, optim.Muon(convs, lr=0.02), torch.optim.AdamW(rest, lr=1e-3)

    r = np.random.default_rng(3)
    n = 4000
    pts = np.stack([r.integers(0, 2, n), r.uniform(0, 16, n), r.uniform(-8, 8, n), r.uniform(-2, 2, n), r.uniform(0, 1, n)], 1).astype(np.float32)
    pts = torch.from_numpy(pts[np.argsort(pts[:, 0], kind="stable")]).to(cuda_device)
    runs = []
    for _ in range(2):
        model, muon, adam = build()
        before = [p.detach().clone() for p in model.parameters()]
        grads = None
        for _ in range(2):
            bd = model[1](model[0]({"points": pts, "batch_size": 2}))
            dense = bd["encoded_spconv_tensor"].dense()
            loss = dense.square().mean()
            muon.zero_grad(set_to_none=True)
            adam.zero_grad(set_to_none=True)
            loss.backward()
            grads = [p.grad for p in model.parameters()]
            assert all(g is not None and bool(torch.isfinite(g).all()) for g in grads)
            muon.step()
            adam.step()
        assert all(not torch.equal(p, q) for p, q in zip(model.parameters(), before))
        runs.append([p.detach().clone() for p in model.parameters()])
    assert all(torch.allclose(p, q, rtol=1e-3, atol=1e-4) for p, q in zip(*runs))
