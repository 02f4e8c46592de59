"""Rows looked up by index and the table's gradient by sorted index (csrc/lookup.hip; scatter.lookup_rows, scatter.sort_index) against
plain float64 forms.  The forward is one product rounded once.  A gradient row of k entries is a sum in binary32 along a chain of at
most L F additions inside blocks of L levels (F = 16, 32 or 64 entries; a level is there if the one before has 256 blocks), a tail, 2 (F - 1)
blocks of each level but the last, and of that one 255 or, on the highest, k / F^L.  F = 16 up to 2^23 entries: L <= 4, 64 + 1 + 90 + 255.
F = 32 up to 2^24: L <= 4, 128 + 1 + 186 + 255.  F = 64: L = 3, 192 + 1 + 252 + 255, or k / 64^3 for the last; L = 4 (a list of 2^26),
256 + 1 + 378 + k / 64^4 <= 128.  Fewer than 828 + k / 64^3 roundings of partial sums no
larger than sum |dout|; then the scale and one rounding more:
|error| <= (828 + k / 64^3 + 1) * 2^-24 * sum |dout| |scale| + eps / 2 |value|."""
import pytest
import torch

from openpcdet_amd import scatter, vfe

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def make_index(n, m, kind, dev, g, dtype):
    u = torch.rand(n, device=dev, generator=g)
    if kind == "one":
        i = torch.full((n,), m // 2, device=dev)
    elif kind == "skewed":
        i = (u ** 6 * m).long()
    elif kind == "outside":
        i = (u * (m + 9)).long() - 4
    elif kind == "sorted":
        i = torch.sort((u * m).long())[0]
    else:
        i = (u * m).long().clamp(max=m - 1)
    return i.to(dtype)


def check(dev, n, m, w, dtype=torch.float32, itype=torch.int64, kind="uniform", scale=1.0, seed=0, misalign=False):
    g = torch.Generator(device=dev).manual_seed(seed + 13 * n + m)
    index = make_index(n, m, kind, dev, g, itype)
    table = torch.randn(m, w, device=dev, generator=g).to(dtype)
    dout = torch.randn(n, w, device=dev, generator=g).to(dtype)
    if misalign:
        table = torch.cat([table.new_zeros(1), table.reshape(-1)])[1:].view(m, w)
        dout = torch.cat([dout.new_zeros(1), dout.reshape(-1)])[1:].view(n, w)
    leaf = table.requires_grad_(True)
    out = scatter.lookup_rows(leaf, index, scale=scale)
    inside = (index >= 0) & (index < m)
    at = index.long().clamp(0, m - 1)
    scale32 = float(torch.tensor(scale, dtype=torch.float32))
    want = torch.where(inside.unsqueeze(1), (table.detach().float() * scale32)[at], torch.zeros((), device=dev)).to(dtype)
    assert torch.equal(out.detach(), want), "forward of %d from %d x %d" % (n, m, w)
    got, = torch.autograd.grad(out, leaf, dout, retain_graph=True)
    d64 = dout.double() * inside.unsqueeze(1)
    ref = torch.zeros(m, w, dtype=torch.float64, device=dev).index_add_(0, at, d64) * scale32
    mag = torch.zeros(m, w, dtype=torch.float64, device=dev).index_add_(0, at, d64.abs()) * abs(scale32)
    count = torch.bincount(at[inside], minlength=m).double().unsqueeze(1)
    chain = torch.minimum(count, 828 + count / 64 ** 3) + 1
    bound = chain * U * mag
    bound = bound + torch.finfo(dtype).eps / 2 * (ref.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = (got.double() - ref).abs()
    assert got.dtype == dtype and not bool((err > bound).any()), "gradient of %d into %d x %d: %.3g" % (n, m, w, float((err - bound).max()))
    assert torch.equal(torch.autograd.grad(out, leaf, dout, retain_graph=True)[0], got)
    s = scatter.sort_index(index, m)
    shared = scatter.lookup_rows(leaf, index, scale=scale, sort=s)
    assert torch.equal(torch.autograd.grad(shared, leaf, dout)[0], got)


def check_sort(dev, n, m, kind, itype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + n)
    index = make_index(n, m, kind, dev, g, itype)
    s = scatter.sort_index(index, m)
    key = torch.where((index >= 0) & (index < m), index.long(), torch.full((), m, device=dev))
    keys, order = torch.sort(key, stable=True)
    assert torch.equal(s.order.long(), order) and torch.equal(s.keys.long(), keys)
    assert torch.equal(s.offsets.long(), torch.searchsorted(keys, torch.arange(m + 1, device=dev)))


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
@pytest.mark.parametrize("kind", ["uniform", "skewed", "one", "outside", "sorted"])
def test_sort_is_stable(cuda_device, kind, itype):
    for n, m in ((1, 1), (2, 1), (63, 5), (64, 300), (65, 70000), (1023, 255), (1025, 256), (8192, 257), (8192, 1 << 20), (8193, 1), (8193, 2047),
                 (20000, 2048), (100003, 33), (100003, 3000000), (262144, 4194303), (50001, 4194304), (70000, 2000000000)):
        if m < 100000000 or kind == "uniform" and itype == torch.int64:      # offsets of 2e9 rows: once
            check_sort(cuda_device, n, m, kind, itype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["uniform", "skewed", "one", "outside", "sorted"])
def test_lookup_and_gradient(cuda_device, dtype, kind):
    check(cuda_device, 83, 10, 64, dtype, kind=kind, scale=8.0)
    check(cuda_device, 70000, 31007, 32, dtype, torch.int32, kind)
    check(cuda_device, 40000, 700, 37, dtype, kind=kind, scale=-0.3)


@pytest.mark.parametrize("n,m,w", [(1, 1, 1), (1, 5, 3), (63, 1, 8), (64, 1, 8), (65, 2, 16), (1024, 1, 4), (33000, 1, 4), (70001, 1, 4),
                                   (2100000, 3, 2), (5, 200001, 24), (300, 7, 1), (2049, 64, 130), (100, 9, 2050)])
def test_sizes(cuda_device, n, m, w):
    for kind in ("one", "uniform"):
        check(cuda_device, n, m, w, torch.bfloat16, kind=kind, scale=1.0)
        check(cuda_device, n, m, w, torch.float32, torch.int32, kind=kind, scale=3.0)


def test_alignment_shapes_and_empty(cuda_device):
    check(cuda_device, 5000, 100, 32, torch.bfloat16, misalign=True)
    check(cuda_device, 5000, 100, 32, torch.float32, misalign=True)
    table = torch.randn(6, 4, 5, device=cuda_device, requires_grad=True)
    index = torch.tensor([[0, 5, -1], [2, 2, 6]], device=cuda_device)
    out = scatter.lookup_rows(table, index)
    assert out.shape == (2, 3, 4, 5) and torch.equal(out[0, 0], table[0]) and torch.equal(out[1, 1], table[2])
    assert float(out[0, 2].abs().max()) == 0 and float(out[1, 2].abs().max()) == 0
    out.sum().backward()                                                  # a gradient of stride 0
    assert torch.equal(table.grad.amax((1, 2)).cpu(), torch.tensor([1.0, 0, 2, 0, 0, 1]))
    strided = torch.randn(8, 40, device=cuda_device)[:, ::2]
    pick = torch.arange(16, device=cuda_device)[::2] // 2
    assert torch.equal(scatter.lookup_rows(strided, pick), strided[pick])
    vector = torch.randn(9, device=cuda_device, requires_grad=True)       # rows of one value
    assert torch.equal(scatter.lookup_rows(vector, pick), vector[pick])
    for n, m, w in ((0, 4, 8), (5, 0, 8), (5, 4, 0), (0, 0, 3)):
        t = torch.zeros(m, w, device=cuda_device, requires_grad=True)
        o = scatter.lookup_rows(t, torch.zeros(n, dtype=torch.long, device=cuda_device))
        assert o.shape == (n, w) and float(o.abs().sum()) == 0
        o.sum().backward()
        assert t.grad.shape == (m, w) and float(t.grad.abs().sum()) == 0
    big = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32 + 1, 1], device=cuda_device)   # int64 entries that 32 bits would wrap into the table
    assert torch.equal(scatter.lookup_rows(table.detach(), big)[:3], torch.zeros(3, 4, 5, device=cuda_device))
    assert scatter.sort_index(big, 6).keys.tolist() == [1, 6, 6, 6]


def test_special_values(cuda_device):
    table = torch.tensor([[1.0, float("inf")], [float("nan"), -2.0], [3.0, 4.0]], device=cuda_device, requires_grad=True)
    out = scatter.lookup_rows(table, torch.tensor([2, -1, 0], device=cuda_device), scale=2.0)
    assert torch.equal(out.detach().cpu(), torch.tensor([[6.0, 8.0], [0.0, 0.0], [2.0, float("inf")]]))
    up = torch.tensor([[1.0, 1.0], [float("nan"), float("nan")], [1.0, float("inf")]], device=cuda_device)
    g, = torch.autograd.grad(out, table, up)                              # the dropped entry's NaN goes nowhere
    assert torch.equal(g.cpu(), torch.tensor([[2.0, float("inf")], [0.0, 0.0], [2.0, 2.0]]))


def test_offsets_past_32_bits(cuda_device):
    m, w = 17000000, 256                                                  # 4.35e9 half-precision values
    table = torch.zeros(m, w, dtype=torch.float16, device=cuda_device)
    rows = torch.tensor([0, 8388608, 16777216, m - 1], device=cuda_device)
    table[rows] = torch.arange(1, 5, device=cuda_device, dtype=torch.float16).unsqueeze(1)
    assert torch.equal(scatter.lookup_rows(table, rows)[:, 255].cpu(), torch.arange(1, 5, dtype=torch.float16))
    del table
    d = torch.ones(4, w, dtype=torch.float16, device=cuda_device)
    leaf = torch.empty(m, w, dtype=torch.float16, device=cuda_device, requires_grad=True)
    g, = torch.autograd.grad(scatter.lookup_rows(leaf, rows), leaf, d)
    assert float(g.sum(dtype=torch.float64)) == 4 * w and torch.equal(g[rows], d)


def test_streams_and_graph(cuda_device):
    torch.manual_seed(1)
    for n, m in ((500, 40), (60000, 5000)):
        table = torch.randn(m, 32, device=cuda_device)
        idx = [torch.randint(-1, m, (n,), device=cuda_device) for _ in range(3)]
        ups = [torch.randn(n, 32, device=cuda_device) for _ in range(3)]

        def step(i, up):
            t = table.detach().requires_grad_(True)
            out = scatter.lookup_rows(t, i, scale=0.5)
            return out.detach(), torch.autograd.grad(out, t, up)[0]

        want = [step(i, u) for i, u in zip(idx, ups)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(idx[1], ups[1])
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want[1]))
        i0, u0 = idx[0].clone(), ups[0].clone()
        graphs = []
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                out = step(i0, u0)
            graphs.append((gr, out))
        for k in (1, 2, 0, 1):
            i0.copy_(idx[k])
            u0.copy_(ups[k])
            for gr, _ in graphs:
                gr.replay()
            step(idx[2], ups[2])
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(p, q) for p, q in zip(out, want[k]))


def test_voxel_encoder_layer_uses_it(cuda_device):
    """PFNLayerV2's broadcast of the voxel maxima to the points: same values as indexing, same gradient up to the order of sums"""
    torch.manual_seed(3)
    layer = vfe.PFNLayerV2(10, 32).to(cuda_device)
    x = torch.randn(4000, 10, device=cuda_device)
    inv = torch.randint(0, 500, (4000,), device=cuda_device, dtype=torch.int32)
    a = x.clone().requires_grad_(True)
    out = layer(a, inv, 500)
    up = torch.randn_like(out)
    got, = torch.autograd.grad(out, a, up)
    b = x.clone().requires_grad_(True)
    h = layer.relu(layer.norm(layer.linear(b)))
    top = scatter.scatter_max(h, inv, dim=0, dim_size=500)[0]
    want_out = torch.cat([h, top[inv.long(), :]], dim=1)
    want, = torch.autograd.grad(want_out, b, up)
    assert torch.equal(out, want_out)
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-5)


def test_refusals_on_the_device(cuda_device):
    t, i = torch.zeros(4, 8, device=cuda_device), torch.zeros(3, dtype=torch.long, device=cuda_device)
    with pytest.raises(RuntimeError):
        scatter.lookup_rows(t.cpu(), i)
    with pytest.raises(RuntimeError):
        scatter.lookup_rows(t, i.cpu())
    with pytest.raises(TypeError):
        scatter.lookup_rows(t.double(), i)
    with pytest.raises(TypeError):
        scatter.lookup_rows(t, i.short())
    with pytest.raises(ValueError):
        scatter.lookup_rows(t[0, 0], i)
    with pytest.raises(ValueError):
        scatter.lookup_rows(t, i, sort=scatter.sort_index(i, 5))
    with pytest.raises(ValueError):
        scatter.lookup_rows(t, i, sort=scatter.sort_index(i[:2], 4))
    with pytest.raises(ValueError):
        scatter.sort_index(i, 0)
