"""What is timed of the training-step operators beside the sparse convolutions: group norm with an activation over the rows of a
sparse tensor (or a dense channels-last map), rows looked up in a table with their gradient by sorted index, and the Newton-Schulz
orthogonalisation of weight updates.

`run` computes a case in plain torch operations, or, where `own` is true, through the framework.  Sizes are those of the sparse
backbones (16 to 128 channels, 10^2 to 10^6 active sites, 3 x 3 x 3 convolutions), of the dynamic voxel encoders (points looked up in
their voxels) and generic ones for dense layers and large tables."""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)        # the quintic a x + b x^3 + c x^5 on the singular values
STEPS = 5
NORM_EPS = 1e-5
ORTHO_EPS = 1e-7

# every convolution of a residual 8x voxel backbone with 5 input channels as (Cout) x (K Cin)
RES8X = ",".join(["16x135"] + ["16x432"] * 4 + ["32x432"] + ["32x864"] * 4 + ["64x864"] + ["64x1728"] * 4 + ["128x1728"]
                 + ["128x3456"] * 4 + ["128x384"])


def listed():
    return [
        # one frame's deepest level in serving: the launch is what counts
        dict(name="norm, few rows", op="norm", rows=300, samples=1, channels=16, groups=4, dtype="float32", act="relu", residual=False,
             layout="ragged", train=False),
        # the second normalisation of a residual block at a middle level, four frames, forward and backward
        dict(name="norm, residual block step", op="norm", rows=117301, samples=4, channels=64, groups=8, dtype="bfloat16", act="silu",
             residual=True, layout="ragged", train=True),
        # a dense bird's-eye map kept channels last, 188 x 188 cells of three frames, groups of 3 channels
        dict(name="norm, dense map", op="norm", rows=3 * 188 * 188, samples=3, channels=96, groups=32, dtype="float16", act="relu",
             residual=False, layout="dense", train=False),
        # the widest level of a large training batch, forward and backward in 32 bits
        dict(name="norm, widest level step", op="norm", rows=520013, samples=8, channels=128, groups=16, dtype="float32", act="gelu",
             residual=False, layout="ragged", train=True),
        # class rows for the boxes that one head keeps in serving
        dict(name="lookup, kept boxes", op="lookup", tokens=83, rows=10, width=64, dtype="float32", index="int64", spread="uniform",
             outside=0.0, scale=8.0, train=False),
        # points of a frame look their voxel's features up (a dynamic encoder's second layer); 5 % lie outside the range
        dict(name="lookup, points in voxels", op="lookup", tokens=240000, rows=31007, width=32, dtype="float32", index="int32",
             spread="scan", outside=0.05, scale=1.0, train=True),
        # a table much longer than the list, rows of odd width
        dict(name="lookup, sparse in long table", op="lookup", tokens=70001, rows=999983, width=37, dtype="float16", index="int64",
             spread="uniform", outside=0.0, scale=6.0, train=True),
        # a large table under a skewed distribution: one row takes a large share of the list
        dict(name="lookup, large and skewed", op="lookup", tokens=1048579, rows=250007, width=128, dtype="bfloat16", index="int64",
             spread="skewed", outside=0.0, scale=math.sqrt(128.0), train=True),
        # one narrow layer: latency
        dict(name="orthogonalize, one layer", op="orthogonalize", shapes="16x432", dtype="float32"),
        # every convolution of a residual backbone, as an optimiser's step has them
        dict(name="orthogonalize, backbone", op="orthogonalize", shapes=RES8X, dtype="float32"),
        # odd sizes, one taller than wide
        dict(name="orthogonalize, odd layers", op="orthogonalize", shapes="1001x2003,1201x577,77x333", dtype="float32"),
        # one wide dense layer
        dict(name="orthogonalize, wide layer", op="orthogonalize", shapes="2048x4096", dtype="bfloat16"),
    ]


def _between(rng, low, high):
    """a whole number between `low` and `high`, even over the logarithm"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_norm(rng):
    channels = rng.choice([8, 16, 24, 32, 37, 48, 64, 96, 128, 130, 192, 256])
    groups = rng.choice([g for g in (1, 2, 3, 4, 5, 8, 16, 32, 37, 64) if channels % g == 0])
    most = min(1200000, 520013 * 128 // channels)
    samples = rng.randint(1, 8)
    train = rng.random() < 0.6
    # the derivative of a ReLU steps at zero, where 32 bits do not decide the side: its gradients are not compared
    act = rng.choice(["none", "silu", "gelu"] if train else ["none", "relu", "silu", "gelu"])
    layout = rng.choice(["ragged", "ragged", "mixed", "dense"])
    rows = _between(rng, 16, most)
    if layout == "dense":
        rows = max(1, rows // samples) * samples
    return dict(op="norm", rows=rows, samples=samples, channels=channels, groups=groups, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                act=act, residual=rng.random() < 0.4, layout=layout, train=train)


def _draw_lookup(rng):
    width = rng.choice([1, 3, 8, 16, 32, 37, 64, 100, 128, 200, 256])
    most = 1048579 * 128 // width
    tokens = _between(rng, 1, min(4000000, most))
    return dict(op="lookup", tokens=tokens, rows=_between(rng, 1, min(1000000, most)), width=width,
                dtype=rng.choice(["float32", "bfloat16", "float16"]), index=rng.choice(["int32", "int64"]),
                spread=rng.choice(["uniform", "skewed", "scan"]), outside=rng.choice([0.0, 0.0, 0.05, 0.5]),
                scale=rng.choice([1.0, 0.125, math.sqrt(width)]), train=rng.random() < 0.7)


def _draw_orthogonalize(rng):
    shapes, left = [], 2048 * 2048 * 4096
    for _ in range(rng.choice([1, 1, 2, 5, 12])):
        r, c = _between(rng, 2, 2048), _between(rng, 2, 4096)
        cost = min(r, c) ** 2 * max(r, c)
        if cost <= left:
            shapes.append("%dx%d" % (r, c))
            left -= cost
    return dict(op="orthogonalize", shapes=",".join(shapes), dtype=rng.choice(["float32", "bfloat16", "float16"]))


def draw(rng):
    return rng.choice([_draw_norm, _draw_lookup, _draw_orthogonalize])(rng)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _prepare_norm(case, g):
    dev, dtype = "cuda", getattr(torch, case["dtype"])
    n, c, b = case["rows"], case["channels"], case["samples"]
    # a convolution's outputs: a mean and a spread of its own for each channel
    x = torch.randn(n, c, device=dev, generator=g)
    x = x * (torch.rand(c, device=dev, generator=g) * 1.5 + 0.25) + torch.randn(c, device=dev, generator=g) * 0.7
    s = dict(case=case, x=x.to(dtype), weight=torch.rand(c, device=dev, generator=g) + 0.5, bias=torch.randn(c, device=dev, generator=g) * 0.3,
             residual=torch.randn(n, c, device=dev, generator=g).to(dtype) if case["residual"] else None,
             dy=(torch.randn(n, c, device=dev, generator=g) * 0.05).to(dtype) if case["train"] else None, offsets=None, order=None)
    if case["layout"] == "dense":
        sample = torch.arange(b, device=dev).repeat_interleave(n // b)
    else:
        # frames of unequal size; of three or more, the second is empty
        cuts = torch.sort(torch.rand(b - 1, device=dev, generator=g) * n)[0].long()
        if b >= 3:
            cuts[1] = cuts[0]
        edges = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), n)])
        sample = torch.repeat_interleave(torch.arange(b, device=dev), edges[1:] - edges[:-1], output_size=n)
        if case["layout"] == "mixed":        # rows of the frames in any order
            sample = sample[torch.randperm(n, device=dev, generator=g)]
            s["order"] = torch.sort(sample, stable=True)[1].int()
        s["offsets"] = edges.int()
    s["sample"] = sample
    for k in ("x", "weight", "bias", "residual"):
        if case["train"] and s[k] is not None:
            s[k].requires_grad_(True)
    return s


def _prepare_lookup(case, g):
    dev, dtype = "cuda", getattr(torch, case["dtype"])
    n, m, w = case["tokens"], case["rows"], case["width"]
    u = torch.rand(n, device=dev, generator=g, dtype=torch.float64)
    if case["spread"] == "uniform":
        index = (u * m).long()
    elif case["spread"] == "skewed":         # row k with a share of about 1 / (k + 1)
        index = (torch.exp(u * math.log(m + 1.0)) - 1.0).long()
        index = torch.randperm(m, device=dev, generator=g)[index.clamp(0, m - 1)]
    else:                                    # a scan: near cells hold many points, neighbours in the list share their cell
        cell = (u * u * m).long().clamp(0, m - 1)
        run = torch.arange(n, device=dev) // 3
        index = cell[run * 3]
    index = index.clamp(0, m - 1)
    if case["outside"] > 0:
        index = torch.where(torch.rand(n, device=dev, generator=g) < case["outside"], torch.full_like(index, -1), index)
    s = dict(case=case, index=index.to(getattr(torch, case["index"])), table=torch.randn(m, w, device=dev, generator=g).to(dtype),
             dout=(torch.randn(n, w, device=dev, generator=g) * 0.1).to(dtype) if case["train"] else None)
    if case["train"]:
        s["table"].requires_grad_(True)
    return s


def _prepare_orthogonalize(case, g):
    dev, dtype = "cuda", getattr(torch, case["dtype"])
    mats = []
    for r, c in _shapes(case):
        k = max(1, min(r, c) // 4)           # a gradient: a few strong directions over noise
        strength = torch.linspace(1.0, 0.1, k, device=dev)
        low = (torch.randn(r, k, device=dev, generator=g) * strength) @ torch.randn(k, c, device=dev, generator=g) / math.sqrt(k)
        mats.append(((low + 0.5 * torch.randn(r, c, device=dev, generator=g)) * 1e-3).to(dtype))
    return dict(case=case, matrices=mats)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return {"norm": _prepare_norm, "lookup": _prepare_lookup, "orthogonalize": _prepare_orthogonalize}[case["op"]](case, g)


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _by_sample(values, sample, count):
    """sums of the rows [N, G] of each sample, as products with the rows' memberships in slices of 512 rows, in 64 bits: [count, G]"""
    n, g = values.shape
    slices = (n + 511) // 512
    pad = slices * 512 - n
    member = (sample.unsqueeze(0) == torch.arange(count, device=sample.device).unsqueeze(1)).double()
    member = torch.nn.functional.pad(member, (0, pad)).view(count, slices, 512).transpose(0, 1).contiguous()
    values = torch.nn.functional.pad(values, (0, 0, 0, pad)).view(slices, 512, g)
    return (member @ values).sum(0)


def _by_row(values, index, count):
    """sums of the rows [n, w] with the same index: sorted by index, then differences of the running sums in 64 bits"""
    index, by_index = torch.sort(index, stable=True)
    running = torch.nn.functional.pad(torch.cumsum(values[by_index].t().double().contiguous(), 1), (1, 0))
    ends = torch.searchsorted(index, torch.arange(count + 1, device=index.device))
    return (running[:, ends[1:]] - running[:, ends[:-1]]).t()


def _plain_norm(s):
    case = s["case"]
    n, c, b, g = case["rows"], case["channels"], case["samples"], case["groups"]
    dtype, sample, act = s["x"].dtype, s["sample"], case["act"]
    with torch.no_grad():
        x = s["x"].float().view(n, g, c // g)
        size = (_by_sample(torch.ones(n, 1, dtype=torch.float64, device=x.device), sample, b) * (c // g)).clamp(min=1.0)
        mean = (_by_sample(x.sum(2, dtype=torch.float64), sample, b) / size).float()
        d = x - mean[sample].unsqueeze(2)
        var = (_by_sample((d * d).sum(2, dtype=torch.float64), sample, b) / size).float()
        rstd = torch.rsqrt(var + NORM_EPS)[sample].unsqueeze(2)
        xhat = (d * rstd).view(n, c)
        z = xhat * s["weight"] + s["bias"]
        if s["residual"] is not None:
            z = z + s["residual"].float()
        if act == "relu":
            y, slope = z.clamp(min=0.0), (z > 0).float()
        elif act == "silu":
            p = 1.0 / (1.0 + torch.exp(-z))
            y, slope = z * p, p * (1.0 + z * (1.0 - p))
        elif act == "gelu":
            p = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
            y, slope = z * p, p + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
        else:
            y, slope = z, torch.ones_like(z)
        out = {"y": y.to(dtype)}
        if case["train"]:
            gz = s["dy"].float() * slope
            out["dweight"] = (gz * xhat).sum(0, dtype=torch.float64).float()
            out["dbias"] = gz.sum(0, dtype=torch.float64).float()
            if s["residual"] is not None:
                out["dresidual"] = gz.to(dtype)
            gx = (gz * s["weight"]).view(n, g, c // g)
            xh = xhat.view(n, g, c // g)
            m0 = (_by_sample(gx.sum(2, dtype=torch.float64), sample, b) / size).float()[sample].unsqueeze(2)
            m1 = (_by_sample((gx * xh).sum(2, dtype=torch.float64), sample, b) / size).float()[sample].unsqueeze(2)
            out["dx"] = (rstd * (gx - m0 - xh * m1)).view(n, c).to(dtype)
    return out


def _plain_lookup(s):
    case, table = s["case"], s["table"]
    with torch.no_grad():
        inside = (s["index"] >= 0).unsqueeze(1)
        at = s["index"].long().clamp(min=0)
        out = {"out": (table.float()[at] * case["scale"] * inside).to(table.dtype)}
        if case["train"]:
            d = s["dout"].float() * case["scale"] * inside
            out["dtable"] = _by_row(d, at, table.shape[0]).to(table.dtype).contiguous()
    return out


def _plain_orthogonalize(s):
    a, b, c = COEFFICIENTS

    def one(m):
        x = m.float()
        x = x if m.shape[0] <= m.shape[1] else x.t()
        x = x / (torch.sqrt((x * x).sum()) + ORTHO_EPS)
        for _ in range(STEPS):
            gram = x @ x.t()
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        return (x if m.shape[0] <= m.shape[1] else x.t()).to(m.dtype)

    return [one(m) for m in s["matrices"]]


# ---- the framework's calls ----------------------------------------------------------------------------------------------

def _own_norm(s):
    from openpcdet_amd.spconv.pytorch import norm
    case, x, res = s["case"], s["x"], s["residual"]
    act = None if case["act"] == "none" else case["act"]
    if case["layout"] == "dense":
        shape = (case["samples"], case["rows"] // case["samples"], case["channels"])
        y = norm.group_norm_act(x.view(shape), case["groups"], s["weight"], s["bias"], eps=NORM_EPS, act=act,
                                residual=res.view(shape) if res is not None else None).view(x.shape)
    else:
        y = norm.group_norm_act(x, case["groups"], s["weight"], s["bias"], eps=NORM_EPS, act=act, residual=res, offsets=s["offsets"],
                                order=s["order"])
    out = {"y": y}
    if case["train"]:
        names = ["x", "weight", "bias"] + (["residual"] if res is not None else [])
        grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
        out.update({"d" + k: v for k, v in zip(names, grads)})
    return out


def _own_lookup(s):
    from openpcdet_amd import scatter
    out = {"out": scatter.lookup_rows(s["table"], s["index"], scale=s["case"]["scale"])}
    if s["case"]["train"]:
        out["dtable"] = torch.autograd.grad(out["out"], s["table"], s["dout"])[0]
    return out


def _own_orthogonalize(s):
    from openpcdet_amd import optim
    return optim.orthogonalize(s["matrices"], steps=STEPS, coefficients=COEFFICIENTS, eps=ORTHO_EPS)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "lookup": _own_lookup, "orthogonalize": _own_orthogonalize}[op](state)
    return {"norm": _plain_norm, "lookup": _plain_lookup, "orthogonalize": _plain_orthogonalize}[op](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "orthogonalize":
        size = {"float32": 4}.get(case["dtype"], 2)
        flops = moved = 0
        for r, c in _shapes(case):
            m, n = min(r, c), max(r, c)
            flops += STEPS * (3 * m * m * n + m * m * m)     # both products with a symmetric result need half of it
            moved += 2 * r * c * size
        return {"bytes": moved, "flops": flops}
    size = {"float32": 4}.get(case["dtype"], 2)
    if case["op"] == "norm":
        e = case["rows"] * case["channels"]
        tensors = (2 + case["residual"]) * (2 if case["train"] else 1)       # x, y (residual), and their gradients
        params = 4 * case["channels"] * (4 if case["train"] else 2)
        return {"bytes": e * size * tensors + params, "flops": e * (30 if case["train"] else 10)}
    n, m, w = case["tokens"], case["rows"], case["width"]
    moved = n * {"int32": 4, "int64": 8}[case["index"]] + min(n, m) * w * size + n * w * size
    if case["train"]:
        moved += n * w * size + m * w * size
    return {"bytes": moved, "flops": n * w * (2 if case["train"] else 1)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def _exact_norm(s):
    """each sample by itself as [1, C, rows] through the library's definition and its derivative"""
    case, act = s["case"], s["case"]["act"]
    x, w, b = (s[k].detach().double() for k in ("x", "weight", "bias"))
    res = s["residual"].detach().double() if s["residual"] is not None else None
    y = torch.zeros_like(x)
    grads = {"dx": torch.zeros_like(x), "dweight": torch.zeros_like(w), "dbias": torch.zeros_like(b)}
    if res is not None:
        grads["dresidual"] = torch.zeros_like(x)
    for k in range(case["samples"]):
        rows = torch.nonzero(s["sample"] == k).flatten()
        if rows.numel() == 0:
            continue
        leaves = [x[rows].requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
        if rows.numel() * (case["channels"] // case["groups"]) > 1:
            z = torch.nn.functional.group_norm(leaves[0].t().unsqueeze(0), case["groups"], leaves[1], leaves[2], NORM_EPS)[0].t()
        else:                                # a single value has no spread: its normalised value is 0
            z = leaves[0] * 0.0 * leaves[1] + leaves[2]
        if res is not None:
            leaves.append(res[rows].requires_grad_(True))
            z = z + leaves[3]
        v = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act](z)
        y[rows] = v.detach()
        if case["train"]:
            got = torch.autograd.grad(v, leaves, s["dy"][rows].double())
            grads["dx"][rows] = got[0]
            grads["dweight"] += got[1]
            grads["dbias"] += got[2]
            if res is not None:
                grads["dresidual"][rows] = got[3]
    return {"y": y, **(grads if case["train"] else {})}


def _exact_lookup(s):
    table = s["table"].detach().double()
    inside = torch.nonzero(s["index"] >= 0).flatten()
    at = s["index"][inside].long()
    out = torch.zeros(s["index"].shape[0], table.shape[1], dtype=torch.float64, device=table.device)
    out[inside] = table.index_select(0, at) * s["case"]["scale"]
    got = {"out": out}
    if s["case"]["train"]:
        by_row = torch.argsort(at)
        d = torch.zeros_like(table)
        d.index_put_((at[by_row],), s["dout"][inside][by_row].double() * s["case"]["scale"], accumulate=True)
        got["dtable"] = d
    return got


def _exact_orthogonalize(s):
    """the odd polynomial applied to the singular values, in the form (a + (b + c A) A) X"""
    a, b, c = COEFFICIENTS
    found = []
    for m in s["matrices"]:
        x = m.double() if m.shape[0] <= m.shape[1] else m.double().t().contiguous()
        x = x / (torch.linalg.matrix_norm(x) + ORTHO_EPS)
        one = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
        for _ in range(STEPS):
            gram = x @ x.t()
            x = (a * one + (b * one + c * gram) @ gram) @ x
        found.append(x if m.shape[0] <= m.shape[1] else x.t())
    return found


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "lookup": _exact_lookup, "orthogonalize": _exact_orthogonalize}[case["op"]](s)
