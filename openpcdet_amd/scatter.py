"""scatter_mean / scatter_max along dim 0 -- the two torch_scatter functions the reference's dynamic VFEs import
(pcdet/models/backbones_3d/vfe/dynamic_pillar_vfe.py:5-9,40,105; dynamic_mean_vfe.py:65).  Same call shape
(`scatter_mean(src, index, dim=0)`, `scatter_max(src, index, dim=0) -> (values, argmax)`), backed by
pvx_scatter_mean / pvx_scatter_max; both are differentiable (PFN weights train through scatter_max).
`index` may be int32 or int64; negative entries are skipped.  `dim_size` avoids the host read of index.max().

`lookup_rows` is the way back, rows of a table picked by index (times a scale), with the table's gradient summed by sorted index
(pvx_lookup_rows, pvx_sort_index, pvx_lookup_rows_grad); `sort_index` hands that sort out, for an index that several calls share."""
import torch

from . import _lib


def _prep(src, index, dim, dim_size):
    assert dim == 0, "only dim=0 is used by pcdet and implemented here"
    assert src.is_cuda and index.is_cuda and index.dim() == 1 and index.shape[0] == src.shape[0]
    n = src.shape[0]
    if dim_size is None:
        dim_size = int(index.max().item()) + 1 if n > 0 else 0
    src2 = src.reshape(n, -1).float().contiguous()
    return src2, index.to(torch.int32).contiguous(), n, src2.shape[1], int(dim_size)


class _ScatterMean(torch.autograd.Function):
    @staticmethod
    def forward(ctx, src, index, m):
        L = _lib.lib()
        n, c = src.shape
        out = torch.empty((m, c), dtype=torch.float32, device=src.device)
        ws = _lib.workspace(L.pvx_scatter_mean_workspace_bytes(m, c), src.device)
        with torch.cuda.device(src.device):
            _lib.check(L.pvx_scatter_mean(_lib.ptr(src), _lib.ptr(index), n, None, c, m, _lib.ptr(out), _lib.ptr(ws), ws.numel(),
                                          _lib.stream()), "pvx_scatter_mean")
        ctx.save_for_backward(index)
        ctx.m = m
        return out

    @staticmethod
    def backward(ctx, grad):
        index, = ctx.saved_tensors
        idx = index.long().clamp(min=0)
        cnt = torch.bincount(idx[index >= 0], minlength=ctx.m).clamp(min=1).to(grad.dtype)
        g = (grad / cnt.unsqueeze(1))[idx]
        g = torch.where((index >= 0).unsqueeze(1), g, torch.zeros_like(g))
        return g, None, None


class _ScatterMax(torch.autograd.Function):
    @staticmethod
    def forward(ctx, src, index, m):
        L = _lib.lib()
        n, c = src.shape
        out = torch.empty((m, c), dtype=torch.float32, device=src.device)
        arg = torch.empty((m, c), dtype=torch.int32, device=src.device)
        with torch.cuda.device(src.device):
            _lib.check(L.pvx_scatter_max(_lib.ptr(src), _lib.ptr(index), n, None, c, m, _lib.ptr(out), _lib.ptr(arg), _lib.stream()),
                       "pvx_scatter_max")
        ctx.save_for_backward(arg)
        ctx.n = n
        ctx.mark_non_differentiable(arg)
        return out, arg

    @staticmethod
    def backward(ctx, grad, _):
        arg, = ctx.saved_tensors
        g = grad.new_zeros((ctx.n + 1, grad.shape[1]))          # row n collects the empty segments
        g.scatter_(0, arg.long(), grad)
        return g[:ctx.n], None, None


def scatter_mean(src, index, dim=0, out=None, dim_size=None):
    assert out is None
    s, i, n, c, m = _prep(src, index, dim, dim_size)
    r = _ScatterMean.apply(s, i, m)
    return r.reshape((m,) + tuple(src.shape[1:])).to(src.dtype)


def scatter_max(src, index, dim=0, out=None, dim_size=None):
    assert out is None
    s, i, n, c, m = _prep(src, index, dim, dim_size)
    v, a = _ScatterMax.apply(s, i, m)
    shape = (m,) + tuple(src.shape[1:])
    return v.reshape(shape).to(src.dtype), a.reshape(shape).long()


# ---- rows by index -------------------------------------------------------------------------------------------------------
class IndexSort:
    """What `sort_index` returns for an index of n entries into num_rows rows: `order` [n] int32, the positions by ascending index
    (equal ones by position, entries outside the rows at the end), `keys` [n] int32, the sorted indices (num_rows for those outside), and
    `offsets` [num_rows + 1] int32: row v was named by the positions order[offsets[v]:offsets[v + 1]]."""

    def __init__(self, order, keys, offsets, num_rows):
        self.order, self.keys, self.offsets, self.num_rows = order, keys, offsets, num_rows


def _check_index(index):
    if not index.is_cuda:
        raise RuntimeError("rows are looked up on the GPU only (no CPU fallback): got an index on %s" % index.device)
    if index.dtype not in (torch.int32, torch.int64):
        raise TypeError("index must be int32 or int64, got %s" % index.dtype)


def sort_index(index, num_rows):
    """stable sort of `index` (int32 or int64, any shape, flattened) into runs of equal entries -> IndexSort; no host read"""
    _check_index(index)
    num_rows = int(num_rows)
    if num_rows < 1:
        raise ValueError("num_rows must be at least 1, got %d" % num_rows)
    _lib.check_counts("sort_index", num_rows, index.numel())
    index = index.reshape(-1).contiguous()
    n, dev = index.shape[0], index.device
    L = _lib.lib()
    with _lib.on(dev):
        order = torch.empty(n, dtype=torch.int32, device=dev)
        keys = torch.empty(n, dtype=torch.int32, device=dev)
        offsets = torch.empty(num_rows + 1, dtype=torch.int32, device=dev)
        size = L.pvx_sort_index_workspace_bytes(n)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        rc = L.pvx_sort_index(index.data_ptr(), index.dtype == torch.int64, n, num_rows, order.data_ptr(), keys.data_ptr(),
                              offsets.data_ptr(), ws.data_ptr(), size, _lib.raw_stream(dev))
        if rc:
            _lib.check(rc, "pvx_sort_index")
    return IndexSort(order, keys, offsets, num_rows)


def _lookup(table, index, scale):
    """table [m, w] contiguous, index [n] contiguous -> [n, w]"""
    n, (m, w) = index.shape[0], table.shape
    dev = table.device
    with _lib.on(dev):
        out = table.new_empty((n, w))
        rc = _lib.lib().pvx_lookup_rows(table.data_ptr(), _lib.DTYPE_CODE[table.dtype], index.data_ptr(), index.dtype == torch.int64, n, m, w, scale,
                                        out.data_ptr(), _lib.raw_stream(dev))
        if rc:
            _lib.check(rc, "pvx_lookup_rows")
    return out


class _LookupRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale, sort):
        ctx.save_for_backward(index)
        ctx.scale, ctx.sort, ctx.rows = scale, sort, table.shape[0]
        return _lookup(table, index, scale)

    @staticmethod
    def backward(ctx, grad):
        index, = ctx.saved_tensors
        f = _LookupRowsGrad.apply if torch.is_grad_enabled() else _lookup_grad
        return f(grad, index, ctx.scale, ctx.sort, ctx.rows), None, None, None


class _LookupRowsGrad(torch.autograd.Function):
    """the gradient, under create_graph: linear as the lookup is, and its own gradient is the lookup"""

    @staticmethod
    def forward(ctx, grad, index, scale, sort, m):
        ctx.save_for_backward(index)
        ctx.scale, ctx.sort = scale, sort
        return _lookup_grad(grad, index, scale, sort, m)

    @staticmethod
    def backward(ctx, dtable):
        index, = ctx.saved_tensors
        dtable = dtable.contiguous()
        out = _LookupRows.apply(dtable, index, ctx.scale, ctx.sort) if torch.is_grad_enabled() else _lookup(dtable, index, ctx.scale)
        return out, None, None, None, None


def _lookup_grad(grad, index, scale, sort, m):
    """grad [n, w], index [n] contiguous -> [m, w]"""
    n, w = grad.shape
    dev = index.device
    grad = grad.contiguous()
    dtable = grad.new_empty((m, w))
    if m > 0 and w > 0:
        L = _lib.lib()
        with _lib.on(dev):
            size = L.pvx_lookup_rows_grad_workspace_bytes(n, w, sort is not None)
            ws = grad.new_empty(size, dtype=torch.uint8)
            order, keys = (sort.order.data_ptr(), sort.keys.data_ptr()) if sort is not None else (None, None)
            rc = L.pvx_lookup_rows_grad(grad.data_ptr(), _lib.DTYPE_CODE[grad.dtype], index.data_ptr(), index.dtype == torch.int64, order, keys,
                                        n, m, w, scale, dtable.data_ptr(), ws.data_ptr(), size, _lib.raw_stream(dev))
            if rc:
                _lib.check(rc, "pvx_lookup_rows_grad")
    return dtable


def lookup_rows(table, index, scale=1.0, sort=None):
    """scale * table[index]: table [m, ...] float32 / float16 / bfloat16, index int32 or int64 of any shape -> [*index.shape, ...] in the
    table's dtype.  Entries outside [0, m) give zeros and pass no gradient.  The gradient with respect to the table (and only to it) adds
    each row's entries in 32 bits and in an order of its own, without atomics, and can be differentiated again.  `sort`: sort_index(index, m)
    of this very index, where the caller has it (the backward sorts otherwise)."""
    if not table.is_cuda:
        raise RuntimeError("rows are looked up on the GPU only (no CPU fallback): got a table on %s" % table.device)
    _check_index(index)
    if table.device != index.device:
        raise RuntimeError("table and index are on different devices: %s and %s" % (table.device, index.device))
    if table.dtype not in _lib.DTYPE_CODE:
        raise TypeError("unsupported table dtype %s" % table.dtype)
    if table.dim() < 1:
        raise ValueError("table must have a dimension of rows")
    if sort is not None and (sort.num_rows != table.shape[0] or sort.order.shape[0] != index.numel() or sort.order.device != table.device):
        raise ValueError("sort is that of another index: %d entries into %d rows, wanted %d into %d"
                         % (sort.order.shape[0], sort.num_rows, index.numel(), table.shape[0]))
    shape = tuple(index.shape) + tuple(table.shape[1:])
    width = 1
    for d in table.shape[1:]:
        width *= d
    _lib.check_counts("lookup_rows", table.shape[0], width, index.numel())
    flat = table.contiguous() if table.dim() == 2 else table.reshape(table.shape[0], width).contiguous()
    idx = index.contiguous() if index.dim() == 1 else index.reshape(-1).contiguous()
    if _lib.differentiated(flat):
        out = _LookupRows.apply(flat, idx, float(scale), sort)
    else:
        out = _lookup(flat, idx, float(scale))
    return out if out.shape == shape else out.view(shape)
