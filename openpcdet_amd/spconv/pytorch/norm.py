"""BatchNorm1d (+ residual) + ReLU over a sparse tensor's feature matrix in one fused op for the TRAINING step: what
`norm_fn(C) -> nn.ReLU()` (pcdet/models/backbones_3d/spconv_backbone.py:21-25) and `bn -> += identity -> relu` (:52-64) compute,
on csrc/batchnorm.hip.  The modules stay plain `nn.BatchNorm1d` / `nn.ReLU` (state-dict keys, `.eval()`, SyncBatchNorm conversion
all unchanged); `SparseSequential` and `SparseBasicBlock` call `bn_act` where they see the pattern.  Anything the kernels do not
take -- eval mode, SyncBatchNorm, momentum=None, CPU tensors, odd channel counts -- goes through the modules themselves.

Group norm (+ residual) + activation over the rows of each sample, `group_norm_act` and the module `SparseGroupNorm`, is the
normalisation that needs no batch and no all-reduce (csrc/group_norm.hip); the same in training and in evaluation."""
import os

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ... import _lib
from .core import SparseConvTensor
from .modules import SparseModule

_ENABLED = os.environ.get("PVX_FUSED_BN", "1") != "0"       # A/B switch


class _BNAct(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, running_mean, running_var, residual, eps, momentum, relu):
        L = _lib.lib()
        x = x.contiguous()
        n, c = x.shape
        code = _lib.DTYPE_CODE[x.dtype]
        dev = x.device
        if residual is not None:
            residual = residual.to(x.dtype).contiguous()
        y = torch.empty_like(x)
        mean = torch.empty(c, dtype=torch.float32, device=dev)
        invstd = torch.empty(c, dtype=torch.float32, device=dev)
        w = weight.detach().float().contiguous() if weight is not None else None
        b = bias.detach().float().contiguous() if bias is not None else None
        with torch.cuda.device(dev):
            ws = _lib.workspace(L.pvx_bn_act_workspace_bytes(c), dev)
            _lib.check(L.pvx_bn_act_fwd(_lib.ptr(x), n, c, code, _lib.ptr(w), _lib.ptr(b), float(eps), float(momentum),
                                        _lib.ptr(running_mean), _lib.ptr(running_var), _lib.ptr(residual), int(relu), _lib.ptr(y),
                                        _lib.ptr(mean), _lib.ptr(invstd), _lib.ptr(ws), ws.numel(), _lib.stream()), "pvx_bn_act_fwd")
        ctx.save_for_backward(x, y, w, mean, invstd)
        ctx.relu, ctx.has_res = bool(relu), residual is not None
        ctx.param_dtypes = (weight.dtype if weight is not None else None, bias.dtype if bias is not None else None)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, y, w, mean, invstd = ctx.saved_tensors
        L = _lib.lib()
        n, c = x.shape
        dev = x.device
        dy = dy.to(x.dtype).contiguous()
        dx = torch.empty_like(x)
        dres = torch.empty_like(x) if ctx.has_res else None
        dgamma = torch.empty(c, dtype=torch.float32, device=dev)
        dbeta = torch.empty(c, dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            ws = _lib.workspace(L.pvx_bn_act_workspace_bytes(c), dev)
            _lib.check(L.pvx_bn_act_bwd(_lib.ptr(dy), _lib.ptr(x), _lib.ptr(y), n, c, _lib.DTYPE_CODE[x.dtype], _lib.ptr(w), _lib.ptr(mean),
                                        _lib.ptr(invstd), int(ctx.relu), _lib.ptr(dx), _lib.ptr(dres), _lib.ptr(dgamma), _lib.ptr(dbeta),
                                        _lib.ptr(ws), ws.numel(), _lib.stream()), "pvx_bn_act_bwd")
        wd, bd = ctx.param_dtypes
        return (dx, dgamma.to(wd) if wd is not None else None, dbeta.to(bd) if bd is not None else None, None, None, dres, None, None, None)


class _SyncBNAct(Function):
    """the same op with statistics over every rank of `group` (torch.nn.SyncBatchNorm's semantics, torch/nn/modules/_functions.py):
    local column sums + row count -> one all-reduce (RCCL) -> finish and apply; no host synchronisation"""

    @staticmethod
    def forward(ctx, x, weight, bias, running_mean, running_var, residual, eps, momentum, relu, group):
        import torch.distributed as dist
        L = _lib.lib()
        x = x.contiguous()
        n, c = x.shape
        code = _lib.DTYPE_CODE[x.dtype]
        dev = x.device
        if residual is not None:
            residual = residual.to(x.dtype).contiguous()
        y = torch.empty_like(x)
        mean = torch.empty(c, dtype=torch.float32, device=dev)
        invstd = torch.empty(c, dtype=torch.float32, device=dev)
        sums = torch.empty(2 * c + 1, dtype=torch.float64, device=dev)
        w = weight.detach().float().contiguous() if weight is not None else None
        b = bias.detach().float().contiguous() if bias is not None else None
        with torch.cuda.device(dev):
            ws = _lib.workspace(L.pvx_bn_act_workspace_bytes(c), dev)
            args = (_lib.ptr(x), n, c, code, _lib.ptr(w), _lib.ptr(b), float(eps), float(momentum), _lib.ptr(running_mean),
                    _lib.ptr(running_var), _lib.ptr(residual), int(relu), _lib.ptr(y), _lib.ptr(mean), _lib.ptr(invstd), _lib.ptr(sums))
            _lib.check(L.pvx_bn_act_fwd_sync(*args, 0, 1, _lib.ptr(ws), ws.numel(), _lib.stream()), "pvx_bn_act_fwd_sync")
            dist.all_reduce(sums, op=dist.ReduceOp.SUM, group=group)
            _lib.check(L.pvx_bn_act_fwd_sync(*args, 0, 2, _lib.ptr(ws), ws.numel(), _lib.stream()), "pvx_bn_act_fwd_sync")
        ctx.save_for_backward(x, y, w, mean, invstd)
        ctx.relu, ctx.has_res, ctx.group = bool(relu), residual is not None, group
        ctx.param_dtypes = (weight.dtype if weight is not None else None, bias.dtype if bias is not None else None)
        return y

    @staticmethod
    def backward(ctx, dy):
        import torch.distributed as dist
        x, y, w, mean, invstd = ctx.saved_tensors
        L = _lib.lib()
        n, c = x.shape
        dev = x.device
        dy = dy.to(x.dtype).contiguous()
        dx = torch.empty_like(x)
        dres = torch.empty_like(x) if ctx.has_res else None
        dgamma = torch.empty(c, dtype=torch.float32, device=dev)
        dbeta = torch.empty(c, dtype=torch.float32, device=dev)
        sums = torch.empty(2 * c + 1, dtype=torch.float64, device=dev)
        with torch.cuda.device(dev):
            ws = _lib.workspace(L.pvx_bn_act_workspace_bytes(c), dev)
            args = (_lib.ptr(dy), _lib.ptr(x), _lib.ptr(y), n, c, _lib.DTYPE_CODE[x.dtype], _lib.ptr(w), _lib.ptr(mean), _lib.ptr(invstd),
                    int(ctx.relu), _lib.ptr(dx), _lib.ptr(dres), _lib.ptr(dgamma), _lib.ptr(dbeta), _lib.ptr(sums))
            _lib.check(L.pvx_bn_act_bwd_sync(*args, 0, 1, _lib.ptr(ws), ws.numel(), _lib.stream()), "pvx_bn_act_bwd_sync")
            dist.all_reduce(sums, op=dist.ReduceOp.SUM, group=ctx.group)
            _lib.check(L.pvx_bn_act_bwd_sync(*args, 0, 2, _lib.ptr(ws), ws.numel(), _lib.stream()), "pvx_bn_act_bwd_sync")
        wd, bd = ctx.param_dtypes
        return (dx, dgamma.to(wd) if wd is not None else None, dbeta.to(bd) if bd is not None else None, None, None, dres, None, None, None,
                None)


def _sync_group(bn):
    """the process group a SyncBatchNorm module reduces over, or None when it would not synchronise (torch falls back to plain
    batch_norm then: not training, no process group; a group of ONE rank is handled by bn_act without a collective)"""
    import torch.distributed as dist
    if not (dist.is_available() and dist.is_initialized()):
        return None
    return bn.process_group if bn.process_group is not None else dist.group.WORLD


def fusable(bn, x):
    if type(bn) is nn.SyncBatchNorm:
        # decided from facts every rank of the group shares (module, mode, dtype, channels, group) and never from this rank's row
        # count: the fused path issues ONE all-reduce where torch's SyncBatchNorm issues an all-gather, so two ranks that chose
        # differently (a frame with a single active row at some level, PartA2's fake_sparse_idx) would hang or mix buffers.
        # The kernels take n == 1, and n == 0 as "zero sums, nothing to apply".
        return (_ENABLED and bn.training and bn.momentum is not None and x.is_cuda and x.dim() == 2
                and x.dtype in _lib.DTYPE_CODE and _sync_group(bn) is not None
                and bool(_lib.lib().pvx_bn_act_supported(x.shape[1], _lib.DTYPE_CODE[x.dtype])))
    return (_ENABLED and type(bn) is nn.BatchNorm1d and bn.training and bn.momentum is not None and x.is_cuda and x.dim() == 2
            and x.shape[0] > 1 and x.dtype in _lib.DTYPE_CODE and bool(_lib.lib().pvx_bn_act_supported(x.shape[1], _lib.DTYPE_CODE[x.dtype])))


def bn_act(x, bn, residual=None, relu=True):
    """relu?(bn(x) (+ residual)) for a [N, C] feature matrix; one fused forward and one fused backward when `fusable`"""
    if not fusable(bn, x):
        y = bn(x)
        if residual is not None:
            y = y + residual
        return torch.relu(y) if relu else y
    rm, rv = (bn.running_mean, bn.running_var) if bn.track_running_stats else (None, None)
    if bn.track_running_stats and bn.num_batches_tracked is not None:
        bn.num_batches_tracked.add_(1)
    args = (x, bn.weight if bn.affine else None, bn.bias if bn.affine else None, rm, rv, residual, bn.eps, bn.momentum, relu)
    if type(bn) is nn.SyncBatchNorm:
        group = _sync_group(bn)
        import torch.distributed as dist
        if dist.get_world_size(group) > 1:
            return _SyncBNAct.apply(*args, group)
        # a group of one rank: the statistics are this rank's own, no collective (torch.nn.SyncBatchNorm takes its plain batch_norm
        # path in that case too: need_sync = world_size > 1); the choice depends on the group only, so every rank makes the same one
        if x.shape[0] <= 1:
            y = bn(x)
            if residual is not None:
                y = y + residual
            return torch.relu(y) if relu else y
    return _BNAct.apply(*args)


# ---- group norm ------------------------------------------------------------------------------------------------------------
_ACTS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _hooked(module):
    m = torch.nn.modules.module
    return (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks or m._global_forward_hooks
            or m._global_forward_pre_hooks or m._global_backward_hooks or m._global_backward_pre_hooks)


def act_name(module):
    """the name `group_norm_act` has for an activation module, None if it has none or hooks want the module's own call"""
    if _hooked(module):
        return None
    if type(module) is nn.ReLU:
        return "relu"
    if type(module) is nn.SiLU:
        return "silu"
    if type(module) is nn.GELU and module.approximate == "none":
        return "gelu"
    return None


def _addr(t):
    return t.data_ptr() if t is not None else None


def _group_norm_fwd(x, weight, bias, residual, offsets, order, samples, groups, eps, act):
    """x [n, c] contiguous -> y, statistics [2, samples, groups] (mean, 1 / sqrt(var + eps))"""
    L = _lib.lib()
    n, c = x.shape
    dev = x.device
    with _lib.on(dev):
        y = torch.empty_like(x)
        stats = x.new_empty((2, samples, groups), dtype=torch.float32)
        size = L.pvx_group_norm_act_workspace_bytes(n, c, samples, offsets is not None, groups)
        ws = x.new_empty(size, dtype=torch.uint8)
        base = stats.data_ptr()
        rc = L.pvx_group_norm_act_fwd(x.data_ptr(), n, c, _lib.DTYPE_CODE[x.dtype], samples, _addr(offsets), _addr(order), groups, _addr(weight),
                                      _addr(bias), _param_code(weight, bias), eps, _addr(residual), act, y.data_ptr(), base,
                                      base + 4 * samples * groups, ws.data_ptr(), size, _lib.raw_stream(dev))
        if rc:
            _lib.check(rc, "pvx_group_norm_act_fwd")
    return y, stats


def _param_code(weight, bias):
    p = weight if weight is not None else bias
    return _lib.DTYPE_CODE[p.dtype] if p is not None else _lib.PVX_F32


class _GroupNormAct(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, offsets, order, samples, groups, eps, act):
        y, stats = _group_norm_fwd(x, weight, bias, residual, offsets, order, samples, groups, eps, act)
        ctx.save_for_backward(x, weight, bias, residual, offsets, order, stats)
        ctx.args = (samples, groups, act)
        return y

    @staticmethod
    def backward(ctx, dy):
        return _group_norm_bwd_once(ctx, dy) if torch.is_grad_enabled() else _group_norm_bwd(ctx, dy)


def _group_norm_bwd(ctx, dy):
    x, weight, bias, residual, offsets, order, stats = ctx.saved_tensors
    samples, groups, act = ctx.args
    L = _lib.lib()
    n, c = x.shape
    dev = x.device
    dy = dy.contiguous()
    with _lib.on(dev):
        dx = torch.empty_like(x)
        dres = torch.empty_like(x) if residual is not None else None
        dw = torch.empty_like(weight) if weight is not None else None
        db = torch.empty_like(bias) if bias is not None else None
        size = L.pvx_group_norm_act_workspace_bytes(n, c, samples, offsets is not None, groups)
        ws = x.new_empty(size, dtype=torch.uint8)
        base = stats.data_ptr()
        rc = L.pvx_group_norm_act_bwd(dy.data_ptr(), x.data_ptr(), _addr(residual), n, c, _lib.DTYPE_CODE[x.dtype], samples, _addr(offsets),
                                      _addr(order), groups, _addr(weight), _addr(bias), _param_code(weight, bias), base,
                                      base + 4 * samples * groups, act, dx.data_ptr(), _addr(dres), _addr(dw), _addr(db), ws.data_ptr(), size,
                                      _lib.raw_stream(dev))
        if rc:
            _lib.check(rc, "pvx_group_norm_act_bwd")
    return dx, dw, db, dres, None, None, None, None, None, None


_group_norm_bwd_once = once_differentiable(_group_norm_bwd)      # under create_graph: a second derivative is refused, not left out


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act=None, residual=None, offsets=None, order=None):
    """act(group_norm(x) (+ residual)), channels last.

    x [B, ..., C]: each x[b] is a sample and its statistics go over every position of it and the C / num_groups channels of a group (what
    torch.nn.functional.group_norm computes with the channels moved to dimension 1).  With `offsets` (int32 [B + 1], device, ascending),
    x is [N, C] and sample b owns the positions offsets[b]:offsets[b + 1]; position p is row p, or row order[p] (`order`: int32 [N], a
    permutation).  Rows at positions of no sample get zeros, and a zero gradient.

    x float32 / float16 / bfloat16; weight and bias [C] of one dtype of these; residual like x; act None, "relu", "silu" or "gelu" (with
    the error function).  Gradients with respect to x, weight, bias and residual.  One kernel where each sample is known to fit a
    workgroup, three otherwise; the same bits on every run."""
    if not x.is_cuda:
        raise RuntimeError("group_norm_act runs on the GPU only (no CPU fallback): got a tensor on %s" % x.device)
    if x.dtype not in _lib.DTYPE_CODE:
        raise TypeError("unsupported dtype %s" % x.dtype)
    if x.dim() < 2:
        raise ValueError("x must be [B, ..., C], got %s" % (tuple(x.shape),))
    if act not in _ACTS:
        raise ValueError("act must be one of None, 'relu', 'silu', 'gelu', got %r" % (act,))
    c, num_groups, eps = x.shape[-1], int(num_groups), float(eps)
    if num_groups < 1 or c < 1 or c % num_groups != 0:
        raise ValueError("%d channels do not make %d groups" % (c, num_groups))
    if not eps >= 0.0:
        raise ValueError("eps must not be negative, got %r" % (eps,))
    dev = x.device
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.dim() != 1 or p.shape[0] != c or p.device != dev:
            raise ValueError("%s must be [%d] on %s, got %s on %s" % (name, c, x.device, tuple(p.shape), p.device))
        if p.dtype not in _lib.DTYPE_CODE or (weight is not None and p.dtype != weight.dtype):
            raise TypeError("weight and bias must share one of float32, float16 and bfloat16, got %s for %s" % (p.dtype, name))
    if residual is not None:
        if residual.shape != x.shape or residual.device != dev:
            raise ValueError("residual must be %s on %s, got %s on %s" % (tuple(x.shape), x.device, tuple(residual.shape), residual.device))
        if residual.dtype != x.dtype:
            residual = residual.to(x.dtype)
    if offsets is None:
        if order is not None:
            raise ValueError("order needs offsets")
        samples = x.shape[0]
    else:
        if x.dim() != 2:
            raise ValueError("with offsets, x must be [N, C], got %s" % (tuple(x.shape),))
        for name, t, size in (("offsets", offsets, None), ("order", order, x.shape[0])):
            if t is None:
                continue
            if t.dtype != torch.int32 or t.dim() != 1 or t.device != dev or (size is not None and t.shape[0] != size):
                raise ValueError("%s must be an int32 vector%s on %s, got %s %s on %s" % (
                    name, " of %d" % size if size is not None else "", x.device, t.dtype, tuple(t.shape), t.device))
        samples = offsets.shape[0] - 1
        if samples < 1:
            raise ValueError("offsets must have an entry more than there are samples")
    _lib.check_counts("group_norm_act", x.numel() // c, c, samples)
    if offsets is not None:
        offsets = offsets.contiguous()
        order = order.contiguous() if order is not None else None
    plain = x.dim() == 2
    flat = x.contiguous() if plain else x.reshape(-1, c).contiguous()
    if flat.shape[0] == 0:
        samples = max(samples, 1)
    res = residual
    if res is not None:
        res = res.contiguous() if plain else res.reshape(-1, c).contiguous()
    w = weight.contiguous() if weight is not None else None
    b = bias.contiguous() if bias is not None else None
    args = (flat, w, b, res, offsets, order, samples, num_groups, eps, _ACTS[act])
    if _lib.differentiated(*args[:4]):
        y = _GroupNormAct.apply(*args)
    else:
        y = _group_norm_fwd(*args)[0]
    return y if plain else y.view(x.shape)


class SparseGroupNorm(SparseModule):
    """GroupNorm over a SparseConvTensor: statistics over the sites of each sample (frame) and the channels of a group.  Parameters are
    those of nn.GroupNorm (`weight`, `bias`).  In a SparseSequential a ReLU, SiLU or GELU behind it runs in the same kernels.  (nn.GroupNorm
    itself, given the [N, C] features, takes every site for a sample of its own.)"""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, device=None, dtype=None):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups != 0:
            raise ValueError("%d channels do not make %d groups" % (num_channels, num_groups))
        self.num_groups, self.num_channels, self.eps, self.affine = int(num_groups), int(num_channels), float(eps), bool(affine)
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels, device=device, dtype=dtype))
            self.bias = nn.Parameter(torch.zeros(num_channels, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def extra_repr(self):
        return "{num_groups}, {num_channels}, eps={eps}, affine={affine}".format(**self.__dict__)

    def forward(self, input, act=None, residual=None):
        """act(norm(input) (+ residual)); residual: features of the same sites"""
        assert isinstance(input, SparseConvTensor), "expected a SparseConvTensor"
        offsets, order = input._sample_rows()
        return input.replace_feature(group_norm_act(input.features, self.num_groups, self.weight, self.bias, self.eps, act, residual,
                                                    offsets, order))


def takes_act(module):
    """whether a module is a group norm whose kernels may run what follows it: one with hooks, or a subclass, is called for the norm alone"""
    return type(module) is SparseGroupNorm and not _hooked(module)


def norm_act(x, norm, residual=None, relu=True):
    """relu?(norm(x) (+ residual)) for a SparseConvTensor x and a norm of either kind -> SparseConvTensor"""
    if takes_act(norm):
        return norm(x, act="relu" if relu else None, residual=residual)
    if isinstance(norm, SparseGroupNorm):
        out = norm(x)
        y = out.features if residual is None else out.features + residual.to(out.features.dtype)
        return out.replace_feature(torch.relu(y) if relu else y)
    return x.replace_feature(bn_act(x.features, norm, residual=residual, relu=relu))
