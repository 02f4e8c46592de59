"""Orthogonalised updates for the training step: `orthogonalize` (Newton-Schulz steps on the GPU's matrix cores, many weights in one
call: pvx_orthogonalize) and `Muon`, the optimiser that applies them to momentum.

A convolution weight [Cout, kz, ky, kx, Cin] is the matrix [Cout, kz ky kx Cin] it multiplies unfolded features with.  `Muon` takes the
weights of two and more dimensions; norms, biases and the like belong to another optimiser (the training step's AdamW), and so does
the exchange of gradients between ranks (`dist.allreduce_gradients`, DistributedDataParallel): every rank makes the same update from
the averaged gradient."""
import struct

import torch

from . import _lib

# a s + b s^3 + c s^5: steepest at 0 of those that keep (0, 1] within about 0.7 .. 1.2 (published with the Muon optimiser, K. Jordan et al., 2024)
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_MATRICES, MAX_STEPS, MAX_SIDE = 64, 64, 2 ** 20      # of one call of the C entry


def _launch(mats, outs, steps, coefficients, eps):
    """mats, outs: contiguous matrices of one dtype on one device, none of them empty"""
    L = _lib.lib()
    dev, code = mats[0].device, _lib.DTYPE_CODE[mats[0].dtype]
    a, b, c = coefficients
    with _lib.on(dev):
        stream = _lib.raw_stream(dev)
        for at in range(0, len(mats), MAX_MATRICES):
            part = [v for m, o in zip(mats[at:at + MAX_MATRICES], outs[at:at + MAX_MATRICES]) for v in (m.data_ptr(), o.data_ptr(), *m.shape)]
            count = len(part) // 4
            table = struct.pack("QQii" * count, *part)
            size = L.pvx_orthogonalize_workspace_bytes(table, count, code)
            ws = mats[0].new_empty(size, dtype=torch.uint8)
            rc = L.pvx_orthogonalize(table, count, code, steps, a, b, c, eps, ws.data_ptr(), size, stream)
            if rc:
                _check_coefficients(steps, coefficients)
                _lib.check(rc, "pvx_orthogonalize")


def _check_coefficients(steps, coefficients):
    if not _lib.lib().pvx_orthogonalize_holds(steps, *coefficients):
        raise ValueError("%d steps of the coefficients %r do not keep the singular values within known bounds" % (steps, tuple(coefficients)))


def _check_options(o):
    """of a parameter group of Muon"""
    if not o["lr"] >= 0.0 or not 0.0 <= o["momentum"] < 1.0 or not o["weight_decay"] >= 0.0:
        raise ValueError("lr and weight_decay must not be negative and momentum must be in [0, 1): got %r, %r, %r"
                         % (o["lr"], o["weight_decay"], o["momentum"]))
    if not 0 <= o["steps"] <= MAX_STEPS or not o["eps"] >= 0.0 or len(o["coefficients"]) != 3:
        raise ValueError("steps must be 0 .. %d and eps not negative, with three coefficients: got %r, %r, %r"
                         % (MAX_STEPS, o["steps"], o["eps"], o["coefficients"]))
    _check_coefficients(int(o["steps"]), o["coefficients"])


def orthogonalize(matrices, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """Newton-Schulz orthogonalisation: each matrix M becomes X after `steps` times X <- a X + (b A + c A A) X with A = X X^T, from
    X = M / (|M|_F + eps) (with the shorter side first), (a, b, c) = coefficients: the singular vectors of M with singular values near 1.

    matrices: a matrix [r, c], a batch of them [B, r, c], or a list or tuple of matrices of any sizes; float32 / float16 / bfloat16, on the
    GPU.  The result has the same form, in the inputs' dtypes; whatever they are, the products are as accurate as binary32's.  No gradient flows through it.
    Matrices of one dtype go through the GPU together, up to 64 in a call: the tiles and parts of its products, and so the last bits of a
    result, depend on the list that a matrix is in; the same list gives the same bits.  Coefficients whose polynomial does not keep the singular values
    within known bounds over the steps (a root or a fixed point that repels inside [0, 1], or growth past 1e9) are refused."""
    one = isinstance(matrices, torch.Tensor)
    if one and matrices.dim() not in (2, 3):
        raise ValueError("a matrix [r, c] or a batch [B, r, c] is wanted, got %s" % (tuple(matrices.shape),))
    if len(coefficients) != 3:
        raise ValueError("three coefficients are wanted, got %d" % len(coefficients))
    steps, eps, coefficients = int(steps), float(eps), tuple(float(v) for v in coefficients)
    if not 0 <= steps <= MAX_STEPS or not eps >= 0.0:
        raise ValueError("steps must be 0 .. %d and eps not negative, got %r and %r" % (MAX_STEPS, steps, eps))
    with torch.no_grad():
        mats = list(matrices.detach().contiguous().unbind(0)) if one and matrices.dim() == 3 else [matrices] if one else list(matrices)
        groups, outs = {}, []
        for m in mats:
            if not isinstance(m, torch.Tensor) or m.dim() != 2:
                raise ValueError("matrices are wanted, got %s" % (tuple(m.shape) if isinstance(m, torch.Tensor) else type(m).__name__,))
            if not m.is_cuda:
                raise RuntimeError("orthogonalize runs on the GPU only (no CPU fallback): got a matrix on %s" % m.device)
            if m.dtype not in _lib.DTYPE_CODE:
                raise TypeError("unsupported dtype %s" % m.dtype)
        if one and matrices.dim() == 3:
            whole = torch.empty(matrices.shape, dtype=matrices.dtype, device=matrices.device)
            outs = list(whole.unbind(0))
        else:
            outs = [m.new_empty(m.shape) for m in mats]
        for m, o in zip(mats, outs):
            if m.numel() > 0:
                g = groups.setdefault((m.dtype, m.device), ([], []))
                g[0].append(m.contiguous())
                g[1].append(o)
        for g in groups.values():
            _launch(g[0], g[1], steps, coefficients, eps)
    if one:
        return whole if matrices.dim() == 3 else outs[0]
    return type(matrices)(outs) if isinstance(matrices, (list, tuple)) and type(matrices) in (list, tuple) else outs


class Muon(torch.optim.Optimizer):
    """momentum buf <- momentum buf + grad; update = orthogonalize(grad + momentum buf, or buf without nesterov);
    p <- (1 - lr weight_decay) p - lr max(1, rows / cols)^0.5 update, for parameters of two and more dimensions taken as the matrix
    [shape[0], everything else], of at most 2^20 rows and columns.  All matrices of a group are orthogonalised together.  The momentum is
    float32 whatever the parameter's type (in 8 bits a gradient below 2^-8 of it would be lost), and so is all that follows up to the one
    rounding of the new parameter.  A step that is refused has changed nothing."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
        defaults = dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=int(steps), coefficients=tuple(coefficients),
                        eps=eps)
        _check_options(defaults)
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            _check_options(self.param_groups[-1])
            for p in self.param_groups[-1]["params"]:
                if p.dim() < 2:
                    raise ValueError("Muon takes parameters of two and more dimensions, got %s: give the others to another optimiser"
                                     % (tuple(p.shape),))
        except Exception:
            self.param_groups.pop()
            raise

    def _groups_with_gradients(self):
        """(group, its parameters that have a gradient) of every group, all of them looked at before any state changes"""
        groups = []
        for group in self.param_groups:
            _check_options(group)
            params = [p for p in group["params"] if p.grad is not None and p.numel() > 0]
            for p in params:
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                if max(p.shape[0], p.numel() // p.shape[0]) > MAX_SIDE:
                    raise ValueError("matrices have at most %d rows and columns, got a parameter %s" % (MAX_SIDE, tuple(p.shape)))
                if not p.is_cuda:
                    raise RuntimeError("orthogonalize runs on the GPU only (no CPU fallback): got a matrix on %s" % p.device)
                if p.dtype not in _lib.DTYPE_CODE:
                    raise TypeError("unsupported dtype %s" % p.dtype)
            if params:
                groups.append((group, params))
        return groups

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)              # which gives every state its parameter's type
        saved = [state_dict["state"].get(k, {}) for group in state_dict["param_groups"] for k in group["params"]]
        for p, state in zip((p for group in self.param_groups for p in group["params"]), saved):
            if "momentum_buffer" in state:
                self.state[p]["momentum_buffer"] = state["momentum_buffer"].to(device=p.device, dtype=torch.float32)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group, params in self._groups_with_gradients():
            for p in params:
                if "momentum_buffer" not in self.state[p]:
                    self.state[p]["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
            grads = [p.grad.float() for p in params]                         # (of float32: the gradient itself)
            bufs = [self.state[p]["momentum_buffer"] for p in params]
            torch._foreach_mul_(bufs, group["momentum"])
            torch._foreach_add_(bufs, grads)
            updates = torch._foreach_add(grads, bufs, alpha=group["momentum"]) if group["nesterov"] else bufs
            mats = orthogonalize([u.reshape(u.shape[0], -1) for u in updates], group["steps"], group["coefficients"], group["eps"])
            wide = [p if p.dtype == torch.float32 else p.float() for p in params]
            if group["weight_decay"] != 0.0:
                torch._foreach_mul_(wide, 1.0 - group["lr"] * group["weight_decay"])
            by_scale = {}
            for p, o in zip(wide, mats):
                by_scale.setdefault(max(1.0, o.shape[0] / o.shape[1]) ** 0.5, []).append((p, o.view(p.shape)))
            for scale, pairs in by_scale.items():
                torch._foreach_add_([p for p, _ in pairs], [o for _, o in pairs], alpha=-group["lr"] * scale)
            narrow = [(p, q) for p, q in zip(params, wide) if p is not q]
            if narrow:
                torch._foreach_copy_([p for p, _ in narrow], [q for _, q in narrow])
        return loss
