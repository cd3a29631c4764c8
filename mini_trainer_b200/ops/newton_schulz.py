"""Matrices orthogonalised by Newton-Schulz products, and a parameter's update by its orthogonalised momentum (as the Muon optimiser does it).

``orthogonalise(g)`` of either backend takes a matrix ``[m, n]`` or a stack of them ``[..., m, n]``, bf16 or fp32, and returns in bf16, for each,

    ``X = g / (|g| + 1e-7)``, then ``steps`` times ``X <- (a I + b A + c A^2) X`` with ``A = X X^T``, ``(a, b, c) = (3.4445, -4.7750, 2.0315)``:

singular vectors stay, singular values above about a thousandth of the norm end between 0.7 and 1.2. A zero matrix stays zero; what is not finite stays in its matrix. Matrices may be as large as their type allows.
The kernels' result is 2e-3 to 4e-3 of its norm off, the rounding to bf16 included (matrices of a few rows, columns or entries: up to 2e-2). A norm far below 1e-7 makes the result itself next to nothing: they hold it to 2^-20 of
the norm that an orthogonal matrix of that size has, which is less than three digits of the result where the norm is below 1e-12.

``muon_step`` is one step of a parameter, or of a stack of parameters of one shape, in place:

    ``moment <- momentum moment + coef grad``;  ``u = coef grad + momentum moment`` (without ``nesterov``: ``moment``, as it is stored)
    ``master <- (1 - lr weight_decay) master - lr scale orthogonalised(u)``;  ``param_out <- master``

``scale`` defaults to ``0.2 sqrt(max(m, n))``, which gives the update the root mean square of an AdamW step. It is meant for the matrices inside the blocks; embeddings, the head and vectors
stay with ``adamw_step``. Matrices are whole here: a flat shard that cuts one is gathered first.

Beside the result, a call on the kernels holds a workspace of 8 bytes an element and 4 for each of the square of the shorter side (rows and sides in whole 64s: 1.3 GB for 64 of 2048 x 1024, 1.1 GB for 16384 of 128 x 16)
while it runs, unless it is one launch (csrc/newton_schulz.cu), which has none. The matrices of a stack have nothing to do with one another, so one that leaves no room for it is called in parts.
"""
from __future__ import annotations

import math

import torch

NS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
MOST_STEPS = 64


def _check_steps(steps):
    if isinstance(steps, bool) or not isinstance(steps, int) or not 1 <= steps <= MOST_STEPS:
        raise ValueError(f"1 to {MOST_STEPS} steps, not {steps}")


def check(g, steps):
    """``(stack, m, n)``; arguments without a right answer are refused."""
    if g.dim() < 2 or g.dtype not in (torch.bfloat16, torch.float32) or not g.is_contiguous():
        raise ValueError(f"expected contiguous bf16 or fp32 matrices [..., m, n], not {tuple(g.shape)} {g.dtype} with strides {g.stride()}")
    _check_steps(steps)
    (m, n), stack = g.shape[-2:], math.prod(g.shape[:-2])
    if max(m, n, stack) >= 1 << 24 or min(m, n) > 1 << 16 or g.numel() >= 1 << 40:
        raise ValueError(f"{stack} matrices of {m} x {n} are more than the kernels count")
    return stack, m, n


def check_muon(master, moment, grad, param_out, lr, momentum, weight_decay, grad_coef, scale, steps):
    """``(stack, m, n, keep, step)``: sizes, and the factors of the parameter and of the orthogonalised matrix."""
    stack, m, n = check(grad, steps)
    for what, t, types in (("master", master, (torch.float32,)), ("moment", moment, (torch.float32, torch.bfloat16)), ("param_out", param_out, (torch.bfloat16, torch.float32))):
        if what == "param_out" and t is None:
            continue
        if t.dtype not in types or t.shape != grad.shape or not t.is_contiguous() or t.device != grad.device:
            raise ValueError(f"{what}: expected contiguous {types[0]} {tuple(grad.shape)} on {grad.device}, not {tuple(t.shape)} {t.dtype} on {t.device} with strides {t.stride()}")
    held = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (master, moment, grad, param_out) if t is not None and t.device.type != "meta"]
    if any(a < d and c < b for i, (a, b) in enumerate(held) for c, d in held[:i]):
        raise ValueError("master, moment, gradient and working copy are memory of their own")
    scale = 0.2 * math.sqrt(max(m, n)) if scale is None else float(scale)
    for what, v in (("lr", lr), ("momentum", momentum), ("weight_decay", weight_decay), ("scale", scale), ("the gradient's factor", 0.0 if torch.is_tensor(grad_coef) else grad_coef)):
        if not math.isfinite(v):
            raise ValueError(f"{what} is a finite number, not {v}")
    if torch.is_tensor(grad_coef) and grad_coef.numel() != 1:
        raise ValueError(f"the gradient's factor is one number, not {tuple(grad_coef.shape)}")
    return stack, m, n, 1.0 - lr * weight_decay, lr * scale


# -- plain forms ----------------------------------------------------------------------------
def _iterate(x, steps):
    a, b, c = NS
    x = x.float()
    norm = torch.linalg.matrix_norm(x, keepdim=True)
    small = x * 2.0 ** -96   # where the squares are past the type's range, the numbers need not be
    x = torch.where(torch.isinf(norm), small / torch.linalg.matrix_norm(small, keepdim=True), x / (norm + EPS))
    right = x.shape[-2] > x.shape[-1]
    for _ in range(steps):
        g = x.mT @ x if right else x @ x.mT
        q = b * g + c * (g @ g)
        x = a * x + (x @ q if right else q @ x)
    return x


def plain(g, steps=5):
    check(g, steps)
    return _iterate(g, steps).to(torch.bfloat16)


def plain_muon(master, moment, grad, param_out, lr, momentum, weight_decay, grad_coef=1.0, nesterov=True, steps=5, scale=None):
    *_, keep, step = check_muon(master, moment, grad, param_out, lr, momentum, weight_decay, grad_coef, scale, steps)
    if grad.numel() == 0:
        return
    g = grad.float() * grad_coef
    moment.copy_(momentum * moment.float() + g)
    u = g + momentum * moment.float() if nesterov else moment
    master.mul_(keep).sub_(_iterate(u, steps), alpha=step)
    if param_out is not None:
        param_out.copy_(master)


# -- kernels --------------------------------------------------------------------------------
def _launches(ptr, steps, more):
    """One where the library has asked for no workspace, else two in front of the products, three of these a step and ``more`` behind them."""
    return 1 if ptr is None else 2 + 3 * steps + more


def _workspace(ops, m, n, stack, steps, device):
    """``(tensor, address, bytes)`` of a call's workspace; nothing where the library makes the call one launch, which takes none."""
    size = ops._fn["mtb200_newton_schulz_workspace"](m, n, stack, steps)
    if size == 0:
        return None, None, 0
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), size


def native(ops, g, steps=5):
    stack, m, n = check(g, steps)
    ops.check_device(g)
    with ops.on_device():
        out = torch.empty(g.shape, dtype=torch.bfloat16, device=g.device)
        if out.numel():
            ws, ptr, size = _workspace(ops, m, n, stack, steps, g.device)
            ops._call("mtb200_newton_schulz", g.data_ptr(), int(g.dtype is torch.bfloat16), out.data_ptr(), m, n, stack, steps, ptr, size, ops.status.data_ptr(), ops._st(),
                      n=_launches(ptr, steps, n % 8 != 0))
    return out


def native_muon(ops, master, moment, grad, param_out, lr, momentum, weight_decay, grad_coef=1.0, nesterov=True, steps=5, scale=None):
    stack, m, n, keep, step = check_muon(master, moment, grad, param_out, lr, momentum, weight_decay, grad_coef, scale, steps)
    ops.check_device(grad)
    if param_out is not None and param_out.dtype is not torch.bfloat16:
        raise ValueError(f"the working copy is bf16 on the kernels, not {param_out.dtype}")
    if grad.numel() == 0:
        return
    with ops.on_device():
        if not torch.is_tensor(grad_coef):
            coef = None if grad_coef == 1.0 else torch.full((1,), float(grad_coef), dtype=torch.float32, device=grad.device)
        else:
            coef = grad_coef.to(device=grad.device, dtype=torch.float32).reshape(1)
        ws, ptr, size = _workspace(ops, m, n, stack, steps, grad.device)
        ops._call("mtb200_muon_step", master.data_ptr(), moment.data_ptr(), int(moment.dtype is torch.bfloat16), grad.data_ptr(), int(grad.dtype is torch.bfloat16),
                  None if param_out is None else param_out.data_ptr(), None if coef is None else coef.data_ptr(), m, n, stack, steps, float(momentum), int(bool(nesterov)), keep, step,
                  ptr, size, ops.status.data_ptr(), ops._st(), n=_launches(ptr, steps, 1))
