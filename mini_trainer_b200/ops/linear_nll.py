"""Likelihoods of a language model's head that keep no logits, and their gradients for any weights per token.

``linear_nll`` of either backend returns ``(loss, lse)`` of the logits ``z = logit_scale * x @ w.T``: per token ``loss = lse - z[target]`` and the log-partition
``lse = logsumexp(z)``, both fp32. Nothing of the logits is stored: the product's epilogue reduces its tile. ``linear_nll_bwd`` takes the gradients of the
two, ``dloss`` and ``dlse`` (which may be ``None``), one number per token, and returns ``dx`` and writes ``dw``. So a program may look at the losses first and weight its tokens by them
(advantages, preference losses, a teacher's), score without gradients, or add a z-loss ``c lse^2`` (``dlse = 2 c lse``). It forms the logits again, piece by piece of the
vocabulary: a piece's gradient ``[T, columns]`` is all that exists at a time, ``dw`` of its rows is done with it and rounded once, ``dx`` is summed over the
pieces in fp32. ``linear_ce`` is the form for one uniform weight known beforehand: it needs the product once less.

A target equal to ``ignore_index`` has a loss of zero and no gradient (of ``lse`` either), whatever its logits are, but ``x`` is to be finite there too: a sum over all tokens
multiplies it by zero. Any other target outside the vocabulary counts as ignored and is reported by ``check_status``.
"""
from __future__ import annotations

import torch

PIECE_BYTES = 512 << 20   # of a piece's gradient, about
STATS_BYTES = 512 << 20   # of the forward's statistics at a time, about: 8 bytes per token and 128 columns


def check(x, w, targets, logit_scale):
    """``(T, H, V)``; arguments without a right answer are refused."""
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1] or x.dtype != w.dtype or x.device != w.device:
        raise ValueError(f"expected rows [T, H] and a weight [V, H] of one type on one device, not {tuple(x.shape)} {x.dtype} and {tuple(w.shape)} {w.dtype}")
    (T, H), V = x.shape, w.shape[0]
    if H < 1 or V < 1:
        raise ValueError(f"a weight of {V} x {H} has no logits")
    if targets.dtype != torch.int64 or targets.shape != (T,) or not targets.is_contiguous() or targets.device != x.device:
        raise ValueError(f"targets are {T} contiguous int64 numbers on {x.device}")
    if not 0.0 < abs(float(logit_scale)) < float("inf"):
        raise ValueError(f"logits are scaled by a finite number other than zero, not {logit_scale}")
    return T, H, V


def _per_token(what, t, T, device):
    if t is not None and (t.dtype is not torch.float32 or t.shape != (T,) or not t.is_contiguous() or t.device != device):
        raise ValueError(f"{what}: expected {T} contiguous fp32 numbers on {device}, not {tuple(t.shape)} {t.dtype} on {t.device}")


def _shares(out, others):
    """Whether ``out`` holds bytes of another tensor; of views with gaps, which the kernels do not take, whether both start at the same one."""
    if out.device.type == "meta":
        return False
    a, n = out.data_ptr(), out.nbytes
    for t in others:
        if t is not None and a < (b := t.data_ptr()) + t.nbytes and b < a + n and (a == b or out.is_contiguous() and t.is_contiguous()):
            return True
    return False


def check_bwd(dloss, x, w, targets, loss, lse, dw_out, logit_scale, dlse):
    T, H, V = check(x, w, targets, logit_scale)
    for what, t in (("dloss", dloss), ("loss", loss), ("lse", lse)):
        if t is None:
            raise ValueError(f"{what}: expected {T} contiguous fp32 numbers on {x.device}")
        _per_token(what, t, T, x.device)
    _per_token("dlse", dlse, T, x.device)
    if _shares(dw_out, (w, x, targets, dloss, loss, lse, dlse)):   # all of which the pieces behind the first read again
        raise ValueError("the weight's gradient goes to memory of its own")
    if dw_out.dtype != w.dtype or dw_out.shape != w.shape or dw_out.device != w.device:
        raise ValueError(f"the weight's gradient is {w.dtype} {tuple(w.shape)} on {w.device}, not {dw_out.dtype} {tuple(dw_out.shape)} on {dw_out.device}")
    return T, H, V


# -- plain forms ----------------------------------------------------------------------------
def columns(targets, V, ignore_index):
    """Which targets are a column that counts, and whether there are others that are not ``ignore_index``."""
    inside, other = (targets >= 0) & (targets < V), targets != ignore_index
    return inside & other, (other & ~inside).any()


def plain(x, w, targets, ignore_index=-100, logit_scale=1.0, chunk=2048):
    T, H, V = check(x, w, targets, logit_scale)
    loss, lse = (torch.zeros(T, dtype=torch.float32, device=x.device) for _ in range(2))
    ok, _ = columns(targets, V, ignore_index)
    for a in range(0, T, chunk):
        z = (x[a:a + chunk].float() @ w.float().t()) * logit_scale
        t = targets[a:a + chunk]
        lse[a:a + chunk] = torch.logsumexp(z, -1)
        picked = z.gather(1, t.clamp(0, V - 1).unsqueeze(1)).squeeze(1)
        loss[a:a + chunk] = torch.where(ok[a:a + chunk], lse[a:a + chunk] - picked, 0.0)
    return loss, lse


def plain_bwd(dloss, x, w, targets, loss, lse, dw_out, accumulate_dw=False, ignore_index=-100, logit_scale=1.0, dlse=None, chunk=2048):
    T, H, V = check_bwd(dloss, x, w, targets, loss, lse, dw_out, logit_scale, dlse)
    dx, dw, wf = torch.empty_like(x), torch.zeros(w.shape, dtype=torch.float32, device=x.device), w.float()
    ok, _ = columns(targets, V, ignore_index)
    for a in range(0, T, chunk):
        xc, t = x[a:a + chunk].float(), targets[a:a + chunk]
        d, dz = dloss[a:a + chunk], 0.0 if dlse is None else dlse[a:a + chunk]
        g = torch.exp((xc @ wf.t()) * logit_scale - lse[a:a + chunk, None]) * (d + dz).unsqueeze(1)
        l = loss[a:a + chunk]
        g.scatter_(1, t.clamp(0, V - 1).unsqueeze(1), (d * torch.expm1(-l) + dz * torch.exp(-l)).unsqueeze(1))
        g = torch.where(ok[a:a + chunk, None], g, 0.0) * logit_scale
        dx[a:a + chunk] = (g @ wf).to(x.dtype)
        dw += g.t() @ xc
    if accumulate_dw:
        dw += dw_out.float()
    dw_out.copy_(dw.to(dw_out.dtype))
    return dx


# -- kernels --------------------------------------------------------------------------------
def _check_native(ops, x, w, *more):
    ops.check_device(x)
    H = x.shape[1]
    if x.dtype is not torch.bfloat16 or H % 8:
        raise ValueError(f"the kernels take bf16 rows of a multiple of 8, not {H} {x.dtype}")
    if any(not t.is_contiguous() or t.data_ptr() & 15 for t in (x, w, *more)):
        raise ValueError("rows, the weight and its gradient are contiguous and start on 16 bytes")
    if max(x.shape[0], w.shape[0]) >= 1 << 30:
        raise ValueError(f"{x.shape[0]} tokens and {w.shape[0]} columns are more than the kernels count")


def _form(ops, T, H):
    """Kernel of the two products: as for logits with a cap, whose epilogue does about the same."""
    from . import gemm_plan
    return gemm_plan.capped_form(T, H, ops.use_gemm2, 0 if ops.pair_max_flops <= 0 and not ops.use_gemm2 else ops.cta_pairs())


def native(ops, x, w, targets, ignore_index=-100, logit_scale=1.0):
    T, H, V = check(x, w, targets, logit_scale)
    _check_native(ops, x, w)
    with ops.on_device():
        loss, lse = torch.empty(T, dtype=torch.float32, device=x.device), torch.empty(T, dtype=torch.float32, device=x.device)
        if T == 0:
            return loss, lse
        pieces = -(-V // 128)
        rows = min(T, max(256, STATS_BYTES // (8 * pieces) // 256 * 256))
        scratch = torch.empty(rows * (2 * pieces + 1), dtype=torch.float32, device=x.device)   # statistics, and the targets' logits
        stats, at, form, st, status = scratch.data_ptr(), scratch.data_ptr() + 8 * rows * pieces, _form(ops, rows, H), ops._st(), ops.status.data_ptr()
        for a in range(0, T, rows):
            n, t = min(rows, T - a), targets.data_ptr() + 8 * a
            ops._call("mtb200_linear_nll", x.data_ptr() + 2 * a * H, w.data_ptr(), t, stats, at, n, V, H, float(logit_scale), ignore_index, form, loss.data_ptr() + 4 * a, lse.data_ptr() + 4 * a, status, st, n=2)
    return loss, lse


def piece_columns(T: int, V: int) -> int:
    """Columns of a piece: as few equal pieces as ``PIECE_BYTES`` allow, of whole tiles, and of at least two of them however many tokens there are."""
    most = max(512, PIECE_BYTES // 2 // max(T, 1) // 256 * 256)
    if V <= most:
        return V
    pieces = -(-V // most)
    return -(-V // (pieces * 256)) * 256


def native_bwd(ops, dloss, x, w, targets, loss, lse, dw_out, accumulate_dw=False, ignore_index=-100, logit_scale=1.0, dlse=None):
    T, H, V = check_bwd(dloss, x, w, targets, loss, lse, dw_out, logit_scale, dlse)
    _check_native(ops, x, w, dw_out)
    with ops.on_device():
        dx = torch.empty_like(x)
        if T == 0:
            if not accumulate_dw:
                dw_out.zero_()
            return dx
        n = piece_columns(T, V)
        ldz = -(-n // 64) * 64   # rows of whole 128 bytes
        dz = torch.empty(T, ldz, dtype=torch.bfloat16, device=x.device)
        dx32 = torch.empty(T, H, dtype=torch.float32, device=x.device) if n < V else None
        form, scale, own = _form(ops, T, H), float(logit_scale), ops.own_counters()   # (64 rows of 1024, 151936 columns, captured: 202 us, and 650 with the sum over the vocabulary in one part)
        for a in range(0, V, n):
            c = min(n, V - a)
            wc, dwc = (w, dw_out) if c == V else (w[a:a + c], dw_out[a:a + c])
            ops._call("mtb200_gemm_nll", x.data_ptr(), H, wc.data_ptr(), dz.data_ptr(), ldz, targets.data_ptr(), loss.data_ptr(), lse.data_ptr(), dloss.data_ptr(),
                      None if dlse is None else dlse.data_ptr(), T, c, H, scale, ignore_index, a, V, form, ops.status.data_ptr(), ops._st(), tag="gemm_nt_nll")
            ops.gemm(dz, True, x, True, dwc, c, H, T, residual=dwc if accumulate_dw else None, alpha=scale, counters=own)
            if dx32 is None:
                ops.gemm(dz, False, wc, True, dx, T, H, c, alpha=scale, counters=own)
            else:
                ops.gemm(dz, False, wc, True, dx32, T, H, c, residual=dx32 if a else None, alpha=scale, counters=own)
        if dx32 is not None:
            ops._call("mtb200_f32_to_bf16", dx.data_ptr(), dx32.data_ptr(), T * H, 0, ops._st())
    return dx
