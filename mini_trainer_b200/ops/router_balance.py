"""A router's choice of experts with the losses that keep all of them in use.

``route_balanced`` of either backend takes the logits ``[T, E]`` of a layer's router and returns what ``moe.route`` does, ``(probs, topi, w)``: the fp32
softmax, the ``k`` largest logits of each token (the lower expert of equal ones; what is not a number counts as the largest) and their probabilities, renormalised
over the chosen ones where ``renorm``; and with them a ``RouterBalance``. For every packed sample of ``n`` counted tokens, ``c_e`` of whose (token, slot) pairs
chose expert ``e``, and with ``P_e`` the sum of its probabilities over them:

* ``loss``    ``E / n^2 sum_e c_e P_e``: ``k`` where all experts are used alike, more where they are not (the load-balancing loss that Mixtral's configuration
              weighs by ``router_aux_loss_coef``, for one layer; there over the whole batch, which is one sample here)
* ``z_loss``  the mean of ``logsumexp(logits)^2``, which keeps the logits small

``route_balanced_bwd`` is the gradient of the logits through the weights and both losses, in one pass. Counts are constants of it. Tokens that are not counted, and
those outside all samples, are routed like the others and get their weights' gradient, but have no part in a sample's losses and counts, whatever their
logits are; a sample without counted tokens has losses of zero. The factors of the losses' gradients are tensors, one number per sample, so they can stay on the device.
"""
from __future__ import annotations

import torch

MOST_EXPERTS, MOST_CHOSEN, _BLOCKS_PER_SM = 512, 32, 2   # of csrc/route_balance.cu


class RouterBalance:
    """What the losses of a router are, and what their gradient needs.

    * ``loss``, ``z_loss``  [S] fp32
    * ``counts``            [S, E] int32 pairs that chose an expert
    * ``tokens``            [S] int32 counted tokens
    * ``lse``               [T] fp32 logsumexp of every token's logits
    * ``sample``            [T] int32 sample whose losses a token is in, -1 for none
    * ``usage``             [S, E] fp32 ``E counts / tokens^2``, what an expert's probability weighs in its sample's loss
    * ``inverse``           [T] fp32 one over the sum of a token's chosen probabilities, one where they are not renormalised

    The kernels leave all of them in one buffer of 32-bit words, in the order of ``NAMES``; they are tensors when they are asked for, which a layer's step does for few of them.
    """

    NAMES = ("usage", "counts", "tokens", "sample", "loss", "z_loss", "lse", "inverse")
    WHOLE = ("counts", "tokens", "sample")

    def __init__(self, T, E, S, words=None, **tensors):
        self.T, self.E, self.S, self.words = T, E, S, words
        self.__dict__.update(tensors)

    def offsets(self):
        """First word of each of ``NAMES``, and the number of words."""
        T, S, c = self.T, self.S, self.S * self.E
        d = 2 * c + S + T
        return 0, c, 2 * c, 2 * c + S, d, d + S, d + 2 * S, d + 2 * S + T, d + 2 * S + 2 * T

    def __getattr__(self, name):   # not there yet
        words = self.__dict__.get("words")
        if words is None or name not in self.NAMES:
            raise AttributeError(name)
        i, at = self.NAMES.index(name), self.offsets()
        if name not in self.WHOLE:
            words = self.__dict__.get("numbers")
            if words is None:
                words = self.__dict__["numbers"] = self.words.view(torch.float32)
        self.__dict__[name] = t = words.as_strided((self.S, self.E), (self.E, 1), at[i]) if i < 2 else words.as_strided((at[i + 1] - at[i],), (1,), at[i])
        return t


def _refuse(what, t, dtype, shape, device):
    raise ValueError(f"{what}: expected contiguous {dtype} {tuple(shape)} on {device}, not {tuple(t.shape)} {t.dtype} on {t.device} with strides {t.stride()}")


def _expect(what, t, dtype, shape, device):
    if t is not None and (t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous()):
        _refuse(what, t, dtype, shape, device)


def check(logits, k, cu_seqlens, counted):
    """``(T, E, S)`` of a call's arguments, which are refused where they have no right answer. Starts of samples are read by the kernels: ascending, from 0 to T at most."""
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32) or not logits.is_contiguous():
        raise ValueError(f"router logits are contiguous bf16 or fp32 rows, not {tuple(logits.shape)} {logits.dtype} with strides {logits.stride()}")
    T, E = logits.shape
    if not 0 < E <= MOST_EXPERTS or T >= 1 << 30:
        raise ValueError(f"{T} tokens and {E} experts: the kernels take up to 2^30 and {MOST_EXPERTS}")
    if isinstance(k, bool) or not isinstance(k, int) or not 0 < k <= min(E, MOST_CHOSEN):
        raise ValueError(f"a token chooses 1 to {min(E, MOST_CHOSEN)} of {E} experts, not {k}")
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2:
            raise ValueError(f"starts of samples are a list of at least two, not {tuple(cu_seqlens.shape)}")
        _expect("cu_seqlens", cu_seqlens, torch.int32, cu_seqlens.shape, logits.device)
    if counted is not None:
        _expect("counted", counted, torch.bool, (T,), logits.device)
    return T, E, 1 if cu_seqlens is None else cu_seqlens.shape[0] - 1


def check_bwd(probs, topi, w, dw, bal, dloss, dz, dtype):
    """``(T, E, k, S)`` of a gradient's arguments."""
    if probs.dim() != 2 or topi.dim() != 2:
        raise ValueError("probs [T, E] and topi [T, k] are what the forward returned")
    (T, E), k, S, device = probs.shape, topi.shape[1], bal.S, probs.device
    if (T, E) != (bal.T, bal.E) or not 0 < k <= min(E, MOST_CHOSEN):
        raise ValueError(f"{T} tokens, {k} of {E} experts: not what the forward returned")
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"the gradient of the logits is bf16 or fp32, not {dtype}")
    if dw is None and dloss is None and dz is None:
        raise ValueError("without a gradient of the weights or of a loss there is nothing to do")
    f32, pairs = torch.float32, (T, k)
    _expect("probs", probs, f32, (T, E), device)
    _expect("topi", topi, torch.int64, pairs, device)
    _expect("w", w, f32, pairs, device)
    _expect("dw", dw, f32, pairs, device)
    _expect("dloss", dloss, f32, (S,), device)
    _expect("dz", dz, f32, (S,), device)
    if (bal.lse if bal.words is None else bal.words).device != device:
        raise ValueError(f"the losses are on another device than the probabilities, {device}")
    return T, E, k, S


# -- plain forms ----------------------------------------------------------------------------
def _samples(T, cu, counted, device):
    """``[T]`` int64: the sample whose losses a token is in, or -1."""
    at = torch.arange(T, device=device)
    sample = torch.zeros_like(at) if cu is None else torch.searchsorted(cu[1:].long().contiguous(), at, right=True)
    if cu is not None:
        sample = torch.where((sample < cu.shape[0] - 1) & (at >= cu[0]), sample, -1)
    return sample if counted is None else torch.where(counted, sample, -1)


def plain(logits, k, renorm, cu_seqlens=None, counted=None):
    T, E, S = check(logits, k, cu_seqlens, counted)
    l = logits.float()
    probs, lse = torch.softmax(l, -1), torch.logsumexp(l, -1)
    topi = torch.argsort(l, dim=-1, descending=True, stable=True)[:, :k].contiguous()
    top = probs.gather(1, topi)
    w = top / top.sum(-1, keepdim=True) if renorm else top
    sample = _samples(T, cu_seqlens, counted, l.device)
    ok = sample >= 0
    sums = torch.zeros(S, E, dtype=torch.float64, device=l.device).index_add_(0, sample[ok], probs[ok].double())
    counts = torch.zeros(S * E, dtype=torch.int64, device=l.device)
    chosen = (sample[ok, None] * E + topi[ok]).reshape(-1)
    counts = counts.index_add_(0, chosen, torch.ones_like(chosen)).view(S, E)
    tokens = torch.zeros(S, dtype=torch.int64, device=l.device).index_add_(0, sample[ok], torch.ones_like(sample[ok]))
    n = tokens.clamp_min(1).double()
    z = torch.zeros(S, dtype=torch.float64, device=l.device).index_add_(0, sample[ok], lse[ok].double().square())
    loss, z = (E * (counts * sums).sum(1) / n.square()).float(), (z / n).float()
    inverse = 1.0 / top.sum(-1) if renorm else torch.ones(T, device=l.device)
    usage = (E * counts / n.square()[:, None]).float()
    return probs, topi, w, RouterBalance(T, E, S, usage=usage, inverse=inverse, loss=loss, z_loss=z, counts=counts.to(torch.int32), tokens=tokens.to(torch.int32), lse=lse, sample=sample.to(torch.int32))


def plain_bwd(probs, topi, w, dw, renorm, bal, dloss=None, dz=None, dtype=torch.bfloat16):
    T, E, k, S = check_bwd(probs, topi, w, dw, bal, dloss, dz, dtype)
    ok = bal.sample >= 0
    sample = bal.sample.long()
    n = bal.tokens.clamp_min(1).float()
    g = torch.zeros_like(probs)
    if dw is not None:
        d = (dw - (dw * w).sum(-1, keepdim=True)) * bal.inverse[:, None] if renorm else dw
        g.scatter_add_(1, topi, d)
    if dloss is not None:
        g[ok] += (dloss[:, None] * bal.usage)[sample[ok]]
    g = g - (g * probs).sum(-1, keepdim=True)
    if dz is not None:
        g[ok] += (2.0 * bal.lse[ok] * (dz / n)[sample[ok]])[:, None]
    return (probs * g).to(dtype)


# -- kernels --------------------------------------------------------------------------------
def native(ops, logits, k, renorm, cu_seqlens=None, counted=None):
    T, E, S = check(logits, k, cu_seqlens, counted)
    ops.check_device(logits)
    dev, f32 = logits.device, torch.float32
    with ops.on_device():
        probs, topi, w = torch.empty(T, E, dtype=f32, device=dev), torch.empty(T, k, dtype=torch.int64, device=dev), torch.empty(T, k, dtype=f32, device=dev)
        bal = RouterBalance(T, E, S)
        usage, counts, tokens, sample, loss, z, lse, inverse, words = bal.offsets()
        bal.words = torch.empty(words, dtype=torch.int32, device=dev)
        if T == 0:
            bal.words.zero_()
            return probs, topi, w, bal
        rows, at = _BLOCKS_PER_SM * ops.sms + S, bal.words.data_ptr()
        scratch = torch.empty(rows * (E + 1), dtype=torch.int64, device=dev)   # held until the kernels are queued: nobody else is given it before
        part = scratch.data_ptr()
        ops._call("mtb200_route_balanced", logits.data_ptr(), logits.dtype is f32, None if cu_seqlens is None else cu_seqlens.data_ptr(), None if counted is None else counted.data_ptr(),
                  T, E, k, S, bool(renorm), probs.data_ptr(), topi.data_ptr(), w.data_ptr(), at + 4 * lse, at + 4 * inverse, at + 4 * sample, part, part + 8 * rows * E, rows,
                  at + 4 * loss, at + 4 * z, at + 4 * counts, at + 4 * tokens, at + 4 * usage, ops._st(), n=2)
    return probs, topi, w, bal


def native_bwd(ops, probs, topi, w, dw, renorm, bal, dloss=None, dz=None, dtype=torch.bfloat16):
    T, E, k, S = check_bwd(probs, topi, w, dw, bal, dloss, dz, dtype)
    ops.check_device(probs)
    with ops.on_device():
        out = torch.empty(T, E, dtype=dtype, device=probs.device)
        if T:
            if bal.words is not None:
                at = bal.words.data_ptr()
                usage, _, tokens, sample, _, _, lse, inverse, _ = (at + 4 * i for i in bal.offsets())
            else:
                usage, tokens, sample, lse, inverse = (t.data_ptr() for t in (bal.usage, bal.tokens, bal.sample, bal.lse, bal.inverse))
            ops._call("mtb200_route_balanced_bwd", probs.data_ptr(), topi.data_ptr(), w.data_ptr(), None if dw is None else dw.data_ptr(), lse, inverse, sample, usage, tokens,
                      None if dloss is None else dloss.data_ptr(), None if dz is None else dz.data_ptr(), T, E, k, S, bool(renorm), out.data_ptr(), dtype is torch.float32,
                      ops.status.data_ptr(), ops._st())
    return out
