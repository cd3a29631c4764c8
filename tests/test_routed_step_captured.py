"""Steps of a routed layer captured into a graph (the layer of ``test_routed_step``): what three replays leave is, bit for bit, what three runs leave."""
import pytest
import torch

from .test_routed_step import BAL, E, HEADZ, K, LENS, LR, MU, T, WD, Z, model


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
def test_replayed_steps_are_the_steps_run(wide):
    """``wide``: a head whose products split their reduction."""
    from mini_trainer_b200.ops import get_ops
    ops = get_ops(torch.device("cuda:0"))

    def make():
        w, x, t, cu, ok = model("cuda", torch.bfloat16, 5)
        if wide:
            g = torch.Generator().manual_seed(6)
            w["head"] = (torch.randn(30016, w["head"].shape[1], generator=g) / 4).bfloat16().cuda()
        moment = {k: torch.zeros(v.shape, device="cuda") for k, v in w.items()}
        master = {k: v.float().clone() for k, v in w.items()}
        coef, S, n = torch.full((1,), 0.5, device="cuda"), len(LENS), ok.sum()
        dbal, dz = torch.full((S,), BAL / S, device="cuda"), torch.full((S,), Z / S, device="cuda")

        def run():
            logits = x.float() @ w["router"].float().t()
            probs, topi, p, bal = ops.route_balanced(logits, K, True, cu, ok)
            picked = torch.einsum("th,eoh->teo", x.float(), w["experts"].float()).gather(1, topi[:, :, None].expand(-1, -1, x.shape[1]))
            y = (x.float() + (p[:, :, None] * picked).sum(1)).bfloat16()
            loss, lse = ops.linear_nll(y, w["head"], t)
            weight = torch.where(ok, torch.clamp(loss / (loss.sum() / n), 0.2, 3.0), 0.0) / n   # (loss is zero where not counted)
            dhead = torch.empty_like(w["head"])
            dy = ops.linear_nll_bwd(weight, y, w["head"], t, loss, lse, dhead, dlse=2 * HEADZ * lse / T).float()
            dl = ops.route_balanced_bwd(probs, topi, p, (dy[:, None] * picked).sum(-1), True, bal, dbal, dz, torch.float32)
            dexp = torch.stack([(dy * torch.where(topi == e, p, 0.0).sum(1)[:, None]).t() @ x.float() for e in range(E)])
            for k, g in (("head", dhead), ("router", dl.t() @ x.float()), ("experts", dexp)):
                ops.muon_step(master[k], moment[k], g.contiguous(), w[k], LR, MU, WD, coef)
            return loss, lse, bal.loss, bal.z_loss, bal.counts, dhead, dl
        return run, w, master, moment
    run, w, master, moment = make()
    run2, w2, master2, moment2 = make()
    first = {k: v.clone() for k, v in master.items()}
    want = [tuple(t.clone() for t in run()) for _ in range(3)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run2()
    for step in want:
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step))
    for a, b in ((w, w2), (master, master2), (moment, moment2)):
        assert all(torch.equal(a[k], b[k]) for k in a)
    # the weights were updated: an orthogonal matrix's norm, times LR and the scale, is what a step moves them by
    assert all(float((master[k] - first[k]).norm()) > 0.5 * LR * 0.2 * min(first[k].shape[-2:]) ** 0.5 for k in master)
    ops.check_status()
