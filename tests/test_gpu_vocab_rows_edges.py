"""Losses over rows of a vocabulary softmax in memory where one value could hide another."""
import pytest
import torch

from test_gpu_vocab_rows import dev, make  # noqa: F401

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("kl", [0.0, 0.1])
def test_a_zero_advantage_hides_no_nan(dev, kl):
    """A token that names no word, a NaN log-probability and a NaN old log-probability make the loss and the row's gradient NaN at
    an advantage of 0 as well; an infinite ratio does not."""
    from pevae_amd import ops
    V = 60
    y = torch.tensor([[3, 4, 5], [6, 7, 8]], device=dev)
    adv = torch.zeros(2, device=dev)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        z = make((2, 3, V), dtype, dev, 400).requires_grad_()
        old = ops.token_logprobs(z, y).detach()
        cases = [(y.clone(), old.clone(), True) for _ in range(4)] + [(y.clone(), old.clone(), False)]
        cases[0][0][1, 2], cases[1][0][1, 2], cases[2][0][1, 2] = V, -1, (1 << 33) + 4
        cases[3][1][1, 2] = NAN
        cases[4][1][1, 2] = -INF                        # r is infinite: 0 times it is 0 here
        for t, o, lost in cases:
            for ent in (0.0, 0.1):
                loss, stats = ops.vocab_policy_loss(z, t, o, adv, old if kl else None, -7, kl_coef=kl, ent_coef=ent)
                d, = torch.autograd.grad(loss, z)
                rows = torch.zeros(2, 3, dtype=torch.bool, device=dev)
                rows[1, 2] = lost
                assert bool(torch.isnan(loss)) == lost and bool(torch.isnan(stats[0])) == lost
                assert torch.equal(torch.isnan(d).all(-1), rows) and torch.equal(torch.isnan(d).any(-1), rows)
    lp = old.clone().requires_grad_()
    for which in ("logp", "old", "ratio"):
        x, o = lp.detach().clone(), old.clone()
        if which == "ratio":
            o[1, 2] = -INF
        else:
            (x if which == "logp" else o)[1, 2] = NAN
        x.requires_grad_()
        loss, stats = ops.policy_loss(x, y, o, adv, old if kl else None, -7, kl_coef=kl)
        d, = torch.autograd.grad(loss, x)
        lost = which != "ratio"
        assert bool(torch.isnan(loss)) == lost and bool(torch.isnan(stats[0])) == lost
        assert torch.isnan(d).tolist() == [[False] * 3, [False, False, lost]]
    hid, w, b = (make(s, torch.float32, dev, k, 0.3).requires_grad_() for k, s in ((401, (2, 3, 16)), (402, (V, 16)), (403, (V,))))
    for t, o, lost in cases:
        loss, _ = ops.projected_policy_loss(hid, w, b, t, o, adv, old if kl else None, -7, kl_coef=kl, ent_coef=0.1)
        gh, = torch.autograd.grad(loss, hid)
        assert bool(torch.isnan(loss)) == lost and bool(torch.isnan(gh[1, 2]).all()) == lost and not bool(torch.isnan(gh[0]).any())
