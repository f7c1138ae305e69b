"""Losses over rows of a vocabulary softmax in memory: where one value could hide another, where two answers share a launch, and
their gradients against differences along the gradient itself."""
import pytest
import torch

from test_gpu_vocab_rows import EXP, dev, labels_of, make  # noqa: F401

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


def test_answers_that_pass_a_launch_only_one_by_one(dev):
    """Two answers of 2^13 x 1 040 rows, 256 threads a row: 2^31.02 threads each, more than 2^32 together.  All rows but a few are
    dead and every row of logits is the same one in memory (strides of 0)."""
    from pevae_amd import ops
    P, L, V = 1 << 13, 1040, 8203
    z = make((V,), torch.bfloat16, dev, 410)
    y = torch.full((P, L), -7, dtype=torch.int64, device=dev)
    y[0, 0], y[P - 1, L - 1], y[77, 3] = 5, V - 1, 100
    yr = y.clone()
    yr[P - 1, L - 1] = 7
    rows = z.expand(P, L, V)
    loss, rc, rr = ops.vocab_preference_loss(rows, y, rows, yr, ignore_index=-7, beta=0.3, avg_type=None)
    lp = torch.log_softmax(z.double(), -1)
    want_c, want_r = torch.zeros(P, dtype=torch.float64, device=dev), torch.zeros(P, dtype=torch.float64, device=dev)
    want_c[0], want_c[77], want_c[P - 1] = lp[5], lp[100], lp[V - 1]
    want_r[0], want_r[77], want_r[P - 1] = lp[5], lp[100], lp[7]
    for got, want in ((rc, 0.3 * want_c), (rr, 0.3 * want_r)):
        assert float((got.double() - want).abs().max()) <= EXP * (1 + float(want.abs().max()))
    total = -torch.nn.functional.logsigmoid(0.3 * (want_c - want_r)).sum()
    assert abs(float(loss) - float(total)) <= EXP * float(total)


def test_preference_of_an_impossible_answer(dev):
    """Rewards of -inf and inf: the term that does not count (label_smoothing 0 or 1) adds nothing, the other one 0 or inf."""
    from pevae_amd import ops
    y = torch.ones(1, 1, dtype=torch.int64, device=dev)
    zero = torch.zeros(1, 1, device=dev)
    none = torch.full((1, 1), -INF, device=dev)
    for c, r, smooth, want in ((none, zero, 0.0, INF), (none, zero, 1.0, 0.0), (zero, none, 0.0, 0.0), (zero, none, 1.0, INF),
                               (none, zero, 0.25, INF), (zero, none, 0.25, INF)):
        c, r = c.clone().requires_grad_(), r.clone().requires_grad_()
        loss, _, _ = ops.preference_loss(c, y, r, y, beta=0.5, label_smoothing=smooth)
        assert float(loss) == want, (smooth, float(loss))
        dc, dr = torch.autograd.grad(loss, [c, r])
        sig = 0.0 if float(c) < 0 else 1.0              # of the difference of the rewards
        slope = 0.5 * (smooth * sig - (1 - smooth) * (1 - sig))
        assert float(dc) == slope and float(dr) == -slope


@pytest.mark.parametrize("kind", ["logp", "distill", "policy", "preference"])
def test_gradients_against_differences_along_them(dev, kind):
    """Along w = d / |d| the derivative is |d|.  Central differences at h and 2 h, combined so that the h^2 term cancels, leave
    h^4 / 30 of the fifth derivative along w; each loss is off by EXP (1 + |loss|) at most, which enters
    (4 / 3 + 1 / 6) / h times.  Fifth derivatives: those of ln sum e^z along a unit direction are cumulants of a variable of
    range R <= sqrt 2, |k5| = |m5 - 10 m2 m3| <= R^5 / 4 + 10 (R^2 / 4) (R^3 / 4) < 5 (with |m_n| <= R^n / 4); the entropy adds a
    factor of z (below 10 here); a ratio e^lp of about 5 has e^lp times the complete Bell polynomial of such derivatives, below
    52 R^5 = 300, over ten live tokens.  120 covers each.  The ratios of the policy loss stay on their side of the clip range."""
    from pevae_amd import ops
    B, L, V, K, h = 3, 4, 257, 9, 0.05
    z = make((B, L, V), torch.float32, dev, 420, 1.0)
    y = labels_of((B, L), V, dev, 421, 0.2)
    t = make((B, L, V), torch.float32, dev, 422).topk(K, -1)
    lp0 = ops.token_logprobs(z, y, ignore_index=-7)
    old = lp0 - torch.where(torch.arange(B * L, device=dev).view(B, L) % 2 == 0, 0.05, 1.5)     # ratios of 1.05 and 4.5; range 0.5 to 1.5
    adv = torch.tensor([1.0, -0.7, 0.4], device=dev)

    def loss_of(x):
        if kind == "logp":
            lp, H = ops.token_logprobs(x, y, ignore_index=-7, inv_temp=0.9, entropy=True)
            return (lp * old).sum() / 12 + H.sum() / 12
        if kind == "distill":
            return ops.distill_topk(x, t.indices, t.values, y, -7, 1.5, avg_type="word")
        if kind == "policy":
            return ops.vocab_policy_loss(x, y, old, adv, lp0 - 0.1, -7, clip=0.5, kl_coef=0.1, ent_coef=0.05)[0]
        return ops.vocab_preference_loss(x, y, x.flip(0), y.flip(0), lp0, lp0.flip(0) - 0.3, -7, beta=1.0)[0]

    x = z.clone().requires_grad_()
    loss = loss_of(x)
    d, = torch.autograd.grad(loss, x)
    size = float(d.double().norm())
    way = (d.double() / size).float()
    with torch.no_grad():
        at = {s: float(loss_of(z + s * h * way)) for s in (-2, -1, 1, 2)}
    diff = (4 * (at[1] - at[-1]) / 2 - (at[2] - at[-2]) / 4) / (3 * h)
    tol = h ** 4 / 30 * 120 + 1.5 * EXP * (1 + abs(float(loss))) / h
    assert abs(diff - size) <= tol
    assert tol <= 0.1 * size                # a gradient of 0, of the other sign, or a tenth off would not pass
