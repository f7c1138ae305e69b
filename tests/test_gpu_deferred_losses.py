"""Losses over a decoder's DeferredLogProbs on the GPU: scoring and training on one output.
(H, V) = (512, 5003) takes the fused vocabulary kernels, (64, 211) the tile ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu

PATHS = [(512, 5003), (64, 211)]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def decoder(dev, H, V, L=6, E=24, seed=7):
    from pevae_amd.enc2dec import decoders as D
    torch.manual_seed(seed)
    return D.DecoderRNN(V, L, E, H, 1, 2, 3, rnn_cell="gru", embedding=torch.nn.Embedding(V, E, padding_idx=0)).to(dev)


def answers(dev, B, L, V, seed=8):
    gen = torch.Generator(device=dev).manual_seed(seed)
    ids = torch.randint(4, V, (B, L), generator=gen, device=dev)
    y = torch.cat([ids[:, 1:], torch.zeros(B, 1, dtype=torch.long, device=dev)], 1)
    y[0, 3:], y[B - 1, 1:] = 0, 0
    h0 = torch.randn(1, B, 1, generator=gen, device=dev)
    return ids, y, h0, torch.randn(B, generator=gen, device=dev)


@pytest.mark.parametrize("H,V", PATHS)
@pytest.mark.parametrize("route", ["deferred", "dense"])
def test_scoring_and_training_on_one_output(dev, H, V, route):
    """The first step of an on-policy update: the old policy is the output that is then trained.  Every loss has the gradient
    that it has on an output of its own (the same kernels on the same operands: the same bits)."""
    from pevae_amd import criterions
    from pevae_amd.enc2dec import decoders as D
    B, L = 5, 6
    dec = decoder(dev, H, V)
    ids, y, h0, adv = answers(dev, B, L, V)
    h0 = (h0 * 0.3).expand(1, B, H).contiguous()
    params = list(dec.parameters())
    nll, policy, ppl = criterions.NLLEntropy(0, None), criterions.ClippedPolicyLoss(0, None), criterions.Perplexity(0, None)
    distill = criterions.TopKDistill(0, None)
    t = torch.randn(B, L, V, device=dev).topk(4, -1)

    def output():
        return dec(B, ids, h0, mode=D.TEACH_FORCE)[0]

    def view(out):
        return out if route == "deferred" else out.materialize()

    def score(out):
        with torch.no_grad():
            ppl(view(out), y), nll(view(out), y)
            return criterions.token_log_probs(view(out), y, 0)

    losses = [lambda o, old: nll(view(o), y), lambda o, old: policy(view(o), y, old, adv)[0], lambda o, old: ppl(view(o), y),
              lambda o, old: distill(view(o), y, t.indices, t.values),
              lambda o, old: policy(view(o), y, old, adv)[0] + nll(view(o), y),
              lambda o, old: nll(view(o), y) + policy(view(o), y, old, adv)[0]]
    old = score(output())
    for loss in losses:
        for p in params:
            p.grad = None
        loss(output(), old).backward()
        want = [None if p.grad is None else p.grad.clone() for p in params]
        for p in params:
            p.grad = None
        out = output()
        mine = score(out)
        assert torch.equal(mine, old) and not mine.requires_grad
        got = loss(out, mine)
        assert got.requires_grad
        got.backward()
        for p, w in zip(params, want):
            assert (p.grad is None) == (w is None) and (w is None or torch.equal(p.grad, w))
        assert float(dec.project.weight.grad.abs().max()) > 0


def test_ignored_labels_of_any_number(dev):
    """Rows of an ignored label are dead whatever its number, also where it does not fit 32 bits."""
    from pevae_amd.enc2dec import decoders as D
    gen = torch.Generator(device=dev).manual_seed(31)
    for H, V in PATHS:
        hid, w, b = (torch.randn(*s, generator=gen, device=dev) * 0.3 for s in ((2, 5, H), (V, H), (V,)))
        w.requires_grad_()
        y = torch.randint(1, V, (2, 5), generator=gen, device=dev)
        want = D.DeferredLogProbs(hid, w, b, 1.0).token_logp(y, 0)
        for ignore in (-1, V, V + 9, -100, 1 << 40, -(1 << 40)):
            dead = y.clone()
            dead[1, 2:] = ignore
            got = D.DeferredLogProbs(hid, w, b, 1.0).token_logp(dead, ignore)
            assert float(got[1, 2:].abs().max()) == 0.0 and torch.equal(got[0], want[0]) and torch.equal(got[1, :2], want[1, :2]), ignore


BAD = (lambda V: V, lambda V: -1, lambda V: (1 << 40) + 5, lambda V: -(1 << 50))


@pytest.mark.parametrize("H,V", PATHS + [(512, 4096 + 77)])
@pytest.mark.parametrize("ignore", [0, -7])
@pytest.mark.parametrize("frozen", [False, True])
def test_labels_that_name_no_word(dev, H, V, ignore, frozen):
    """A live label outside [0, V) has a NaN log-probability and a NaN gradient of its state; the other rows keep theirs.  With
    frozen states and weights the kernel without a backward pass runs."""
    from pevae_amd import criterions, ops
    from pevae_amd.enc2dec import decoders as D
    gen = torch.Generator(device=dev).manual_seed(30)
    B, L = 3, 7
    hid, w, b = (torch.randn(*s, generator=gen, device=dev) * 0.3 for s in ((B, L, H), (V, H), (V,)))
    xs = hid, w, b = [x.requires_grad_(not frozen) for x in (hid, w, b)]
    y = torch.randint(1, V, (B, L), generator=gen, device=dev)
    y[0, 5:], y[2, 2] = ignore, ignore
    places = [(0, 1), (1, 0), (1, 6), (2, 4)]
    bad = y.clone()
    for (i, j), f in zip(places, BAD):
        bad[i, j] = f(V)
    hit = bad != y
    want = D.DeferredLogProbs(hid, w, b, 1.0).token_logp(y, ignore)
    out = D.DeferredLogProbs(hid, w, b, 1.0)
    got = out.token_logp(bad, ignore)
    assert torch.equal(torch.isnan(got), hit) and torch.equal(got[~hit], want[~hit])
    old, adv = (want.detach() - 0.1), torch.ones(B, device=dev)
    for loss in (criterions.NLLEntropy(ignore, None)(out, bad), criterions.ClippedPolicyLoss(ignore, None)(out, bad, old, adv)[0],
                 criterions.NLLEntropy(ignore, None)(D.DeferredLogProbs(hid, w, b, 1.0), bad),
                 criterions.ClippedPolicyLoss(ignore, None)(D.DeferredLogProbs(hid, w, b, 1.0), bad, old, torch.zeros(B, device=dev))[0],
                 criterions.PreferenceLoss(ignore, None)(D.DeferredLogProbs(hid, w, b, 1.0), bad, D.DeferredLogProbs(hid, w, b, 1.0), y)[0]):
        assert bool(torch.isnan(loss))
    if frozen:
        return
    up = torch.randn(B, L, generator=gen, device=dev)
    up[0, 0] = 0.0                                               # nothing asked of a live row
    gh, gw, gb = torch.autograd.grad((got * up)[~hit].sum() + got[hit].sum(), xs)
    wh, _, _ = torch.autograd.grad((want * up)[~hit].sum() + want[hit].sum(), xs)
    assert torch.equal(torch.isnan(gh).any(-1), hit) and torch.isnan(gh).all(-1)[hit].all()
    assert torch.equal(gh[~hit], wh[~hit])
    assert bool(torch.isnan(gw).all()) and bool(torch.isnan(gb).all())
    sums = D.DeferredLogProbs(hid, w, b, 1.0)                    # the sum alone, as a training step asks for it
    gh, gw, gb = torch.autograd.grad(criterions.NLLEntropy(ignore, None)(sums, bad), xs)
    assert torch.equal(torch.isnan(gh).all(-1), hit) and torch.equal(torch.isnan(gh).any(-1), hit) and bool(torch.isnan(gw).all())


@pytest.mark.parametrize("H,V", PATHS)
def test_nothing_of_a_bad_batch_stays(dev, H, V):
    """The NaN of one batch's gradients does not reach the next batch's through a workspace."""
    from pevae_amd import criterions
    from pevae_amd.enc2dec import decoders as D
    gen = torch.Generator(device=dev).manual_seed(33)
    B, L = 9, 29
    xs = [(torch.randn(*s, generator=gen, device=dev) * 0.3).requires_grad_() for s in ((B, L, H), (V, H), (V,))]
    y = torch.randint(1, V, (B, L), generator=gen, device=dev)
    bad = y.clone()
    bad[:, 4], y[:, 7:11] = V + 3, 0
    old, adv = torch.randn(B, L, generator=gen, device=dev) - 7, torch.randn(B, generator=gen, device=dev)

    def grads(labels):
        out = D.DeferredLogProbs(*xs, 1.0)
        loss = criterions.NLLEntropy(0, None)(out, labels) + criterions.ClippedPolicyLoss(0, None)(out, labels, old, adv)[0]
        more = criterions.ClippedPolicyLoss(0, None, ent_coef=0.1)(out, labels, old, adv)[0]
        return torch.autograd.grad(loss, xs) + torch.autograd.grad(more, xs)

    want = grads(y)
    assert all(bool(torch.isnan(g).any()) for g in grads(bad))
    assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(grads(y), want))


@pytest.mark.parametrize("loss", ["distill", "explore", "dense"])
@pytest.mark.parametrize("order", [(0, 1), (1, 0), (1, 0, 1), (0, 1, 0)])
def test_several_decoder_passes_in_one_backward_pass(dev, loss, order):
    """A loss whose weight gradient is a product of its own, on one decoder output, and the NLL, which accumulates into the same
    gradient beside the recurrences, on others, in every order: the sum of the gradients of each alone.  Each output's share is
    computed as it is alone; what is left are the roundings of the fp32 additions, at most one of 2^-24 of the partial sum for
    each of the V + B L terms of an element: 1e-4 of the largest is granted an output."""
    from pevae_amd import criterions
    from pevae_amd.dls_vae import DLSVAE
    from pevae_amd.enc2dec import decoders as D
    B, L, H, V = 8, 12, 512, 5003
    dec = decoder(dev, H, V, L)
    ids, y, h0, adv = answers(dev, B, L, V)
    h0 = (h0 * 0.3).expand(1, B, H).contiguous().requires_grad_()
    t = torch.randn(B, L, V, device=dev).topk(8, -1)
    with torch.no_grad():
        old = criterions.token_log_probs(dec(B, ids, h0, mode=D.TEACH_FORCE)[0], y, 0) - 0.1
    one = {"distill": lambda o: criterions.TopKDistill(0, None)(o, y, t.indices, t.values),
           "explore": lambda o: criterions.ClippedPolicyLoss(0, None, ent_coef=0.1)(o, y, old, adv)[0],
           "dense": lambda o: criterions.TopKDistill(0, None)(o.materialize(), y, t.indices, t.values)}[loss]
    other = lambda o: criterions.NLLEntropy(0, None)(o, y)
    params = list(dec.parameters()) + [h0]

    def grads(chosen):
        for p in params:
            p.grad = torch.zeros_like(p)
        terms = [f(dec(B, ids, h0, mode=D.TEACH_FORCE)[0]) for f in chosen]
        DLSVAE._run_backward(lambda: torch.autograd.backward(terms))
        return [p.grad.clone() for p in params]

    alone = [grads([one]), grads([other])]
    for _ in range(3):
        for p, got, *each in zip(params, grads([(one, other)[k] for k in order]), *[alone[k] for k in order]):
            top = max(float(e.abs().max()) for e in each)
            assert float((got - sum(each)).abs().max()) <= 1e-4 * len(each) * top


def test_empty_projections(dev):
    """Without a row every operand has a zero gradient, whichever of them asks."""
    from pevae_amd import ops
    V, H = 9, 16
    w, b = torch.randn(V, H, device=dev), torch.randn(V, device=dev)
    for shape in ((0, 4, H), (4, 0, H)):
        y = torch.zeros(shape[:2], dtype=torch.int64, device=dev)
        f = torch.zeros(shape[:2], device=dev)
        for asks in ((True, True, True), (False, True, True), (False, False, True), (True, False, False)):
            xs = [x.detach().clone().requires_grad_(a) for x, a in zip((torch.zeros(shape, device=dev), w, b), asks)]
            for loss in (ops.projected_distill_topk(*xs, y[..., None], f[..., None]), ops.projected_policy_loss(*xs, y, f, f)[0]):
                assert float(loss) == 0.0
                wanted = [x for x in xs if x.requires_grad]
                for x, g in zip(wanted, torch.autograd.grad(loss, wanted)):
                    assert g.shape == x.shape and int(torch.count_nonzero(g)) == 0


def test_policy_loss_behind_the_tile_kernels_captured(dev):
    """Forward and backward of a policy step at a hidden size of the tile kernels, replayed with eager work and changed inputs and
    labels between: the live rows, and with them the tiles that are skipped, differ from replay to replay."""
    from pevae_amd import criterions
    from pevae_amd.enc2dec import decoders as D
    B, L, H, V = 40, 7, 64, 1003
    gen = torch.Generator(device=dev).manual_seed(50)
    params = [torch.randn(*s, generator=gen, device=dev) * 0.3 for s in ((B, L, H), (V, H), (V,))]
    y0 = torch.randint(1, V, (B, L), generator=gen, device=dev)
    old, adv = torch.randn(B, L, generator=gen, device=dev) - 7, torch.randn(B, generator=gen, device=dev)
    policy = criterions.ClippedPolicyLoss(0, None)

    def step(xs, y):
        loss, stats = policy(D.DeferredLogProbs(*xs, 1.0), y, old, adv)
        return [loss.detach(), stats] + list(torch.autograd.grad(loss, xs))

    held, y = [x.clone().requires_grad_() for x in params], y0.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(held, y)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(held, y)
    for turn in range(5):
        keep = torch.rand(B, L, generator=gen, device=dev) < (0.9, 0.1, 0.5, 0.02, 1.0)[turn]
        with torch.no_grad():
            y.copy_(torch.where(keep, y0, torch.zeros_like(y0)))
            for x, v in zip(held, params):
                x.copy_(v * (1.0 + 0.1 * turn))
        want = step([(v * (1.0 + 0.1 * turn)).requires_grad_() for v in params], y.clone())
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn


@pytest.mark.parametrize("cell", ["gru", "lstm"])
@pytest.mark.parametrize("B,H", [(5, 48), (7, 64), (16, 80)])
def test_decoder_step_with_padded_states_captured(dev, cell, B, H):
    """A policy step through the decoder, batch and hidden sizes that the recurrence pads, replayed with eager work and changed
    weights, inputs and labels between."""
    import copy
    from pevae_amd import criterions
    from pevae_amd.enc2dec import decoders as D
    torch.manual_seed(9)
    L, E, V = 7, 24, 211
    held = D.DecoderRNN(V, L, E, H, 1, 2, 3, rnn_cell=cell, embedding=torch.nn.Embedding(V, E, padding_idx=0)).to(dev)
    eager = copy.deepcopy(held)
    ids, y, _, adv = answers(dev, B, L, V)
    state = torch.randn(2, 1, B, H, device=dev) * 0.3
    old = torch.randn(B, L, device=dev) - 5
    policy = criterions.ClippedPolicyLoss(0, None)

    def step(dec):
        h0 = (state[0], state[1]) if cell == "lstm" else state[0]
        loss, stats = policy(dec(B, ids, h0, mode=D.TEACH_FORCE)[0], y, old, adv)
        return [loss.detach(), stats] + list(torch.autograd.grad(loss, list(dec.parameters())))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(held)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(held)
    for turn in range(5):
        gen = torch.Generator(device=dev).manual_seed(60 + turn)
        with torch.no_grad():
            ids.copy_(torch.randint(4, V, (B, L), generator=gen, device=dev))
            y[:, :-1] = ids[:, 1:]
            y[1, turn:] = 0
            state.copy_(torch.randn(2, 1, B, H, generator=gen, device=dev) * 0.3)
            for p, q in zip(held.parameters(), eager.parameters()):
                q.mul_(1.05)
                p.copy_(q)
        want = step(eager)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn


@pytest.mark.parametrize("H,V", PATHS)
def test_the_first_ratio_is_one(dev, H, V):
    """Scores made under no_grad are, bit for bit, the log-probabilities that the loss computes: the ratio of the first on-policy
    step is 1, and its gradient that of minus the advantage times the log-probability."""
    from pevae_amd import criterions, ops
    from pevae_amd.enc2dec import decoders as D
    B, L = 5, 6
    dec = decoder(dev, H, V)
    ids, y, h0, adv = answers(dev, B, L, V)
    out = dec(B, ids, (h0 * 0.3).expand(1, B, H).contiguous(), mode=D.TEACH_FORCE)[0]
    with torch.no_grad():
        old = criterions.token_log_probs(out, y, 0)
    lp = criterions.token_log_probs(out, y, 0)
    assert lp.requires_grad and torch.equal(lp, old)
    loss, stats = criterions.ClippedPolicyLoss(0, None, avg_type=None)(out, y, old, adv)
    live = (y != 0).double()
    assert abs(float(loss) + float((live * adv.double()[:, None]).sum())) <= 2.0 ** -24 * float((live * adv.double().abs()[:, None]).sum())
    d, = torch.autograd.grad(ops.policy_loss(lp, y, old, adv, ignore_index=0, avg_type=None)[0], lp)
    assert torch.equal(d, torch.where(y != 0, -adv[:, None].expand(B, L), torch.zeros(B, L, device=dev)))
    assert float(stats[2]) == 0.0
