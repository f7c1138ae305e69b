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
