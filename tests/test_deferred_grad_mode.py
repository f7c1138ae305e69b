"""What a decoder's DeferredLogProbs keeps between calls, without a GPU: a result made under torch.no_grad() has no history and
must not be handed to a caller that asks for one.  The kernels' nodes are replaced by torch's own operations."""
import pytest
import torch

from pevae_amd import ops
from pevae_amd.enc2dec.decoders import DeferredLogProbs

B, L, H, V = 2, 3, 4, 7


class PlainNLL(object):
    RETURNED_SUMS = False
    calls = 0

    @classmethod
    def apply(cls, hid, w, b, target, inv_temp, ignore, hid_bf16, layout, drop, pre, sums_only):
        cls.calls += 1
        lp = torch.log_softmax((hid @ w.t() + b) * inv_temp, -1)
        nll = -lp.gather(-1, target[:, None])[:, 0]
        return torch.where(target != ignore, nll, torch.zeros_like(nll)), None


class PlainSum(object):
    @staticmethod
    def apply(x, tgt, ignore):
        return torch.stack([x.sum(), (tgt != ignore).sum().to(x.dtype)])


class PlainHead(object):
    @staticmethod
    def apply(sums, batch):
        return sums[0] / batch, torch.exp(sums[0] / sums[1])


class PlainDense(object):
    calls = 0

    @classmethod
    def apply(cls, hid, w, b, inv_temp):
        cls.calls += 1
        return torch.log_softmax((hid @ w.t() + b) * inv_temp, -1)


@pytest.fixture
def deferred(monkeypatch):
    for name, plain in (("VocabNLL", PlainNLL), ("MaskedSum", PlainSum), ("NllHead", PlainHead), ("VocabLogProbDense", PlainDense)):
        monkeypatch.setattr(ops, name, plain)
    PlainNLL.calls = PlainDense.calls = 0
    gen = torch.Generator().manual_seed(5)
    hid, w, b = (torch.randn(*s, generator=gen, dtype=torch.float64).requires_grad_() for s in ((B, L, H), (V, H), (V,)))
    y = torch.tensor([[1, 3, 0], [6, 0, 0]])
    return DeferredLogProbs(hid, w, b, 1.0), y


ASKS = [lambda o, y: o.token_nll(y, 0)[0].sum(), lambda o, y: o.token_nll_sums(y, 0)[0], lambda o, y: o.loss_head(y, 0)[0],
        lambda o, y: o.materialize().square().sum()]


@pytest.mark.parametrize("first", range(4))
@pytest.mark.parametrize("then", range(4))
def test_nothing_without_history_is_handed_out_for_training(deferred, first, then):
    out, y = deferred
    with torch.no_grad():
        assert not ASKS[first](out, y).requires_grad
    loss = ASKS[then](out, y)
    got = torch.autograd.grad(loss, [out.hid, out.weight, out.bias])
    fresh = DeferredLogProbs(out.hid, out.weight, out.bias, 1.0)
    want = torch.autograd.grad(ASKS[then](fresh, y), [out.hid, out.weight, out.bias])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_results_with_history_serve_both(deferred):
    out, y = deferred
    a = out.token_nll(y, 0)[0]
    dense = out.materialize()
    with torch.no_grad():
        assert out.token_nll(y, 0)[0] is a and out.materialize() is dense
        out.loss_head(y, 0)
    assert out.token_nll(y, 0)[0] is a and out.materialize() is dense
    assert (PlainNLL.calls, PlainDense.calls) == (1, 1)


def test_scores_are_computed_once_in_each_mode(deferred):
    out, y = deferred
    for _ in range(2):
        with torch.no_grad():
            out.token_nll(y, 0), out.materialize()
    assert (PlainNLL.calls, PlainDense.calls) == (1, 1)
    for _ in range(2):
        out.token_nll(y, 0), out.materialize()
    with torch.no_grad():
        out.token_nll(y, 0), out.materialize()
    assert (PlainNLL.calls, PlainDense.calls) == (2, 2)


def test_one_copy_is_held_once_training_asks(deferred):
    """A result with a history takes the place of the one without: dense rows are not held twice."""
    out, y = deferred
    with torch.no_grad():
        scored = out.materialize()
    trained = out.materialize()
    dense = [t for t in out._nll_cache.values() if torch.is_tensor(t) and t.shape == scored.shape]
    assert len(dense) == 1 and dense[0] is trained and out._dense is trained and trained is not scored
