"""Losses over rows of a vocabulary softmax in memory, on the GPU, against their definitions in 64 bits.

Tolerances, derived from the arithmetic (u = 2^-24 is half a step of fp32, relative):
 * an exponential e = 2^x: x carries three roundings of |x| <= 40 (difference, product, the constant) and 2^x one step, so its
   relative error is at most 40 * 0.69 * 3 u + 2 u < 6e-6; weighted by the probabilities |x| is at most about 12, and a sum of
   up to 131071 of them adds about 40 roundings a thread and in the trees: ln s is off by at most 5e-6 absolute;
 * a log-probability: 5e-6 + u |value|; an entropy: the same plus 6e-6 of it -> EXP = 1e-5 absolute and relative covers both;
 * a gradient element: EXP of the sum of its terms' magnitudes (they may cancel), then ONE rounding to the logits' type, at
   most finfo.eps / 2 relative, or half of the smallest subnormal;
 * ratios and divergences of the policy loss multiply the error of a log-probability by the ratio: EXP of their magnitudes;
 * sums over rows run in fp64: EXP of the sum of magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EXP = 1e-5
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from pevae_amd import ops
    assert "gfx950" in ops.device_info()["arch"]
    return torch.device("cuda:0")


def close(got, want, mag, what=""):
    """|got - want| <= EXP * mag + the rounding of got's type; infinities and NaN have to be where they are in want."""
    got_, want = got.detach().double(), want.double()
    mag = torch.as_tensor(mag, dtype=torch.float64, device=want.device).expand(want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got_), torch.isnan(want)), what + ": NaN"
    inf = torch.isinf(want)
    assert torch.equal(got_[inf], want[inf]), what + ": infinities"
    info = torch.finfo(got.dtype)
    tol = EXP * mag[fin] + info.eps / 2 * want[fin].abs() * (1 + EXP) + info.smallest_normal * info.eps / 2
    over = (got_[fin] - want[fin]).abs() / tol
    assert over.numel() == 0 or float(over.max()) <= 1.0, "%s: %.3g of the tolerance" % (what, float(over.max()))


def softmax64(logits, c):
    z = logits.detach().double() * c
    m = z.max(-1, keepdim=True).values
    e = torch.exp(z - m)
    s = e.sum(-1, keepdim=True)
    return e / s, z - m - torch.log(s)


def plogp(p, lq):
    return torch.where(p > 0, p * lq, torch.zeros_like(p))


def rows_grad64(p, lq, H, y, g, h, c):
    """(gradient, magnitude) of the logits for upstream g of log p[y] and h of the entropy; y < 0: no label."""
    hot = torch.zeros_like(p)
    on = y >= 0
    hot.scatter_(-1, y.clamp(min=0)[..., None], on.double()[..., None])
    g, h = g[..., None], h[..., None]
    d = c * (g * (hot - p) - h * (plogp(p, lq) + p * H[..., None]))
    mag = c * (g.abs() * (hot + p) + h.abs() * (plogp(p, lq).abs() + p * H[..., None].abs()) * 4)
    return d, mag


def make(shape, dtype, dev, seed, spread=3.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=dev) * spread).to(dtype)


def labels_of(shape, V, dev, seed, dead=0.3):
    gen = torch.Generator(device=dev).manual_seed(seed)
    y = torch.randint(0, V, shape, generator=gen, device=dev)
    return torch.where(torch.rand(*shape, generator=gen, device=dev) < dead, torch.full_like(y, -7), y)


SHAPES = [(1, 1, 1), (1, 1, 2), (2, 3, 7), (2, 3, 8), (3, 2, 63), (2, 5, 1000), (1, 4, 1009), (2, 2, 4097), (3, 3, 8192),
          (1, 3, 8195), (2, 2, 20004), (1, 2, 33333), (1, 2, 65537), (1, 2, 131071), (300, 1, 129), (1, 1, 200003)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_token_logprobs(dev, dtype, shape):
    from pevae_amd import ops
    B, L, V = shape
    z = make(shape, dtype, dev, 1).requires_grad_()
    y = labels_of((B, L), V, dev, 2)
    c = 1.0 / 0.7
    live = y != -7
    p, lq = softmax64(z, c)
    H = -plogp(p, lq).sum(-1)
    lp = lq.gather(-1, y.clamp(min=0)[..., None])[..., 0]
    zero = torch.zeros_like(lp)
    want_lp, want_H = torch.where(live, lp, zero), torch.where(live, H, zero)
    g, h = make((B, L), torch.float32, dev, 3), make((B, L), torch.float32, dev, 4)
    got_lp, got_H = ops.token_logprobs(z, y, ignore_index=-7, inv_temp=c, entropy=True)
    close(got_lp, want_lp, 1 + want_lp.abs(), "logp")
    close(got_H, want_H, 1 + want_H.abs(), "entropy")
    with torch.no_grad():
        only = ops.token_logprobs(z, y, ignore_index=-7, inv_temp=c)
    assert not only.requires_grad
    close(only, want_lp, 1 + want_lp.abs(), "logp alone")
    yl = torch.where(live, y, torch.full_like(y, -1))
    gl, hl = torch.where(live, g.double(), zero), torch.where(live, h.double(), zero)
    for take_g, take_h in ((1, 1), (1, 0), (0, 1)):
        outs = [t for t, on in ((got_lp, take_g), (got_H, take_h)) if on]
        ups = [t for t, on in ((g, take_g), (h, take_h)) if on]
        d, = torch.autograd.grad(outs, [z], ups, retain_graph=True)
        want, mag = rows_grad64(p, lq, H, yl, gl * take_g, hl * take_h, c)
        assert d.dtype == dtype and d.shape == z.shape
        close(d, want, mag, "dlogits %d%d" % (take_g, take_h))


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_words(dev, dtype):
    """-inf and the type's lowest value in masked words; a row that they fill; NaN in a dead row and in a live one."""
    from pevae_amd import ops
    V, low = 1003, torch.finfo(dtype).min
    z = make((7, V), dtype, dev, 5)
    z[0, ::2] = float("-inf")
    z[1, ::2] = low
    z[2] = low                              # every word masked with the lowest value: uniform
    z[3, :] = float("-inf")
    z[3, 17] = 1.5                          # one word left
    z[4] = float("nan")                     # dead
    z[5] = float("-inf")                    # nothing left: no distribution
    z[6, 3] = float("nan")
    z = z.requires_grad_()
    y = torch.tensor([1, 3, 5, 17, 0, 2, 9], device=dev)
    got, ent = ops.token_logprobs(z, y, ignore_index=0, entropy=True)
    p, lq = softmax64(z, 1.0)
    H = -plogp(p, lq).sum(-1)
    lp = lq.gather(-1, y[:, None])[:, 0]
    for t in (lp, H):
        t[4] = 0.0
        t[5:] = float("nan")
    close(got, lp, 1 + lp.nan_to_num().abs(), "logp")
    close(ent, H, 1 + H.nan_to_num().abs(), "entropy")
    g, h = make((7,), torch.float32, dev, 6), make((7,), torch.float32, dev, 7)
    d, = torch.autograd.grad([got, ent], [z], [g, h])
    want, mag = rows_grad64(p[:4], lq[:4], H[:4], y[:4], g[:4].double(), h[:4].double(), 1.0)
    close(d[:4], want, mag, "dlogits")
    assert float(d[4].abs().max()) == 0.0
    assert bool(torch.isnan(d[5]).all()) and bool(torch.isnan(d[6]).all())
    # the label itself is a masked word: -inf, as log-softmax says
    y2 = torch.tensor([0], device=dev)
    assert float(ops.token_logprobs(z.detach()[:1], y2)) == float("-inf")


def test_tokens_that_name_no_word(dev):
    from pevae_amd import ops
    z = make((5, 99), torch.float32, dev, 8).requires_grad_()
    y = torch.tensor([98, 99, -1, 1 << 40, 0], device=dev)
    got = ops.token_logprobs(z, y, ignore_index=-100)
    assert torch.isnan(got).tolist() == [False, True, True, True, False]
    d, = torch.autograd.grad(got, z, torch.ones_like(got))
    assert torch.isnan(d).all(-1).tolist() == [False, True, True, True, False]
    assert not torch.isnan(d[[0, 4]]).any()
    assert torch.equal(ops.token_logprobs(z, y.clamp(0, 98).int()), ops.token_logprobs(z, y.clamp(0, 98)))      # int32 tokens


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(dev, dtype):
    """The same rows in any layout and at any alignment (which moves the order of the sums)."""
    from pevae_amd import ops
    B, L, V = 3, 5, 1001
    base = make((B, L, V), dtype, dev, 9)
    y = labels_of((B, L), V, dev, 10, dead=0.2)
    up = make((B, L), torch.float32, dev, 11)
    p, lq = softmax64(base, 1.0)
    live = y != -7
    zero = torch.zeros(B, L, dtype=torch.float64, device=dev)
    want = torch.where(live, lq.gather(-1, y.clamp(min=0)[..., None])[..., 0], zero)
    dwant, dmag = rows_grad64(p, lq, zero, torch.where(live, y, torch.full_like(y, -1)), torch.where(live, up.double(), zero), zero, 1.0)

    def check(x, name, pick=lambda t: t):
        x = x.detach().requires_grad_()
        lp = ops.token_logprobs(x, pick(y), ignore_index=-7)
        d, = torch.autograd.grad(lp, x, pick(up))
        assert lp.shape == x.shape[:-1] and d.shape == x.shape
        close(lp, pick(want), 1 + pick(want).abs(), name)
        close(d, pick(dwant).reshape(x.shape), pick(dmag).reshape(x.shape), name + " gradient")

    check(base, "contiguous")
    for start in range(9):
        padded = torch.full((B, L, 1030), float("nan"), dtype=dtype, device=dev)
        padded[..., start:start + V] = base
        check(padded[..., start:start + V], "padded, from %d" % start)
        flat = torch.zeros(B * L * V + start, dtype=dtype, device=dev)
        flat[start:] = base.reshape(-1)
        check(flat[start:].view(B, L, V), "from element %d" % start)
    check(base.transpose(0, 1).contiguous().transpose(0, 1), "time major")
    check(base.permute(2, 0, 1).contiguous().permute(1, 2, 0), "word major")
    check(base.view(B * L, V), "two dimensions", lambda t: t.reshape((B * L,) + t.shape[2:]))
    check(base.view(B, 1, L, 1, V), "five dimensions", lambda t: t.reshape((B, 1, L, 1) + t.shape[2:]))
    check(base[0, 0], "one row", lambda t: t[0, 0])
    # one row shown to all tokens: the gradient of the broadcast input is the sum over them
    one = base[:1, :1].detach().requires_grad_()
    wide = one.expand(B, L, V)
    lp = ops.token_logprobs(wide, y, ignore_index=-7)
    d, = torch.autograd.grad(lp, one, up)
    p, lq = softmax64(wide, 1.0)
    gl = torch.where(y != -7, up, torch.zeros_like(up)).double()
    w, mag = rows_grad64(p, lq, torch.zeros_like(gl), y, gl, torch.zeros_like(gl), 1.0)
    # each of the B * L rows is rounded before the sum: by half a step of its terms, or by half of the smallest subnormal
    info = torch.finfo(dtype)
    rounding = info.eps / 2 * mag.sum((0, 1), keepdim=True) + B * L * info.smallest_normal * info.eps / 2
    close(d, w.sum((0, 1), keepdim=True), mag.sum((0, 1), keepdim=True) + rounding / EXP, "broadcast")


# ------------------------------------------------------------------------------------------------------------
# distillation
# ------------------------------------------------------------------------------------------------------------

def distill64(z, ids, t, live, tau, scale):
    """(loss, its magnitude, gradient, magnitude) by the definition; ids < 0 where the entry does not count."""
    p, lq = softmax64(z, 1.0 / tau)
    empty = torch.isinf(t).all(-1)
    q, lt = softmax64(torch.where(empty[..., None], torch.zeros_like(t), t), 1.0 / tau)
    q = torch.where(torch.isinf(t), torch.zeros_like(q), q)
    term = torch.where(q > 0, q * (lt - lq.gather(-1, ids.clamp(min=0))), torch.zeros_like(q)).sum(-1)
    on = (live & ~empty).double()
    mag = torch.where(q > 0, q * (lt.abs() + lq.gather(-1, ids.clamp(min=0)).abs() + 1), torch.zeros_like(q)).sum(-1)
    target = torch.zeros_like(p).scatter_add_(-1, ids.clamp(min=0), q)
    w = on * tau * scale
    return ((on * term).sum() * tau * tau * scale, (on * mag).sum() * tau * tau * scale, w[..., None] * (p - target),
            w.abs()[..., None] * (p + target))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,K", [((1, 1, 2), 1), ((2, 3, 7), 7), ((2, 3, 1000), 5), ((1, 4, 1009), 64), ((2, 2, 8195), 65),
                                     ((2, 2, 20004), 32), ((1, 2, 65537), 256), ((1, 1, 131071), 100), ((300, 2, 129), 3)])
@pytest.mark.parametrize("avg", ["seq", "word", None])
def test_distill(dev, dtype, shape, K, avg):
    from pevae_amd import ops
    B, L, V = shape
    z = make(shape, dtype, dev, 20).requires_grad_()
    t = (make(shape, torch.float32, dev, 21) + 0.5 * z.detach().float()).topk(K, -1)
    y = labels_of((B, L), V, dev, 22)
    live, tau = y != -7, 1.7
    n = B if avg == "seq" else max(int(live.sum()), 1) if avg == "word" else 1
    tl = t.values.to(dtype)
    loss = ops.distill_topk(z, t.indices, tl, y, -7, tau, 0.75, avg)
    want, mag, dwant, dmag = distill64(z, t.indices, tl, live, tau, 0.75 / n)
    close(loss, want, mag + 1e-30, "loss")
    for up in (None, torch.tensor(3.0, device=dev), None):          # 1, another upstream gradient, 1 again
        d, = torch.autograd.grad(loss, z, up, retain_graph=True)
        k = 1.0 if up is None else 3.0
        close(d, k * dwant, k * dmag, "dlogits %s" % up)
    with torch.no_grad():
        close(ops.distill_topk(z, t.indices, tl, y, -7, tau, 0.75, avg), want, mag + 1e-30, "loss alone")


def test_distill_lists(dev):
    """Short lists padded with -inf whatever their ids are, empty lists, words listed twice, another teacher type, no labels."""
    from pevae_amd import ops
    B, L, V, K = 2, 4, 513, 70
    z = make((B, L, V), torch.bfloat16, dev, 23).requires_grad_()
    gen = torch.Generator(device=dev).manual_seed(24)
    ids = torch.randint(0, V, (B, L, K), generator=gen, device=dev)
    ids[0, 0, 5:9] = ids[0, 0, 4]                   # a word five times
    ids[0, 1] = 7                                   # only one word
    ids[1, 3, 69] = ids[1, 3, 0]
    t = make((B, L, K), torch.float32, dev, 25)
    t[0, 2, 3:] = float("-inf")
    t[1, 0] = float("-inf")                         # nothing left: dead
    t[1, 1, 1:] = float("-inf")
    ids = torch.where(torch.isinf(t), torch.full_like(ids, -1), ids)
    ids[0, 2, 10], ids[0, 2, 11], ids[0, 2, 12] = V, 1 << 40, -(1 << 50)
    safe = torch.where((ids < 0) | (ids >= V), torch.full_like(ids, -1), ids)
    live = torch.ones(B, L, dtype=torch.bool, device=dev)
    for dt in TYPES:
        tl = t.to(dt)
        loss = ops.distill_topk(z, ids, tl, avg_type="word")
        want, mag, dwant, dmag = distill64(z, safe, tl, live, 1.0, 1.0 / (B * L))
        close(loss, want, mag, "loss")
        d, = torch.autograd.grad(loss, z)
        close(d, dwant, dmag, "dlogits")
        assert float(d[1, 0].abs().max()) == 0.0
    # an entry that counts and names no word
    ids[1, 2, 0] = V
    loss = ops.distill_topk(z, ids, t)
    d, = torch.autograd.grad(loss, z)
    assert bool(torch.isnan(loss)) and torch.isnan(d).all(-1).sum() == 1 and bool(torch.isnan(d[1, 2]).all())
    # the teacher's word is masked in the student: infinite loss
    z2 = z.detach().clone()
    z2[0, 0, ids[0, 0, 0]] = float("-inf")
    assert float(ops.distill_topk(z2[:1, :1], ids[:1, :1], t[:1, :1])) == float("inf")
    # a NaN among the teacher's logits
    t[0, 3, 66] = float("nan")
    assert bool(torch.isnan(ops.distill_topk(z[:1], ids[:1], t[:1])))


@pytest.mark.parametrize("K", [2, 16, 17, 33, 64, 65, 130, 256])
def test_distill_words_listed_twice(dev, K):
    """A word at two places of a list, a pair of places a row (all pairs up to 64 entries), and one row without such a word."""
    from pevae_amd import ops
    V = 300
    i, j = torch.triu_indices(K, K, 1, device=dev)
    if K > 64:
        pick = torch.randperm(i.numel(), generator=torch.Generator(device=dev).manual_seed(28), device=dev)[:2000]
        i, j = i[pick], j[pick]
    T = i.numel() + 1
    ids = torch.rand(T, V, generator=torch.Generator(device=dev).manual_seed(29), device=dev).topk(K, -1).indices
    rows = torch.arange(T - 1, device=dev)
    ids[rows, i] = ids[rows, j]
    z = make((T, V), torch.float32, dev, 26).requires_grad_()
    t = make((T, K), torch.float32, dev, 27)
    loss = ops.distill_topk(z, ids, t, avg_type=None)
    want, mag, dwant, dmag = distill64(z, ids, t, torch.ones(T, dtype=torch.bool, device=dev), 1.0, 1.0)
    close(loss, want, mag, "loss")
    for up in (None, torch.tensor(3.0, device=dev)):
        k = 1.0 if up is None else 3.0
        close(torch.autograd.grad(loss, z, up, retain_graph=True)[0], k * dwant, k * dmag, "dlogits")


# ------------------------------------------------------------------------------------------------------------
# policy
# ------------------------------------------------------------------------------------------------------------

def policy64(lp, old, ref, adv, live, lo, hi, kl):
    """per token: policy term, KL term, clipped, slope by lp, and the slope's magnitude."""
    r = torch.exp(lp - old)
    A = adv if adv.shape == lp.shape else adv[:, None].expand_as(lp)
    u, w = r * A, torch.clamp(r, lo, hi) * A
    u, w = torch.where(A == 0, torch.zeros_like(u), u), torch.where(A == 0, torch.zeros_like(w), w)
    cut = u > w
    pg = -torch.where(cut, w, u)
    slope, mag = torch.where(cut, torch.zeros_like(u), -u), torch.where(cut, torch.zeros_like(u), u.abs())
    k3 = torch.zeros_like(pg)
    if ref is not None:
        d = ref - lp
        k3 = torch.expm1(d) - d
        slope, mag = slope - kl * torch.expm1(d), mag + kl * (1 + torch.exp(d))
    zero = torch.zeros_like(pg)
    return [torch.where(live, t, zero) for t in (pg, k3, cut.double(), slope, mag)]


def policy_inputs(lp, dev, seed):
    """old log-probabilities whose ratios keep 1e-3 away from the borders of the clip range, a reference model's, advantages."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    step = torch.randint(0, 8, lp.shape, generator=gen, device=dev)
    off = torch.tensor([-0.6, -0.3, -0.1, 0.0, 0.05, 0.15, 0.3, 0.7], device=dev)[step]
    old = lp.float() - off
    ref = lp.float() + 0.4 * torch.randn(lp.shape, generator=gen, device=dev)
    ref = torch.where(step == 3, lp.float(), ref)
    return old, ref, torch.randn(lp.shape, generator=gen, device=dev)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 2), (2, 3, 7), (2, 5, 1000), (1, 4, 1009), (2, 3, 8195), (2, 2, 20004), (1, 2, 65537),
                                   (1, 1, 131071), (130, 2, 129)])
@pytest.mark.parametrize("avg,kl,ent,per_token", [("word", 0.05, 0.0, False), ("seq", 0.3, 0.02, True), (None, 0.0, 0.5, False)])
def test_vocab_policy_loss(dev, dtype, shape, avg, kl, ent, per_token):
    from pevae_amd import ops
    B, L, V = shape
    z = make(shape, dtype, dev, 30).requires_grad_()
    y = labels_of((B, L), V, dev, 31)
    live = y != -7
    c = 1.0 / 1.3
    p, lq = softmax64(z, c)
    H = -plogp(p, lq).sum(-1)
    lp = lq.gather(-1, y.clamp(min=0)[..., None])[..., 0]
    old, ref, adv = policy_inputs(lp, dev, 32)
    nan = torch.full_like(old, float("nan"))
    old, ref = torch.where(live, old, nan), torch.where(live, ref, nan)         # dead entries are not read
    if not per_token:
        adv = adv[:, 0].contiguous()
    r = ref if kl else None
    loss, stats = ops.vocab_policy_loss(z, y, old, adv, r, -7, c, 0.2, 0.28, kl, ent, 1.5, avg)
    pg, k3, cut, slope, smag = policy64(lp, old.double(), None if r is None else r.double(), adv.double(), live, 0.8, 1.28, kl)
    n = B if avg == "seq" else max(int(live.sum()), 1) if avg == "word" else 1
    on, count = live.double(), max(int(live.sum()), 1)
    row_mag = on * (pg.abs() + smag + kl * k3 + ent * (1 + H))
    close(loss, 1.5 / n * (pg + kl * k3 - ent * H * on).sum(), 1.5 / n * row_mag.sum() + 1e-30, "loss")
    close(stats, torch.stack([pg.sum(), k3.sum(), cut.sum(), (H * on).sum()]) / count,
          torch.stack([(pg.abs() + smag).sum(), (k3 + on * (1 if kl == 0 else smag / max(kl, 1e-9))).sum(), on.sum(),
                       ((1 + H) * on).sum()]) / count + 1e-30, "stats")
    assert not stats.requires_grad
    yl = torch.where(live, y, torch.full_like(y, -1))
    dwant, _ = rows_grad64(p, lq, H, yl, 1.5 / n * slope, -1.5 / n * ent * on, c)
    _, dmag = rows_grad64(p, lq, H, yl, 1.5 / n * 3 * smag, -1.5 / n * ent * on, c)
    for up in (None, torch.tensor(-0.5, device=dev), None):
        d, = torch.autograd.grad(loss, z, up, retain_graph=True)
        k = 1.0 if up is None else -0.5
        close(d, k * dwant, dmag, "dlogits %s" % up)


@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (256, 50), (7, 1023), (1, 5000), (700, 401), (9,)])
@pytest.mark.parametrize("avg,kl,per_token", [("word", 0.05, False), ("seq", 0.0, True), (None, 0.3, False)])
def test_policy_loss_from_log_probabilities(dev, shape, avg, kl, per_token):
    from pevae_amd import ops
    y = labels_of(shape, 1000, dev, 40)
    live = y != -7
    lp = -4 * torch.rand(*shape, device=dev, generator=torch.Generator(device=dev).manual_seed(41))
    old, ref, adv = policy_inputs(lp, dev, 42)
    if not per_token and len(shape) == 2:
        adv = adv[:, 0].contiguous()
    adv.view(-1)[0] = 0.0
    lp = torch.where(live, lp, torch.full_like(lp, float("nan"))).requires_grad_()
    r = ref if kl else None
    loss, stats = ops.policy_loss(lp, y, old, adv, r, -7, 0.2, 0.28, kl, 2.0, avg)
    x = lp.detach().double().nan_to_num()
    pg, k3, cut, slope, mag = policy64(x, old.double(), None if r is None else r.double(), adv.double(), live, 0.8, 1.28, kl)
    n = shape[0] if avg == "seq" else max(int(live.sum()), 1) if avg == "word" else 1
    count = max(int(live.sum()), 1)
    close(loss, 2.0 / n * (pg + kl * k3).sum(), 2.0 / n * (pg.abs() + mag).sum() + 1e-30, "loss")
    close(stats, torch.stack([pg.sum(), k3.sum(), cut.sum(), 0 * pg.sum()]) / count,
          torch.stack([(pg.abs() + mag).sum(), k3.sum() + 1e-3 * count, cut.sum(), 0 * pg.sum()]) / count + 1e-30, "stats")
    d, = torch.autograd.grad(loss, lp, torch.tensor(0.5, device=dev), retain_graph=True)
    close(d, slope / n, mag / n, "dlogp")
    d2, = torch.autograd.grad(loss, lp)
    close(d2, 2 * slope / n, 2 * mag / n, "dlogp again")


def test_policy_edges(dev):
    """A zero advantage with a ratio that overflows; a batch without a live token; an old log-probability of -inf."""
    from pevae_amd import ops
    lp = torch.tensor([[-1.0, -2.0], [-3.0, -0.5]], device=dev).requires_grad_()
    old = torch.tensor([[float("-inf"), -2.0], [-200.0, -0.5]], device=dev)
    y = torch.ones(2, 2, dtype=torch.int64, device=dev)
    loss, stats = ops.policy_loss(lp, y, old, torch.tensor([0.0, 0.0], device=dev))
    d, = torch.autograd.grad(loss, lp)
    assert loss.item() == 0.0 and float(d.abs().max()) == 0.0 and stats.tolist() == [0.0] * 4
    # negative advantage and a huge ratio: not clipped, infinite
    loss, _ = ops.policy_loss(lp, y, old, torch.tensor([-1.0, 0.0], device=dev), avg_type=None)
    assert float(loss) == float("inf")
    # positive advantage: clipped at 1.2
    loss, _ = ops.policy_loss(lp, y, old, torch.tensor([1.0, 0.0], device=dev), avg_type=None)
    assert abs(float(loss) + 2.2) < 1e-6
    for avg in ("word", "seq", None):
        z = make((2, 2, 50), torch.float32, dev, 43).requires_grad_()
        loss, stats = ops.vocab_policy_loss(z, torch.zeros_like(y), old, torch.ones(2, device=dev), ignore_index=0, avg_type=avg)
        d, = torch.autograd.grad(loss, z)
        assert float(loss) == 0.0 and stats.tolist() == [0.0] * 4 and float(d.abs().max()) == 0.0
        loss = ops.distill_topk(z, torch.zeros(2, 2, 3, dtype=torch.int64, device=dev), torch.zeros(2, 2, 3, device=dev),
                                torch.zeros_like(y), 0, avg_type=avg)
        d, = torch.autograd.grad(loss, z)
        assert float(loss) == 0.0 and float(d.abs().max()) == 0.0


def test_policy_reports_a_far_reference(dev):
    """A KL coefficient of 0 with a reference model: the term is reported (exp(190) is beyond fp32) and does not enter."""
    from pevae_amd import ops
    z = make((2, 3, 50), torch.float32, dev, 44).requires_grad_()
    y = labels_of((2, 3), 50, dev, 45, 0.0)
    old = ops.token_logprobs(z, y).detach() - 0.1
    ref, adv = old.clone(), torch.tensor([1.0, -0.5], device=dev)
    ref[0, 1] += 190.0
    lp = ops.token_logprobs(z, y)
    for with_ref, without in ((ops.vocab_policy_loss(z, y, old, adv, ref), ops.vocab_policy_loss(z, y, old, adv)),
                              (ops.policy_loss(lp, y, old, adv, ref), ops.policy_loss(lp, y, old, adv))):
        assert float(with_ref[0]) == float(without[0]) and float(with_ref[1][1]) == float("inf")
        a, = torch.autograd.grad(with_ref[0], z, retain_graph=True)
        b, = torch.autograd.grad(without[0], z, retain_graph=True)
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------------------
# preference
# ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("P,Lc,Lr", [(1, 1, 1), (3, 5, 7), (128, 50, 43), (2, 2000, 1), (300, 1, 513), (4, 0, 3)])
@pytest.mark.parametrize("smooth,with_ref,avg", [(0.0, True, "seq"), (0.1, True, None), (0.3, False, "seq")])
def test_preference_loss(dev, P, Lc, Lr, smooth, with_ref, avg):
    from pevae_amd import ops
    gen = torch.Generator(device=dev).manual_seed(50)
    data = []
    for L, seed in ((Lc, 51), (Lr, 52)):
        y = labels_of((P, L), 100, dev, seed)
        if L:
            y[0] = -7                                # an answer without a live token
        lp, ref = (-5 * torch.rand(P, L, generator=gen, device=dev) for _ in range(2))
        dead = y == -7
        lp = torch.where(dead, torch.full_like(lp, float("nan")), lp).requires_grad_()
        data.append((y, lp, torch.where(dead, torch.full_like(ref, float("nan")), ref) if with_ref else None))
    (yc, lc, rc), (yr, lr, rr) = data
    beta = 0.1
    loss, got_c, got_r = ops.preference_loss(lc, yc, lr, yr, rc, rr, -7, beta, smooth, 2.0, avg)

    def total(y, lp, ref):
        d = lp.detach().double() - (0 if ref is None else ref.double())
        d = torch.where(y != -7, d, torch.zeros_like(d))
        return beta * d.sum(1), beta * (d.abs()).sum(1)

    (wc, mc), (wr, mr) = total(yc, lc, rc), total(yr, lr, rr)
    # fp64 sums, times beta as fp32 holds it (off by at most u = 6e-8 of its value: EXP * 6e-3), rounded to fp32 once
    close(got_c, wc, 6e-3 * mc, "chosen")
    close(got_r, wr, 6e-3 * mr, "rejected")
    x = wc - wr
    n = P if avg == "seq" else 1
    rows = -(1 - smooth) * torch.nn.functional.logsigmoid(x) - smooth * torch.nn.functional.logsigmoid(-x)
    # x is rounded to fp32 once: the loss moves by at most that much, plus its own few roundings
    close(loss, 2.0 / n * rows.sum(), 2.0 / n * (rows.abs() + x.abs() + 0.1).sum(), "loss")
    slope = 2.0 / n * beta * (smooth * torch.sigmoid(x) - (1 - smooth) * torch.sigmoid(-x))
    mag = 2.0 / n * beta * (smooth * torch.sigmoid(x) + (1 - smooth) * torch.sigmoid(-x)) * (1 + x.abs())
    dc, dr = torch.autograd.grad(loss, [lc, lr], torch.tensor(-3.0, device=dev))
    close(dc, -3 * slope[:, None] * (yc != -7), 3 * mag[:, None] * (yc != -7), "chosen gradient")
    close(dr, 3 * slope[:, None] * (yr != -7), 3 * mag[:, None] * (yr != -7), "rejected gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P,Lc,Lr,V", [(1, 1, 1, 7), (3, 4, 2, 1009), (2, 3, 5, 20003), (5, 2, 3, 260), (2, 0, 3, 50)])
@pytest.mark.parametrize("smooth,with_ref,avg", [(0.0, True, "seq"), (0.2, False, None)])
def test_vocab_preference_loss(dev, dtype, P, Lc, Lr, V, smooth, with_ref, avg):
    """From the logits: the log-probabilities' errors (5e-6 a token, see above) add up in the rewards."""
    from pevae_amd import ops
    beta, c = 0.25, 1.0 / 0.9
    side = []
    for L, seed in ((Lc, 150), (Lr, 160)):
        z = make((P, L, V), dtype, dev, seed).requires_grad_()
        y = labels_of((P, L), V, dev, seed + 1)
        live = y != -7
        p, lq = softmax64(z, c) if L else (z.detach().double(), z.detach().double())
        lp = lq.gather(-1, y.clamp(min=0)[..., None])[..., 0]
        ref = (lp.float() + 0.3 * make((P, L), torch.float32, dev, seed + 2, 1.0)) if with_ref else None
        d = torch.where(live, lp - (0 if ref is None else ref.double()), torch.zeros_like(lp))
        rmag = (live * (1 + lp.abs() + (0 if ref is None else ref.double().abs()))).sum(1)
        if ref is not None:
            ref = torch.where(live, ref, torch.full_like(ref, float("nan")))
        side.append((z, y, live, p, lq, ref, beta * d.sum(1), beta * rmag))
    (zc, yc, livec, pc, lqc, refc, rwc, mc), (zr, yr, liver, pr, lqr, refr, rwr, mr) = side
    loss, got_c, got_r = ops.vocab_preference_loss(zc, yc, zr, yr, refc, refr, -7, c, beta, smooth, 3.0, avg)
    close(got_c, rwc, mc + 1e-30, "chosen")
    close(got_r, rwr, mr + 1e-30, "rejected")
    x, xmag = rwc - rwr, mc + mr
    n = P if avg == "seq" else 1
    rows = -(1 - smooth) * torch.nn.functional.logsigmoid(x) - smooth * torch.nn.functional.logsigmoid(-x)
    close(loss, 3.0 / n * rows.sum(), 3.0 / n * (rows.abs() + xmag + 0.1).sum(), "loss")
    slope = 3.0 / n * beta * (smooth * torch.sigmoid(x) - (1 - smooth) * torch.sigmoid(-x))
    smag = 3.0 / n * beta * (1 + xmag)
    zero = {True: torch.zeros(P, Lc, dtype=torch.float64, device=dev), False: torch.zeros(P, Lr, dtype=torch.float64, device=dev)}
    for up in (None, torch.tensor(-2.0, device=dev)):
        k = 1.0 if up is None else -2.0
        dc, dr = torch.autograd.grad(loss, [zc, zr], up, retain_graph=True)
        for d, z, y, live, p, lq, sign, side_ in ((dc, zc, yc, livec, pc, lqc, 1, True), (dr, zr, yr, liver, pr, lqr, -1, False)):
            yl = torch.where(live, y, torch.full_like(y, -1))
            h = zero[side_]
            if not y.numel():
                assert d.shape == z.shape
                continue
            want, _ = rows_grad64(p, lq, h, yl, k * sign * slope[:, None] * live, h, c)
            _, mag = rows_grad64(p, lq, h, yl, abs(k) * smag[:, None] * live, h, c)
            close(d, want, mag, "gradient")
    only, = torch.autograd.grad(ops.vocab_preference_loss(zc.detach(), yc, zr, yr, refc, refr, -7, c, beta, smooth, 3.0, avg)[0], zr)
    assert torch.equal(only, torch.autograd.grad(loss, zr)[0])


@pytest.mark.parametrize("V", [200, 5003])
def test_vocab_preference_one_answer_or_two_kinds(dev, V):
    """A gradient for one answer only, and answers of different types and vocabularies, are what two launches of their own give:
    the token log-probabilities and their loss do the same arithmetic."""
    from pevae_amd import ops
    P, Lc, Lr = 4, 5, 3
    yc, yr = labels_of((P, Lc), V, dev, 170), labels_of((P, Lr), V, dev, 171)
    for kinds in ((torch.bfloat16, V, torch.bfloat16, V), (torch.bfloat16, V, torch.float32, V), (torch.float16, V, torch.float16, V + 9)):
        zc, zr = make((P, Lc, kinds[1]), kinds[0], dev, 172), make((P, Lr, kinds[3]), kinds[2], dev, 173)
        got = {}
        for need_c, need_r in ((True, True), (True, False), (False, True)):
            xc, xr = zc.clone().requires_grad_(need_c), zr.clone().requires_grad_(need_r)
            loss = ops.vocab_preference_loss(xc, yc, xr, yr, ignore_index=-7)[0]
            loss.backward()
            got[need_c, need_r] = loss.detach(), xc.grad, xr.grad
        xc, xr = zc.clone().requires_grad_(), zr.clone().requires_grad_()
        loss = ops.preference_loss(ops.token_logprobs(xc, yc, -7), yc, ops.token_logprobs(xr, yr, -7), yr, ignore_index=-7)[0]
        loss.backward()
        for (need_c, need_r), (l, dc, dr) in got.items():
            assert torch.equal(l, loss.detach())
            assert (torch.equal(dc, xc.grad) if need_c else dc is None) and (torch.equal(dr, xr.grad) if need_r else dr is None)


def test_preference_far_apart(dev):
    """Rewards far apart: the loss is 0 or the distance, without overflow; infinite ones stay infinite."""
    from pevae_amd import ops
    y = torch.ones(4, 1, dtype=torch.int64, device=dev)
    c = torch.tensor([[-1e6], [0.0], [0.0], [float("-inf")]], device=dev).requires_grad_()
    r = torch.tensor([[0.0], [-1e6], [0.0], [0.0]], device=dev).requires_grad_()
    loss, rc, rr = ops.preference_loss(c, y, r, y, beta=1.0, avg_type=None)
    assert float(loss) == float("inf") and float(rc[3]) == float("-inf")
    loss, _, _ = ops.preference_loss(c[:3], y[:3], r[:3], y[:3], beta=1.0, avg_type=None)
    assert abs(float(loss) - (1e6 + math.log(2.0))) <= 0.07            # half a step of fp32 at 1e6, 0.03125, and ln 2's
    dc, dr = torch.autograd.grad(loss, [c, r])
    assert dc[:, 0].tolist() == [-1.0, 0.0, -0.5, 0.0] and dr[:, 0].tolist() == [1.0, 0.0, 0.5, 0.0]


# ------------------------------------------------------------------------------------------------------------
# gradients against differences
# ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["logp", "distill", "policy", "preference"])
def test_gradients_against_differences(dev, kind):
    """Central differences of the loss along a random direction.  With |z| of a few and step h the truncation is below
    h^2 |d|^3 (third derivatives of these losses are below 6 per unit), the loss's rounding adds EXP (1 + |loss|) / h."""
    from pevae_amd import ops
    B, L, V, K = 3, 4, 257, 9
    z = make((B, L, V), torch.float32, dev, 60, 1.0)
    y = labels_of((B, L), V, dev, 61, 0.2)
    t = make((B, L, V), torch.float32, dev, 62).topk(K, -1)
    old = ops.token_logprobs(z, y, ignore_index=-7) - 0.05
    adv = make((B,), torch.float32, dev, 63)

    def loss_of(x):
        if kind == "logp":
            lp, H = ops.token_logprobs(x, y, ignore_index=-7, inv_temp=0.9, entropy=True)
            return (lp * old).sum() / 12 + H.sum() / 12
        if kind == "distill":
            return ops.distill_topk(x, t.indices, t.values, y, -7, 1.5, avg_type="word")
        if kind == "policy":
            return ops.vocab_policy_loss(x, y, old, adv, old - 0.1, -7, kl_coef=0.1, ent_coef=0.05)[0]
        lp = ops.token_logprobs(x, y, ignore_index=-7)
        return ops.preference_loss(lp, y, 0.5 * lp, y, old, old, -7, beta=0.2)[0]

    x = z.clone().requires_grad_()
    loss = loss_of(x)
    d, = torch.autograd.grad(loss, x)
    way = make(z.shape, torch.float32, dev, 64, 1.0)
    way = way / way.norm()
    h = 0.05
    with torch.no_grad():
        diff = (loss_of(z + h * way) - loss_of(z - h * way)).double() / (2 * h)
    want = (d.double() * way.double()).sum()
    assert abs(float(diff - want)) <= 6 * h * h + EXP * (1 + abs(float(loss))) / h


# ------------------------------------------------------------------------------------------------------------
# sizes, streams, graphs
# ------------------------------------------------------------------------------------------------------------

def test_more_logits_than_32_bits_count(dev):
    """Rows behind the 2^31st element (and, in bytes, the 2^32nd)."""
    from pevae_amd import ops
    T, V = 16500, 131072
    z = torch.empty(T, V, dtype=torch.bfloat16, device=dev)
    z[:-3].zero_()
    tail = make((3, V), torch.bfloat16, dev, 70)
    z[-3:] = tail
    y = torch.full((T,), -7, dtype=torch.int64, device=dev)
    y[-3:] = torch.tensor([0, V - 1, 4242], device=dev)
    z.requires_grad_()
    p, lq = softmax64(tail, 1.0)
    H = -plogp(p, lq).sum(-1)
    one, none = torch.ones(3, dtype=torch.float64, device=dev), torch.zeros(3, dtype=torch.float64, device=dev)
    lp = ops.token_logprobs(z, y, ignore_index=-7)
    want = lq.gather(1, y[-3:, None])[:, 0]
    close(lp[-3:], want, 1 + want.abs(), "logp")
    assert float(lp[:-3].abs().max()) == 0.0
    d, = torch.autograd.grad(lp, z, torch.ones(T, device=dev))
    close(d[-3:], *rows_grad64(p, lq, H, y[-3:], one, none, 1.0), "dlogits")
    assert int(torch.count_nonzero(d[:-3])) == 0
    del d
    top = tail.float().topk(4, -1)
    ids, t = torch.zeros(T, 4, dtype=torch.int64, device=dev), torch.zeros(T, 4, device=dev)
    ids[-3:], t[-3:] = top.indices, top.values
    loss = ops.distill_topk(z, ids, t, y, -7, avg_type=None)
    want, mag, dwant, dmag = distill64(tail, top.indices, top.values, one > 0, 1.0, 1.0)
    close(loss, want, mag, "loss")
    d, = torch.autograd.grad(loss, z)
    close(d[-3:], dwant, dmag, "dlogits")
    assert int(torch.count_nonzero(d[:-3])) == 0


def test_many_rows(dev):
    """More rows than one workgroup sums, more than a grid's second dimension holds: loss and mean over live rows."""
    from pevae_amd import ops
    T, V = 70001, 33
    z = make((T, V), torch.float32, dev, 71).requires_grad_()
    y = labels_of((T,), V, dev, 72)
    live = y != -7
    t = z.detach().topk(3, -1)
    loss = ops.distill_topk(z, t.indices, t.values, y, -7, avg_type="word")
    want, mag, dwant, dmag = distill64(z, t.indices, t.values, live, 1.0, 1.0 / int(live.sum()))
    close(loss, want, mag, "loss")
    close(torch.autograd.grad(loss, z)[0], dwant, dmag, "dlogits")
    lp = ops.token_logprobs(z, y, ignore_index=-7)
    close(lp, torch.where(live, softmax64(z, 1.0)[1].gather(1, y.clamp(min=0)[:, None])[:, 0], torch.zeros((), dtype=torch.float64,
          device=dev)), 10.0, "logp")


def test_empty_batches(dev):
    from pevae_amd import ops
    z = torch.zeros(0, 4, 9, device=dev, requires_grad=True)
    y = torch.zeros(0, 4, dtype=torch.int64, device=dev)
    f = torch.zeros(0, 4, device=dev)
    lp = ops.token_logprobs(z, y)
    assert lp.shape == (0, 4)
    for loss in (ops.distill_topk(z, y[..., None], f[..., None]), ops.vocab_policy_loss(z, y, f, f)[0],
                 ops.policy_loss(lp, y, f, f)[0], ops.preference_loss(lp, y, lp, y)[0], ops.vocab_preference_loss(z, y, z, y)[0]):
        assert float(loss) == 0.0
        assert torch.autograd.grad(loss, z, retain_graph=True)[0].shape == z.shape


def test_same_bits_every_time_and_on_another_stream(dev):
    from pevae_amd import ops
    B, L, V = 40, 9, 5003
    z = make((B, L, V), torch.bfloat16, dev, 80).requires_grad_()
    y = labels_of((B, L), V, dev, 81)
    t = z.detach().float().topk(6, -1)
    old = make((B, L), torch.float32, dev, 82) - 8
    adv = make((B,), torch.float32, dev, 83)

    def once():
        lp, H = ops.token_logprobs(z, y, ignore_index=-7, entropy=True)
        a = ops.distill_topk(z, t.indices, t.values, y, -7, avg_type="word")
        b, stats = ops.vocab_policy_loss(z, y, old, adv, old + 0.1, -7, kl_coef=0.1, ent_coef=0.01)
        c, rc, rr = ops.preference_loss(lp[:20], y[:20], lp[20:], y[20:], ignore_index=-7)
        e = ops.vocab_preference_loss(z[:20], y[:20], z[20:], y[20:], ignore_index=-7)[0]
        grads = [torch.autograd.grad(x, z, retain_graph=True)[0] for x in (a, b, c, e)]
        return [x.detach() for x in (lp, H, a, b, stats, c, rc, rr, e)] + grads

    first = once()
    torch.cuda.synchronize()
    for other in (False, True):
        if other:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                again = once()
            torch.cuda.current_stream().wait_stream(s)
        else:
            again = once()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_captured_and_replayed(dev):
    """Two graphs of a whole step (forward and backward), replayed in turn with eager work and changed inputs between."""
    from pevae_amd import ops
    B, L, V = 6, 7, 3001
    y = labels_of((2 * B, L), V, dev, 90)
    old, adv = make((2 * B, L), torch.float32, dev, 91) - 8, make((2 * B,), torch.float32, dev, 92)

    def step(z):
        t = z.detach()[..., :64].float()
        ids = torch.arange(64, device=dev).expand(2 * B, L, 64).contiguous()
        lp = ops.token_logprobs(z, y, ignore_index=-7)
        a = ops.distill_topk(z, ids, t, y, -7, avg_type="word")
        b, stats = ops.vocab_policy_loss(z, y, old, adv, old, -7, kl_coef=0.1)
        c = ops.preference_loss(lp[:B], y[:B], lp[B:], y[B:], old[:B], old[B:], -7)[0]
        e = ops.policy_loss(lp, y, old, adv, ignore_index=-7)[0]
        f = ops.vocab_preference_loss(z[:B], y[:B], z[B:], y[B:], old[:B], old[B:], -7)[0]
        grads = [torch.autograd.grad(x, z, retain_graph=True)[0] for x in (a, b, c, e, f)]
        half = torch.autograd.grad(a, z, torch.full_like(a, 0.5), retain_graph=True)[0]
        return [x.detach() for x in (lp, a, b, stats, c, e, f)] + grads + [half]

    inputs = [make((2 * B, L, V), torch.bfloat16, dev, s) for s in (93, 94)]
    held = [x.clone().requires_grad_() for x in inputs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for x in held:
            step(x)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for x in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    for turn in range(4):
        fresh = [make((2 * B, L, V), torch.bfloat16, dev, 100 + 2 * turn + k) for k in range(2)]
        with torch.no_grad():
            for x, v in zip(held, fresh):
                x.copy_(v)
        want = [step(v.requires_grad_()) for v in fresh]
        torch.cuda.synchronize()
        for k in (turn & 1, 1 - (turn & 1)):
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want[k])), (turn, k)


def test_registered_operator(dev):
    import pevae_amd.torch_ops  # noqa: F401
    from pevae_amd import ops
    z = make((3, 4, 501), torch.float16, dev, 120)
    y = labels_of((3, 4), 501, dev, 121)
    assert torch.equal(torch.ops.pevae_amd.token_logprobs(z, y, -7, 0.9), ops.token_logprobs(z, y, -7, 0.9))


def test_refusals_on_the_device(dev):
    """An input changed in place after the forward pass, and a second derivative, are refused."""
    from pevae_amd import ops
    z = make((3, 11), torch.float32, dev, 110).requires_grad_()
    y = torch.tensor([1, 2, 3], device=dev)
    x = z * 1.0
    lp = ops.token_logprobs(x, y)
    x.add_(1.0)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(lp.sum(), z)
    d, = torch.autograd.grad(ops.token_logprobs(z, y).sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), z)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.token_logprobs(z, y.cpu())


# ------------------------------------------------------------------------------------------------------------
# together, behind the decoder
# ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(1, 1, 16, 2), (2, 3, 48, 7), (3, 5, 64, 1003), (4, 33, 128, 777), (2, 9, 512, 20004), (1, 3, 32, 65001)])
@pytest.mark.parametrize("kind", ["distill", "policy"])
def test_losses_behind_a_projection(dev, shape, kind):
    """Against 64 bits on the operands as the products see them (bf16).  A logit sums H products in fp32 (off by less than
    H u of their magnitudes); the logits' gradient is rounded to bf16 once (2^-8 of each element), and the products of it sum
    V or B L terms in fp32 (their count times u of the magnitudes, 4e-3 at most here, far less in fact: 1e-4 is granted)."""
    from pevae_amd import ops
    B, L, H, V = shape
    gen = torch.Generator(device=dev).manual_seed(200 + V)
    hid = (torch.randn(L, B, H, generator=gen, device=dev) * 0.5).transpose(0, 1).requires_grad_()        # time major
    w = (torch.randn(V, H, generator=gen, device=dev) * 0.2).requires_grad_()
    b = torch.randn(V, generator=gen, device=dev).requires_grad_()
    y = labels_of((B, L), V, dev, 201, 0.3)
    live = y != -7
    h64, w64 = hid.detach().bfloat16().double(), w.detach().bfloat16().double()
    z = h64 @ w64.t() + b.detach().double()
    zerr = H * 2.0 ** -24 * (h64.abs() @ w64.abs().t() + b.detach().abs().double()).max() / EXP             # in units of EXP
    c, tau = 1.0 / 0.8, 1.5
    if kind == "distill":
        K = min(V, 6)
        t = (make((B, L, V), torch.float32, dev, 202) + 0.5 * z.float()).topk(K, -1)
        n = max(int(live.sum()), 1)
        loss = ops.projected_distill_topk(hid, w, b, t.indices, t.values, y, -7, c, tau, 2.0, "word")
        p, lq = softmax64(z, c / tau)
        q, lt = softmax64(t.values, 1.0 / tau)
        on = live.double() * 2.0 / n
        rows = (q * (lt - lq.gather(-1, t.indices))).sum(-1)
        want, mag = tau * tau * (on * rows).sum(), tau * tau * (on * ((q * (lt.abs() + lq.gather(-1, t.indices).abs())).sum(-1) + 1)).sum()
        target = torch.zeros_like(p).scatter_add_(-1, t.indices, q)
        dz, dmag = (on * tau * c)[..., None] * (p - target), (on * tau * c)[..., None] * (p + target)
        outs = (loss,)
    else:
        p, lq = softmax64(z, c)
        Hh = -plogp(p, lq).sum(-1)
        lp = lq.gather(-1, y.clamp(min=0)[..., None])[..., 0]
        old, ref, adv = policy_inputs(lp, dev, 203)
        loss, stats = ops.projected_policy_loss(hid, w, b, y, old, adv, ref, -7, c, 0.2, 0.28, 0.1, 0.05, 2.0, "seq")
        pg, k3, cut, slope, smag = policy64(lp, old.double(), ref.double(), adv.double(), live, 0.8, 1.28, 0.1)
        on = live.double() * 2.0 / B
        want = (2.0 / B) * (pg + 0.1 * k3).sum() - 0.05 * (on * Hh).sum()
        mag = (2.0 / B) * (pg.abs() + 3 * smag + 0.1 * k3).sum() + 0.05 * (on * (1 + Hh)).sum()
        yl = torch.where(live, y, torch.full_like(y, -1))
        dz, _ = rows_grad64(p, lq, Hh, yl, (2.0 / B) * slope, -0.05 * on, c)
        _, dmag = rows_grad64(p, lq, Hh, yl, (2.0 / B) * 3 * smag, -0.05 * on, c)
        outs = (loss, stats)
        assert not stats.requires_grad
    close(loss, want, (1 + zerr) * mag + 1e-30, "loss")
    err = (2.0 ** -8 + 1e-4) * dz.abs() + (EXP * (1 + zerr) + 1e-4) * dmag
    d2, e2, h2 = dz.reshape(B * L, V), err.reshape(B * L, V), h64.reshape(B * L, H)
    for up in (None, torch.tensor(-2.5, device=dev), None):
        k = 1.0 if up is None else -2.5
        gh, gw, gb = torch.autograd.grad(loss, [hid, w, b], up, retain_graph=True)
        for got, exact, tol, name in ((gh.reshape(B * L, H), d2 @ w64, e2 @ w64.abs(), "hid"), (gw, d2.t() @ h2, e2.t() @ h2.abs(), "weight"),
                                      (gb, d2.sum(0), e2.sum(0), "bias")):
            over = (got.double() - k * exact).abs() / (abs(k) * tol + 1e-30)
            assert float(over.max()) <= 1.0, "%s: %.3g of the tolerance" % (name, float(over.max()))
    with torch.no_grad():
        again = ops.projected_distill_topk(hid, w, b, t.indices, t.values, y, -7, c, tau, 2.0, "word") if kind == "distill" else \
            ops.projected_policy_loss(hid, w, b, y, old, adv, ref, -7, c, 0.2, 0.28, 0.1, 0.05, 2.0, "seq")[0]
    close(again, want, (1 + zerr) * mag + 1e-30, "loss alone")
    only, = torch.autograd.grad(ops.projected_distill_topk(hid.detach(), w.detach(), b, t.indices, t.values, y, -7, c, tau, 2.0, "word")
                                if kind == "distill" else
                                ops.projected_policy_loss(hid.detach(), w.detach(), b, y, old, adv, ref, -7, c, 0.2, 0.28, 0.1, 0.05,
                                                          2.0, "seq")[0], b)
    assert torch.equal(only, gb)


@pytest.mark.parametrize("shape", [(3, 5, 64, 1003), (2, 64, 40, 301)])
def test_dead_rows_behind_a_projection_hold_anything(dev, shape):
    """NaN and infinities in the states of dead rows reach no result."""
    from pevae_amd import ops
    B, L, H, V = shape
    y = labels_of((B, L), V, dev, 220, 0.4)
    hid, w, b = (make(s, torch.float32, dev, k, 0.3) for k, s in ((221, (B, L, H)), (222, (V, H)), (223, (V,))))
    t = make((B, L, V), torch.float32, dev, 224).topk(5, -1)
    old, adv = make((B, L), torch.float32, dev, 225) - 6, make((B,), torch.float32, dev, 226)
    dead = torch.nonzero((y == -7).view(-1))[:, 0]
    assert dead.numel() >= 2

    def step(h):
        xs = [x.clone().requires_grad_() for x in (h, w, b)]
        loss = ops.projected_distill_topk(*xs, t.indices, t.values, y, -7), \
            ops.projected_policy_loss(*xs, y, old, adv, old, -7, kl_coef=0.1, ent_coef=0.01)[0]
        return [x.detach() for x in loss] + [g for x in loss for g in torch.autograd.grad(x, xs)]

    foul = hid.clone()
    foul.view(B * L, H)[dead[::2]] = float("nan")
    foul.view(B * L, H)[dead[1::2]] = float("inf")
    for a, c in zip(step(hid), step(foul)):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, c)


def test_more_projected_logits_than_32_bits_count(dev):
    """The last rows of 27000 x 81900 logits (2.2e9, behind the 2^31st) have the gradient that they have alone, rows and products
    being the same; sums in another order move it by 1e-5 of the largest at most."""
    from pevae_amd import ops
    T, V, H, K = 27000, 81900, 64, 4
    hid, w, b = (make(s, torch.float32, dev, k, 0.3) for k, s in ((240, (1, T, H)), (241, (V, H)), (242, (V,))))
    ids = torch.randint(0, V // 2, (1, T, 1), generator=torch.Generator(device=dev).manual_seed(243), device=dev) + torch.arange(K, device=dev)
    t = make((1, T, K), torch.float32, dev, 244)
    grads = []
    for at in (0, T - 8):
        x = hid[:, at:].clone().requires_grad_()
        loss = ops.projected_distill_topk(x, w, b, ids[:, at:].contiguous(), t[:, at:].contiguous(), avg_type=None)
        grads.append(torch.autograd.grad(loss, x)[0][0, -8:])
    assert float((grads[0] - grads[1]).abs().max()) <= 1e-5 * float(grads[1].abs().max())


def test_labels_of_deferred_rows(dev):
    """Labels of any integer type and stride (views of one storage among them), and their refusals."""
    from pevae_amd.enc2dec import decoders as D
    B, L, H, V = 2, 4, 64, 77
    hid, w, b = (make(s, torch.float32, dev, k, 0.3) for k, s in ((230, (B, L, H)), (231, (V, H)), (232, (V,))))
    wide = labels_of((B, 2 * L), V, dev, 233)
    out = D.DeferredLogProbs(hid, w, b, 1.0)
    want = torch.log_softmax(out.materialize().double(), -1)
    for y in (wide[:, ::2], wide[:, :L], wide[:, L:], wide[:, :L].to(torch.int32), wide[:, :L].contiguous()):
        lp = out.token_logp(y, -7)
        y = y.long()
        exact = torch.where(y != -7, want.gather(-1, y.clamp(min=0)[..., None])[..., 0], 0.0)
        assert float((lp - exact).abs().max()) <= 2e-4
    with pytest.raises(RuntimeError):
        out.token_logp(wide[:, :L].cpu(), -7)
    with pytest.raises(ValueError):
        out.token_logp(wide, -7)
    with pytest.raises(ValueError):
        out.token_logp(wide[:, :L].float(), -7)


def test_losses_behind_a_projection_captured(dev):
    """A graph of forward and backward, replayed with eager work and changed inputs between."""
    from pevae_amd import ops
    B, L, H, V = 5, 7, 64, 2003
    y = labels_of((B, L), V, dev, 210)
    ids = torch.arange(9, device=dev).expand(B, L, 9).contiguous()
    t = make((B, L, 9), torch.float32, dev, 211)
    old, adv = make((B, L), torch.float32, dev, 212) - 8, make((B,), torch.float32, dev, 213)
    params = [make(s, torch.float32, dev, k, 0.3) for k, s in ((214, (B, L, H)), (215, (V, H)), (216, (V,)))]

    def step(xs):
        a = ops.projected_distill_topk(*xs, ids, t, y, -7)
        b = ops.projected_policy_loss(*xs, y, old, adv, old, -7, kl_coef=0.1, ent_coef=0.01)[0]
        return [a.detach(), b.detach()] + [g for x in (a, b) for g in torch.autograd.grad(x, xs)]

    held = [x.clone().requires_grad_() for x in params]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(held)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(held)
    for turn in range(3):
        with torch.no_grad():
            for x, v in zip(held, params):
                x.copy_(v * (1.0 + 0.1 * turn))
        want = step([(v * (1.0 + 0.1 * turn)).requires_grad_() for v in params])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn


def test_decoder_learns_from_a_teacher_and_from_judgments(dev):
    """A decoder scores sampled answers, distils a teacher, takes a policy and a preference step: through its DeferredLogProbs
    (the fused projection) and through its dense rows, both against the losses of the dense rows in 64 bits.  The projection
    rounds its operands to bf16, the same way on both roads; the gradient of the weights passes through bf16 probabilities
    (relative error 2^-9 a term) on each."""
    from pevae_amd import criterions
    from pevae_amd.enc2dec import decoders as D
    torch.manual_seed(3)
    V, L, E, H, B = 211, 9, 24, 64, 6
    dec = D.DecoderRNN(V, L, E, H, 1, 2, 3, rnn_cell="gru", embedding=torch.nn.Embedding(V, E, padding_idx=0)).to(dev)
    ids = torch.randint(4, V, (B, L), device=dev)
    y = torch.cat([ids[:, 1:], torch.zeros(B, 1, dtype=torch.long, device=dev)], 1)
    y[2, 4:] = 0
    h0 = torch.randn(1, B, H, device=dev) * 0.3

    def outs():
        return dec(B, ids, h0, mode=D.TEACH_FORCE)[0]

    with torch.no_grad():
        lp = criterions.token_log_probs(outs(), y, 0)
        dense = outs().materialize()
        close(criterions.token_log_probs(dense, y, 0), torch.where(y != 0, dense.double().gather(-1, y[..., None])[..., 0], 0.0), 10.0)
        assert float((lp - criterions.token_log_probs(dense, y, 0)).abs().max()) <= 2e-4 and float(lp[y == 0].abs().max()) == 0.0
    old, ref, adv = lp - 0.1, lp + 0.05 * torch.randn_like(lp), torch.randn(B, device=dev)
    teacher = torch.randn(B, L, V, device=dev).topk(8, -1)
    policy = criterions.ClippedPolicyLoss(0, None, kl_coef=0.1)
    prefer = criterions.PreferenceLoss(0, None, beta=0.5)
    distill = criterions.TopKDistill(0, None, temperature=2.0)
    explore = criterions.ClippedPolicyLoss(0, None, kl_coef=0.1, ent_coef=0.1)
    h = B // 2
    half = [outs_slice for outs_slice in (slice(0, h), slice(h, B))]

    def losses(view):
        def part(s):
            return dec(h, ids[s], h0[:, s].contiguous(), mode=D.TEACH_FORCE)[0]
        return [distill(view(outs()), y, teacher.indices, teacher.values),
                policy(view(outs()), y, old, adv, ref)[0],
                prefer(view(part(half[0])), y[half[0]], view(part(half[1])), y[half[1]], ref[half[0]], ref[half[1]])[0],
                explore(view(outs()), y, old, adv, ref)[0]]

    roads = []
    for view in (lambda o: o, lambda o: o.materialize()):
        got = []
        for k in range(4):
            dec.zero_grad()
            loss = losses(view)[k]
            loss.backward()
            got.append((float(loss), dec.project.weight.grad.clone(), dec.project.bias.grad.clone()))
        roads.append(got)
    live = y != 0
    x = dense.double()
    want0 = distill64(dense, teacher.indices, teacher.values, live, 2.0, 1.0 / B)[0]
    lp64 = torch.where(live, x.gather(-1, y[..., None])[..., 0], torch.zeros((), dtype=torch.float64, device=dev))
    pg, k3, _, _, _ = policy64(lp64, old.double(), ref.double(), adv.double(), live, 0.8, 1.2, 0.1)
    want1 = (pg + 0.1 * k3).sum() / int(live.sum())
    dl = torch.where(live, lp64 - ref.double(), torch.zeros_like(lp64)).sum(1)
    want2 = -torch.nn.functional.logsigmoid(0.5 * (dl[:h] - dl[h:])).mean()
    ent = -plogp(torch.exp(x), x).sum(-1)
    want3 = want1 - 0.1 * torch.where(live, ent, torch.zeros_like(ent)).sum() / int(live.sum())
    for road in roads:
        for (loss, gw, gb), want in zip(road, (want0, want1, want2, want3)):
            assert abs(loss - float(want)) <= 2e-3 * (1 + abs(float(want)))
            assert float(gw.abs().max()) > 0 and bool(torch.isfinite(gw).all())
    for a, b in zip(*roads):
        for i in (1, 2):
            assert float((a[i] - b[i]).abs().max()) <= 2e-2 * float(b[i].abs().max())


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("drop", [0.0, 0.3])
def test_losses_of_one_forward_pass_add_up(dev, sink, drop):
    """The NLL, distillation, a policy loss and one with an entropy bonus on ONE decoder output, backward in one pass with the
    framework's side streams, with and without gradients that are accumulated into: the sum of the gradients of each alone,
    under the same dropout masks (a mask goes by the generator's step and the call's number: nothing advances the one, and the
    other starts at 0 for every pass).  The projection's gradients are sums of the same fp32 terms (V, H and B L of them: 1e-4 of
    the largest is granted); what passes the recurrence is rounded to bf16 on the way, once for the sum and once for each
    alone.  A policy loss in front of the NLL shares its node, whose weight gradient rounds p_v g_t to bf16: once for the sum of
    both g, once for each alone, half a step (2^-8) of |p_v g_t| at most each, so that an element is off by no more than
    2 * 2^-8 * sum_t |p_v - [v = y_t]| |g_t| |h_t|, with |h| <= 1 / (1 - drop)."""
    from pevae_amd import criterions, ops
    from pevae_amd.dls_vae import DLSVAE
    from pevae_amd.enc2dec import decoders as D
    torch.manual_seed(11)
    V, L, E, H, B = 5003, 12, 64, 512, 8
    dec = D.DecoderRNN(V, L, E, H, 1, 2, 3, rnn_cell="gru", dropout_p=drop, input_dropout_p=drop,
                       embedding=torch.nn.Embedding(V, E, padding_idx=0)).to(dev).train()
    ids = torch.randint(4, V, (B, L), device=dev)
    y = torch.cat([ids[:, 1:], torch.zeros(B, 1, dtype=torch.long, device=dev)], 1)
    y[1, 5:], y[6, 1:] = 0, 0
    h0 = (torch.randn(1, B, H, device=dev) * 0.3).requires_grad_()
    teacher = torch.randn(B, L, V, device=dev).topk(8, -1)
    adv = torch.randn(B, device=dev)
    with torch.no_grad():
        old = criterions.token_log_probs(dec(B, ids, h0, mode=D.TEACH_FORCE)[0], y, 0) - 0.1
    losses = [lambda o: criterions.NLLEntropy(0, None)(o, y),
              lambda o: criterions.TopKDistill(0, None, weight=0.5)(o, y, teacher.indices, teacher.values),
              lambda o: criterions.ClippedPolicyLoss(0, None)(o, y, old, adv)[0],
              lambda o: criterions.ClippedPolicyLoss(0, None, ent_coef=0.1)(o, y, old, adv)[0]]
    params = [p for p in dec.parameters()] + [h0]

    def grads(chosen):
        for p in params:
            p.grad = torch.zeros_like(p) if sink else None
        for m in dec.modules():
            if isinstance(m, ops.Dropout):
                m.calls = 0
        out = dec(B, ids, h0, mode=D.TEACH_FORCE)[0]
        terms = [f(out) for f in chosen]
        DLSVAE._run_backward(lambda: torch.autograd.backward(terms))
        return [p.grad.clone() for p in params]

    alone = [grads([f]) for f in losses]
    lp = (old + 0.1).requires_grad_()
    g = 1.0 / B + float(torch.autograd.grad(ops.policy_loss(lp, y, old, adv, ignore_index=0)[0], lp)[0].abs().max()) * 4
    count = torch.bincount(y[y != 0], minlength=V).max()         # rows that have a word as their target; p adds less than 1 to them
    shared = 2 * 2.0 ** -8 * (float(count) + 1) * g / (1 - drop)
    for chosen in ((0, 1, 2, 3), (3, 2, 1, 0), (0, 1)):
        for p, got, *each in zip(params, grads([losses[k] for k in chosen]), *[alone[k] for k in chosen]):
            want, top = sum(each), max(float(e.abs().max()) for e in each)
            share = 1e-4 if p is dec.project.weight or p is dec.project.bias else 2e-2
            extra = shared if chosen == (3, 2, 1, 0) and p is dec.project.weight else 0.0
            assert float((got - want).abs().max()) <= share * len(each) * top + extra
