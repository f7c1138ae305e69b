"""The operators with which a decoder learns from another model's answers and from judgments of its own: per-token
log-probabilities of a vocabulary softmax, distillation from a teacher's top logits, the clipped policy loss with a KL
term, and the preference loss over pairs of answers -- forward and backward, in their plain form (elementary torch
operations in 32 bits) and as calls of this package.

Shapes: B sequences of L token rows, V words.  A label of 0 is padding (padding_idx of the criterions): its row is dead,
adds nothing to a loss and has a zero gradient.  Sequences end at random places, so about half of the rows of a batch with
L > 1 are dead, as in the synthetic review batches of this repository's benchmark."""
import math

import torch

own = False

PAD = 0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # serving: the score of one sampled word
        dict(name="score-one", kind="logp", B=1, L=1, V=20004, dtype="f32", temp=0.8, entropy=False, grad=False, padded=False),
        # the old policy's (or a reference model's) log-probabilities and entropies of a batch of sampled answers
        dict(name="score-batch", kind="logp", B=256, L=50, V=20004, dtype="bf16", temp=1.0, entropy=True, grad=False, padded=False),
        # any loss of a user's own on top of the log-probabilities; rows padded to a multiple of 64 words
        dict(name="logp-train", kind="logp", B=64, L=50, V=20004, dtype="f32", temp=1.0, entropy=True, grad=True, padded=True),
        # distillation: a unit-test sized batch, where launches count
        dict(name="distill-small", kind="distill", B=4, L=13, V=1009, K=5, dtype="f32", temp=1.0, avg="seq"),
        # distillation at the benchmark's batch, on the dense fp32 rows that the decoder materialises
        dict(name="distill-batch", kind="distill", B=256, L=50, V=20004, K=32, dtype="f32", temp=2.0, avg="seq"),
        # distillation with a large odd vocabulary, rows that start at odd addresses
        dict(name="distill-wide", kind="distill", B=8, L=127, V=131071, K=64, dtype="bf16", temp=1.0, avg="word"),
        # policy: a handful of answers, the loss scaled outside before its backward pass as half precision asks for
        dict(name="policy-small", kind="policy", B=2, L=9, V=20004, dtype="f16", avg="seq", kl=0.05, ent=0.0, up=1024.0),
        # policy: the benchmark's batch of sampled answers, from bf16 logits
        dict(name="policy-batch", kind="policy", B=256, L=50, V=20004, dtype="bf16", avg="word", kl=0.05, ent=0.0),
        # policy with an entropy bonus, a larger odd vocabulary; the loss scale of half precision given as the loss's weight
        dict(name="policy-wide", kind="policy", B=16, L=255, V=64001, dtype="f16", avg="word", kl=0.1, ent=0.01, weight=4096.0),
        # policy from log-probabilities, as the fused vocabulary projection hands them over
        dict(name="policy-tokens", kind="policy_tokens", B=256, L=50, avg="word", kl=0.05),
        # preference from log-probabilities: pairs of long answers
        dict(name="preference-tokens", kind="preference_tokens", B=512, L=1000, L2=911, smooth=0.0),
        # a preference step from the logits of both answers to their gradients
        dict(name="preference-train", kind="preference", B=64, L=50, L2=43, V=20004, dtype="bf16", smooth=0.1),
    ]


def draw(rng):
    """Sizes over the listed ranges: 1 to 256 sequences, 1 to 255 tokens, 500 to 160 000 words, at most 2^27 logits; 1 to 64
    teacher entries; up to 512 pairs of up to 1024 tokens."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["logp", "distill", "policy", "preference", "distill", "policy", "policy_tokens", "preference_tokens"])
    if kind == "policy_tokens":
        return dict(kind=kind, B=log_int(1, 512), L=log_int(1, 1024), avg=rng.choice(["seq", "word"]), kl=rng.choice([0.0, 0.05]))
    if kind == "preference_tokens":
        return dict(kind=kind, B=log_int(1, 512), L=log_int(1, 1024), L2=log_int(1, 1024), smooth=rng.choice([0.0, 0.1]))
    V, L = log_int(500, 160000), log_int(1, 255)
    B = log_int(1, max(1, min(256, (1 << 27) // (V * L * (2 if kind == "preference" else 1)))))
    L = max(1, min(L, (1 << 27) // (V * B)))
    c = dict(kind=kind, B=B, L=L, V=V, dtype=rng.choice(["f32", "bf16", "f16"]))
    if kind == "logp":
        c.update(temp=rng.choice([0.8, 1.0, 1.3]), entropy=rng.random() < 0.5, grad=rng.random() < 0.6, padded=rng.random() < 0.3)
    elif kind == "distill":
        c.update(K=log_int(1, 64), temp=rng.choice([1.0, 2.0]), avg=rng.choice(["seq", "word"]))
    elif kind == "policy":
        c.update(avg=rng.choice(["seq", "word"]), kl=rng.choice([0.0, 0.05]), ent=rng.choice([0.0, 0.0, 0.01]))
    else:
        c.update(L2=max(1, L - rng.randint(0, 7)), smooth=rng.choice([0.0, 0.1]))
    if c["dtype"] == "f16" and kind != "logp":      # gradients of 1 / tokens leave half precision's range without a scale
        c[rng.choice(["weight", "up"])] = 4096.0
    elif kind != "logp" and rng.random() < 0.2:     # one term of several in a total
        c[rng.choice(["weight", "up"])] = 0.5
    return c


# ------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------

def _labels(B, L, V, gen, dev):
    """Words 1 .. V - 1 up to a length that is uniform over 1 .. L, PAD behind it."""
    ids = torch.randint(1, V, (B, L), generator=gen, device=dev)
    length = torch.randint(1, L + 1, (B, 1), generator=gen, device=dev)
    return torch.where(torch.arange(L, device=dev) < length, ids, torch.full_like(ids, PAD))


def _logits(labels, V, dtype, gen, padded=False):
    """Rows of a trained decoder: normal scores of spread 2 with the target raised by 5."""
    B, L = labels.shape
    ld = (V + 63) // 64 * 64 if padded else V
    z = torch.randn(B, L, ld, generator=gen, device=labels.device).mul_(2.0)
    z.scatter_add_(2, labels[..., None], torch.full((B, L, 1), 5.0, device=labels.device))
    return z.to(dtype)[..., :V].detach().requires_grad_()


def _near(logp, spread, gen):
    """Log-probabilities that another state of the model gave the same words."""
    return (logp + spread * torch.randn(logp.shape, generator=gen, device=logp.device)).clamp_(max=0.0)


def _moved(logp, way, gen):
    """The reference model's log-probabilities after some steps of preference training: 0.2 to 0.5 a word below (way -1, the
    answers that were preferred) or above (way 1, the others)."""
    return (logp + way * (0.2 + 0.3 * torch.rand(logp.shape, generator=gen, device=logp.device))).clamp_(max=0.0)


def _randn(gen, dev, *shape):
    return torch.randn(*shape, generator=gen, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(1000003 * seed + 17)
    kind, B, L = case["kind"], case["B"], case["L"]
    s = dict(case=case, up=torch.full((), case.get("up", 1.0), device=dev) if "up" in case else None)
    with torch.no_grad():
        if kind.endswith("_tokens"):
            s["labels"] = _labels(B, L, 20004, gen, dev)
            s["logp"] = (-4.0 * torch.rand(B, L, generator=gen, device=dev)).requires_grad_()
            if kind == "preference_tokens":
                L2 = case["L2"]
                s["labels2"] = _labels(B, L2, 20004, gen, dev)
                s["logp2"] = (-4.0 * torch.rand(B, L2, generator=gen, device=dev)).requires_grad_()
                s["ref"], s["ref2"] = _moved(s["logp"], -1, gen), _moved(s["logp2"], 1, gen)
                return s
            s["old"], s["ref"] = _near(s["logp"], 0.15, gen), _near(s["logp"], 0.3, gen)
            s["adv"] = _randn(gen, dev, B)
            return s
        V, dtype = case["V"], TYPES[case["dtype"]]
        s["labels"] = _labels(B, L, V, gen, dev)
        s["logits"] = _logits(s["labels"], V, dtype, gen, case.get("padded", False))
        if kind == "logp":
            s["dlogp"], s["dent"] = _randn(gen, dev, B, L), _randn(gen, dev, B, L)
        elif kind == "distill":
            # the teacher agrees with the student about half: its own noise on half the student's scores
            t = _randn(gen, dev, B, L, V).mul_(1.5).add_(s["logits"].detach(), alpha=0.5)
            top = t.topk(case["K"], dim=-1)
            s["t_logits"], s["t_ids"] = top.values.to(dtype), top.indices
        elif kind == "policy":
            lp = _plain_logp(s["logits"], s["labels"], 1.0)[0]
            s["old"], s["ref"] = _near(lp, 0.15, gen), _near(lp, 0.3, gen)
            s["adv"] = _randn(gen, dev, B)
        else:
            s["labels2"] = _labels(B, case["L2"], V, gen, dev)
            s["logits2"] = _logits(s["labels2"], V, dtype, gen)
            s["ref"] = _moved(_plain_logp(s["logits"], s["labels"], 1.0)[0], -1, gen)
            s["ref2"] = _moved(_plain_logp(s["logits2"], s["labels2"], 1.0)[0], 1, gen)
    return s


# ------------------------------------------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits, one rounding at the end
# ------------------------------------------------------------------------------------------------------------

BETA, CLIP = 0.1, 0.2


def _plain_softmax(logits, inv_temp):
    """(probabilities, log-probabilities) of the rows."""
    z = logits.detach().float() * inv_temp
    z = z - z.amax(-1, keepdim=True)
    p = z.exp()
    s = p.sum(-1, keepdim=True)
    return p / s, z - s.log()


def _plain_logp(logits, labels, inv_temp):
    p, lq = _plain_softmax(logits, inv_temp)
    return lq.gather(-1, labels[..., None])[..., 0], p, lq


def _scale(avg, live):
    """What the sum over live tokens is divided by: the sequences, or the live tokens."""
    return live.shape[0] if avg == "seq" else live.sum().clamp(min=1).float()


def _plain_rows(p, lq, labels, dlogp, dent, ent, inv_temp, dtype):
    """Gradient of the logits for upstream gradients of the label's log-probability and of the entropy."""
    g = p * -dlogp[..., None]
    if dent is not None:
        g = g - p * (lq + ent[..., None]) * dent[..., None]
    g.scatter_add_(-1, labels[..., None], dlogp[..., None])
    return (g * inv_temp).to(dtype)


def _plain_policy(lp, live, old, ref, adv, kl, avg):
    """Policy and KL term a token, the derivative of their sum by the log-probability, and whether the clip decides."""
    a = adv[:, None]
    r = (lp - old).exp()
    u, w = r * a, r.clamp(1 - CLIP, 1 + CLIP) * a
    cut = u > w
    d = ref - lp
    pg, k3 = -torch.minimum(u, w), d.expm1() - d
    dlp = torch.where(cut, torch.zeros_like(u), -u) - kl * d.expm1()
    n = _scale(avg, live)
    zero = torch.zeros_like(pg)
    return torch.where(live, pg, zero), torch.where(live, k3, zero), torch.where(live, dlp, zero) / n, cut & live, n


def _plain_preference(lp, lp2, s, case):
    live, live2 = s["labels"] != PAD, s["labels2"] != PAD
    d = torch.where(live, lp - s["ref"], torch.zeros_like(lp)).sum(1)
    d2 = torch.where(live2, lp2 - s["ref2"], torch.zeros_like(lp2)).sum(1)
    x, e = BETA * (d - d2), case["smooth"]
    loss = (1 - e) * torch.logaddexp(-x, torch.zeros_like(x)) + e * torch.logaddexp(x, torch.zeros_like(x))
    dx = (e * torch.sigmoid(x) - (1 - e) * torch.sigmoid(-x)) * BETA / len(x)
    zero = torch.zeros((), device=x.device)
    weight = case.get("weight", 1.0)
    dx = dx * (weight * case.get("up", 1.0))
    return (weight * loss.sum() / len(x), BETA * d, BETA * d2, torch.where(live, dx[:, None], zero),
            torch.where(live2, -dx[:, None], zero))


def _run_plain(s):
    case, kind, labels = s["case"], s["case"]["kind"], s["labels"]
    live = labels != PAD
    weight, up = case.get("weight", 1.0), case.get("up", 1.0)
    if kind == "logp":
        c = 1.0 / case["temp"]
        lp, p, lq = _plain_logp(s["logits"], labels, c)
        zero = torch.zeros_like(lp)
        out = {"logp": torch.where(live, lp, zero)}
        ent = None
        if case["entropy"]:
            ent = -(p * lq).sum(-1)
            out["entropy"] = torch.where(live, ent, zero)
        if case["grad"]:
            out["dlogits"] = _plain_rows(p, lq, labels, torch.where(live, s["dlogp"], zero),
                                         torch.where(live, s["dent"], zero) if case["entropy"] else None, ent, c,
                                         s["logits"].dtype)
        return out
    if kind == "distill":
        tau = case["temp"]
        p, lq = _plain_softmax(s["logits"], 1.0 / tau)
        t, lt = _plain_softmax(s["t_logits"], 1.0 / tau)
        rows = (t * (lt - lq.gather(-1, s["t_ids"]))).sum(-1)
        n = _scale(case["avg"], live)
        w = live.float() * (weight * tau * tau / n)
        dz = (p * w[..., None]).scatter_add_(-1, s["t_ids"], -t * w[..., None]) * (up / tau)
        return {"loss": (rows * w).sum(), "dlogits": dz.to(s["logits"].dtype)}
    if kind == "policy":
        lp, p, lq = _plain_logp(s["logits"], labels, 1.0)
        pg, k3, dlp, cut, n = _plain_policy(lp, live, s["old"], s["ref"], s["adv"], case["kl"], case["avg"])
        ent = torch.where(live, -(p * lq).sum(-1), torch.zeros_like(lp))
        dlp = dlp * (weight * up)
        dent = -case["ent"] * weight * up / n * live.float() if case["ent"] else None
        count = live.sum().clamp(min=1)
        return {"loss": weight * (pg + case["kl"] * k3 - case["ent"] * ent).sum() / n,
                "stats": torch.stack([pg.sum(), k3.sum(), cut.sum().float(), ent.sum()]) / count,
                "dlogits": _plain_rows(p, lq, labels, dlp, dent, ent, 1.0, s["logits"].dtype)}
    if kind == "policy_tokens":
        pg, k3, dlp, cut, n = _plain_policy(s["logp"].detach(), live, s["old"], s["ref"], s["adv"], case["kl"], case["avg"])
        return {"loss": (pg + case["kl"] * k3).sum() / n,
                "stats": torch.stack([pg.sum(), k3.sum(), cut.sum().float()]) / live.sum().clamp(min=1), "dlogp": dlp}
    if kind == "preference_tokens":
        loss, rc, rr, dc, dr = _plain_preference(s["logp"].detach(), s["logp2"].detach(), s, case)
        return {"loss": loss, "chosen": rc, "rejected": rr, "dlogp": dc, "dlogp2": dr}
    lp, p, lq = _plain_logp(s["logits"], labels, 1.0)
    lp2, p2, lq2 = _plain_logp(s["logits2"], s["labels2"], 1.0)
    loss, rc, rr, dc, dr = _plain_preference(lp, lp2, s, case)
    return {"loss": loss, "chosen": rc, "rejected": rr,
            "dlogits": _plain_rows(p, lq, labels, dc, None, None, 1.0, s["logits"].dtype),
            "dlogits2": _plain_rows(p2, lq2, s["labels2"], dr, None, None, 1.0, s["logits2"].dtype)}


# ------------------------------------------------------------------------------------------------------------
# the same through this package
# ------------------------------------------------------------------------------------------------------------

def _run_own(s):
    from pevae_amd import criterions, ops
    case, kind, labels = s["case"], s["case"]["kind"], s["labels"]
    if kind == "logp":
        if not case["grad"]:
            with torch.no_grad():
                got = ops.token_logprobs(s["logits"], labels, ignore_index=PAD, inv_temp=1.0 / case["temp"], entropy=case["entropy"])
        else:
            got = ops.token_logprobs(s["logits"], labels, ignore_index=PAD, inv_temp=1.0 / case["temp"], entropy=case["entropy"])
        got = got if case["entropy"] else (got,)
        out = dict(zip(("logp", "entropy"), (t.detach() for t in got)))
        if case["grad"]:
            out["dlogits"], = torch.autograd.grad(got, [s["logits"]], [s["dlogp"], s["dent"]][:len(got)])
        return out
    if kind == "distill":
        crit = criterions.TopKDistill(PAD, None, temperature=case["temp"], weight=case.get("weight", 1.0), avg_type=case["avg"])
        loss = crit(s["logits"], labels, s["t_ids"], s["t_logits"])
        return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, s["logits"], s["up"])[0]}
    if kind == "policy":
        crit = criterions.ClippedPolicyLoss(PAD, None, clip=CLIP, kl_coef=case["kl"], ent_coef=case["ent"],
                                            weight=case.get("weight", 1.0), avg_type=case["avg"])
        loss, stats = crit(s["logits"], labels, s["old"], s["adv"], s["ref"])
        return {"loss": loss.detach(), "stats": stats, "dlogits": torch.autograd.grad(loss, s["logits"], s["up"])[0]}
    if kind == "policy_tokens":
        loss, stats = ops.policy_loss(s["logp"], labels, s["old"], s["adv"], s["ref"], ignore_index=PAD, clip=CLIP,
                                      kl_coef=case["kl"], avg_type=case["avg"])
        return {"loss": loss.detach(), "stats": stats[:3], "dlogp": torch.autograd.grad(loss, s["logp"])[0]}
    if kind == "preference_tokens":
        loss, rc, rr = ops.preference_loss(s["logp"], labels, s["logp2"], s["labels2"], s["ref"], s["ref2"], ignore_index=PAD,
                                           beta=BETA, label_smoothing=case["smooth"])
        d = torch.autograd.grad(loss, [s["logp"], s["logp2"]])
        return {"loss": loss.detach(), "chosen": rc, "rejected": rr, "dlogp": d[0], "dlogp2": d[1]}
    crit = criterions.PreferenceLoss(PAD, None, beta=BETA, label_smoothing=case["smooth"], weight=case.get("weight", 1.0))
    loss, rc, rr = crit(s["logits"], labels, s["logits2"], s["labels2"], s["ref"], s["ref2"])
    d = torch.autograd.grad(loss, [s["logits"], s["logits2"]], s["up"])
    return {"loss": loss.detach(), "chosen": rc, "rejected": rr, "dlogits": d[0], "dlogits2": d[1]}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------

def work(case):
    """Every live row of logits read once, every row of the gradient written once, the per-token arrays once."""
    B, L = case["B"], case["L"]
    kind = case["kind"]

    def share(n):
        return (n + 1) / (2.0 * n)           # of the rows that live, for lengths uniform over 1 .. n

    if kind == "policy_tokens":
        return {"bytes": B * L * (8 + 4 * 4) + 4 * B, "flops": 20 * B * L}
    if kind == "preference_tokens":
        T = B * (L + case["L2"])
        return {"bytes": T * (8 + 4 + 4 + 4) + 8 * B, "flops": 4 * T}
    V, es = case["V"], SIZE[case["dtype"]]

    def rows(n, backward, per_token):
        live = B * n * share(n)
        return (live * V * es + (B * n * V * es if backward else 0) + B * n * per_token,
                live * V * ((9 if backward else 5) + (4 if case.get("entropy") or case.get("ent") else 0)))

    if kind == "logp":
        b, f = rows(L, case["grad"], 8 + 4 + (4 if case["entropy"] else 0) + (4 if case["grad"] else 0))
    elif kind == "distill":
        b, f = rows(L, True, 8 + case["K"] * (8 + es))
    elif kind == "policy":
        b, f = rows(L, True, 8 + 4 + 4)
    else:
        b, f = rows(L, True, 8 + 4)
        b2, f2 = rows(case["L2"], True, 8 + 4)
        b, f = b + b2, f + f2
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, row by row
# ------------------------------------------------------------------------------------------------------------

def _lse64(z):
    m = z.max(dim=-1).values
    return m + torch.log(torch.exp(z - m[..., None]).sum(-1))


def _logp64(logits, labels, c):
    """Log-probability of the label and entropy of every token, from sequence to sequence."""
    lp, ent = [], []
    for zb, yb in zip(logits.detach(), labels):
        z = zb.double() * c
        norm = _lse64(z)
        lp.append(z[torch.arange(len(yb), device=yb.device), yb] - norm)
        ent.append(norm - (torch.exp(z - norm[:, None]) * z).sum(-1))
    return torch.stack(lp), torch.stack(ent)


def _dlogits64(logits, labels, c, dlp, dent, ent):
    """d(sum dlp log p[label] + dent H) / d logits = c (dlp (onehot - p) - dent p (log p + H))."""
    out = []
    for b, zb in enumerate(logits.detach()):
        z = zb.double() * c
        lq = z - _lse64(z)[:, None]
        hot = torch.nn.functional.one_hot(labels[b], z.shape[-1])
        row = dlp[b][:, None] * (hot - torch.exp(lq))
        if dent is not None:
            row = row - dent[b][:, None] * torch.exp(lq) * (lq + ent[b][:, None])
        out.append(c * row)
    return torch.stack(out)


def _policy64(lp, s, case):
    on = (s["labels"] != PAD).double()
    n = float(len(on)) if case["avg"] == "seq" else max(float(on.sum()), 1.0)
    count = max(float(on.sum()), 1.0)
    adv = s["adv"].double()[:, None].expand_as(lp)
    ratio = torch.exp(lp - s["old"].double())
    inside = torch.clamp(ratio, 1 - CLIP, 1 + CLIP)
    gain = torch.where(ratio * adv <= inside * adv, ratio * adv, inside * adv)
    cut = (ratio * adv > inside * adv).double()
    away = s["ref"].double() - lp
    k3 = torch.exp(away) - 1 - away
    slope = (-(1 - cut) * ratio * adv + case["kl"] * (1 - torch.exp(away))) * on / n
    means = [float((v * on).sum()) / count for v in (-gain, k3, cut)]
    return ((-gain + case["kl"] * k3) * on).sum() / n, means, slope, on, n, count


def _preference64(lp, lp2, s, case):
    on, on2 = (s["labels"] != PAD).double(), (s["labels2"] != PAD).double()
    rc = BETA * ((lp - s["ref"].double()) * on).sum(1)
    rr = BETA * ((lp2 - s["ref2"].double()) * on2).sum(1)
    x, e = rc - rr, case["smooth"]
    loss = (-(1 - e) * torch.nn.functional.logsigmoid(x) - e * torch.nn.functional.logsigmoid(-x)).mean()
    slope = (-(1 - e) / (1 + torch.exp(x)) + e / (1 + torch.exp(-x))) * BETA / len(x)
    weight = case.get("weight", 1.0)
    slope = slope * (weight * case.get("up", 1.0))
    return weight * loss, rc, rr, slope[:, None] * on, -slope[:, None] * on2


def exact(case, seed):
    s = prepare(case, seed)
    kind, labels = case["kind"], s["labels"]
    with torch.no_grad():
        on = (labels != PAD).double()
        if kind == "logp":
            c = 1.0 / case["temp"]
            lp, ent = _logp64(s["logits"], labels, c)
            out = {"logp": lp * on}
            if case["entropy"]:
                out["entropy"] = ent * on
            if case["grad"]:
                out["dlogits"] = _dlogits64(s["logits"], labels, c, s["dlogp"].double() * on,
                                            s["dent"].double() * on if case["entropy"] else None, ent)
            return out
        if kind == "distill":
            tau = case["temp"]
            n = float(len(on)) if case["avg"] == "seq" else max(float(on.sum()), 1.0)
            total, grads = 0.0, []
            for b, zb in enumerate(s["logits"].detach()):
                z, t, ids = zb.double() / tau, s["t_logits"][b].double() / tau, s["t_ids"][b]
                lt = t - _lse64(t)[:, None]
                lq = z - _lse64(z)[:, None]
                w = on[b] * (case.get("weight", 1.0) * tau * tau / n)
                total = total + (w * (torch.exp(lt) * (lt - lq.gather(1, ids))).sum(1)).sum()
                target = torch.zeros_like(z).scatter_(1, ids, torch.exp(lt))
                grads.append((torch.exp(lq) - target) * (w * case.get("up", 1.0) / tau)[:, None])
            return {"loss": total, "dlogits": torch.stack(grads)}
        if kind == "policy":
            lp, ent = _logp64(s["logits"], labels, 1.0)
            loss, means, slope, on, n, count = _policy64(lp, s, case)
            weight, up = case.get("weight", 1.0), case.get("up", 1.0)
            dent = -case["ent"] * weight * up / n * on if case["ent"] else None
            return {"loss": weight * (loss - case["ent"] * (ent * on).sum() / n),
                    "stats": torch.tensor(means + [float((ent * on).sum()) / count], dtype=torch.float64),
                    "dlogits": _dlogits64(s["logits"], labels, 1.0, slope * (weight * up), dent, ent)}
        if kind == "policy_tokens":
            loss, means, slope, _, _, _ = _policy64(s["logp"].detach().double(), s, case)
            return {"loss": loss, "stats": torch.tensor(means, dtype=torch.float64), "dlogp": slope}
        if kind == "preference_tokens":
            loss, rc, rr, dc, dr = _preference64(s["logp"].detach().double(), s["logp2"].detach().double(), s, case)
            return {"loss": loss, "chosen": rc, "rejected": rr, "dlogp": dc, "dlogp2": dr}
        lp, _ = _logp64(s["logits"], labels, 1.0)
        lp2, _ = _logp64(s["logits2"], s["labels2"], 1.0)
        loss, rc, rr, dc, dr = _preference64(lp, lp2, s, case)
        return {"loss": loss, "chosen": rc, "rejected": rr, "dlogits": _dlogits64(s["logits"], labels, 1.0, dc, None, None),
                "dlogits2": _dlogits64(s["logits2"], s["labels2"], 1.0, dr, None, None)}
