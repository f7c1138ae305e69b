"""Loss modules with the reference's names and signatures (models/criterions.py:24-211) on HIP kernels.

NLLEntropy / Perplexity accept either a dense log-prob tensor (reference behaviour) or the decoder's
`DeferredLogProbs`, in which case the fused vocab GEMM + online-softmax + NLL kernel is used and the [B,L,V]
tensor is never built."""
import os

import torch
from torch.nn.modules.loss import _Loss

from . import ops
from .enc2dec.decoders import DeferredLogProbs

FUSED_HEAD = os.environ.get("PEVAE_NLL_HEAD", "1") == "1"      # ops.NllHead: 'seq' NLL and perplexity in one launch


def _token_nll(net_output, labels, padding_idx):
    """-> (sum of token NLL, number of non-pad tokens) as device scalars."""
    if isinstance(net_output, DeferredLogProbs):
        return net_output.token_nll_sums(labels, padding_idx)
    flat = net_output.reshape(-1, net_output.size(-1))
    tgt = labels.reshape(-1)
    picked = ops.GatherNLL.apply(flat, tgt, padding_idx)
    sums = ops.MaskedSum.apply(picked, tgt, padding_idx)
    return sums[0], sums[1]


class NLLEntropy(_Loss):
    """criterions.py:24-77 (weight=None path).  avg_type: 'seq' = sum / batch, 'word' = token mean, None = sum;
    'real_word' is broken in the reference (reduction=None, :46) and raises here as well."""

    def __init__(self, padding_idx, config, rev_vocab=None, key_vocab=None, avg_type="seq"):
        super().__init__()
        self.padding_idx = padding_idx
        self.avg_type = avg_type
        if rev_vocab is not None and key_vocab is not None:
            raise NotImplementedError("pevae_amd NLLEntropy: per-word loss weights are not supported")
        if avg_type not in ("word", "real_word", "seq", None):
            raise NotImplementedError("Unknown avg type")

    def forward(self, net_output, labels):
        batch_size = net_output.size(0)
        if self.avg_type == 'seq' and isinstance(net_output, DeferredLogProbs) and FUSED_HEAD:
            return net_output.loss_head(labels, self.padding_idx)[0]
        total, count = _token_nll(net_output, labels, self.padding_idx)
        if self.avg_type is None:
            return total
        if self.avg_type == 'seq':
            return total / batch_size
        if self.avg_type == 'word':
            return total / count
        raise ValueError("Unknown avg type")


class Perplexity(_Loss):
    """criterions.py:117-138: exp(token-mean NLL)."""

    def __init__(self, padding_idx, config, rev_vocab=None, key_vocab=None):
        super().__init__()
        self.padding_idx = padding_idx
        if rev_vocab is not None and key_vocab is not None:
            raise NotImplementedError("pevae_amd Perplexity: per-word loss weights are not supported")

    def forward(self, net_output, labels):
        if isinstance(net_output, DeferredLogProbs) and FUSED_HEAD:
            return net_output.loss_head(labels, self.padding_idx)[1]
        total, count = _token_nll(net_output, labels, self.padding_idx)
        return torch.exp(total / count)


class NormKLLoss(_Loss):
    """criterions.py:140-155 (logvar = log sigma^2)."""

    def __init__(self, unit_average=False):
        super().__init__()
        self.unit_average = unit_average

    def forward(self, recog_mu, recog_logvar, prior_mu, prior_logvar):
        _, kl_row = ops.reparam_kl(recog_mu, recog_logvar, prior_mu, prior_logvar, None, mode=0, want_z=False)
        if self.unit_average:
            kl_row = kl_row / recog_mu.size(1)
        return ops.mean(kl_row)


class CatKLLoss(_Loss):
    """criterions.py:157-175."""

    def forward(self, log_qy, log_py, batch_size=None, unit_average=False, average=True):
        if log_qy.dim() > 2:
            log_qy = log_qy.squeeze()
        y_kl = ops.CatRows.apply(log_qy, log_py, 0)
        if not average:
            return y_kl
        if unit_average:
            return ops.mean(y_kl)
        return ops.sum(y_kl) / batch_size


class Entropy(_Loss):
    """criterions.py:196-211."""

    def forward(self, log_qy, batch_size=None, unit_average=False):
        if log_qy.dim() > 2:
            log_qy = log_qy.squeeze()
        h_q = ops.CatRows.apply(log_qy, None, 1)
        if unit_average:
            return ops.mean(h_q)
        return ops.sum(h_q) / batch_size


# ------------------------------------------------------------------------------------------------------------
# Learning from another model's answers and from judgments of one's own: no counterpart in the reference.  Like the losses
# above they take a dense [B, L, V] tensor (log-probabilities or logits, fp32 / bf16 / fp16) or the decoder's DeferredLogProbs.
# ------------------------------------------------------------------------------------------------------------

def token_log_probs(net_output, labels, padding_idx):
    """Log-probability of `labels` [B, L] per token (fp32 [B, L], differentiable; 0 at padding): what the policy and preference
    losses ask of the old policy and of a reference model, under torch.no_grad()."""
    if isinstance(net_output, DeferredLogProbs):
        return net_output.token_logp(labels, padding_idx)
    return ops.token_logprobs(net_output, labels, ignore_index=padding_idx)


class TopKDistill(_Loss):
    """Distillation from a teacher's top logits (ops.distill_topk): forward(net_output, labels, teacher_ids, teacher_logits)
    with teacher_ids / teacher_logits [B, L, K] -> loss.  avg_type as NLLEntropy's: 'seq' = sum / batch, 'word' = token mean,
    None = sum.  A DeferredLogProbs is taken from its projection on (ops.projected_distill_topk): no log-probabilities are
    written, and no gradient of them."""

    def __init__(self, padding_idx, config, temperature=1.0, weight=1.0, avg_type="seq"):
        super().__init__()
        if avg_type not in ("word", "seq", None):
            raise NotImplementedError("Unknown avg type")
        self.padding_idx, self.temperature, self.weight, self.avg_type = padding_idx, temperature, weight, avg_type

    def forward(self, net_output, labels, teacher_ids, teacher_logits):
        if isinstance(net_output, DeferredLogProbs):
            if ops.projection_fits(net_output.size(2)):
                hid, w, b, inv_temp = net_output.projection()
                return ops.projected_distill_topk(hid, w, b, teacher_ids, teacher_logits, labels, self.padding_idx, inv_temp,
                                                  self.temperature, self.weight, self.avg_type)
            net_output = net_output.materialize()
        return ops.distill_topk(net_output, teacher_ids, teacher_logits, labels, self.padding_idx, self.temperature,
                                self.weight, self.avg_type)


class ClippedPolicyLoss(_Loss):
    """Clipped policy loss with a KL term and an entropy bonus (ops.vocab_policy_loss): forward(net_output, labels, old_logp,
    advantages, ref_logp=None) -> (loss, stats), labels = the sampled tokens [B, L], padded.  A DeferredLogProbs goes through
    the fused vocabulary projection (no [B, L, V] tensor), or with an entropy bonus, which needs the rows, through
    ops.projected_policy_loss."""

    def __init__(self, padding_idx, config, clip=0.2, clip_high=None, kl_coef=0.0, ent_coef=0.0, weight=1.0, avg_type="word"):
        super().__init__()
        if avg_type not in ("word", "seq", None):
            raise NotImplementedError("Unknown avg type")
        self.padding_idx, self.clip, self.clip_high = padding_idx, clip, clip_high
        self.kl_coef, self.ent_coef, self.weight, self.avg_type = kl_coef, ent_coef, weight, avg_type

    def forward(self, net_output, labels, old_logp, advantages, ref_logp=None):
        if isinstance(net_output, DeferredLogProbs):
            if self.ent_coef == 0:
                return ops.policy_loss(net_output.token_logp(labels, self.padding_idx), labels, old_logp, advantages, ref_logp,
                                       self.padding_idx, self.clip, self.clip_high, self.kl_coef, self.weight, self.avg_type)
            if ops.projection_fits(net_output.size(2)):
                hid, w, b, inv_temp = net_output.projection()
                return ops.projected_policy_loss(hid, w, b, labels, old_logp, advantages, ref_logp, self.padding_idx, inv_temp,
                                                 self.clip, self.clip_high, self.kl_coef, self.ent_coef, self.weight,
                                                 self.avg_type)
            net_output = net_output.materialize()
        return ops.vocab_policy_loss(net_output, labels, old_logp, advantages, ref_logp, self.padding_idx, 1.0, self.clip,
                                     self.clip_high, self.kl_coef, self.ent_coef, self.weight, self.avg_type)


class PreferenceLoss(_Loss):
    """Preference loss over pairs of answers (ops.preference_loss): forward(chosen_output, chosen_labels, rejected_output,
    rejected_labels, ref_chosen=None, ref_rejected=None) -> (loss, chosen rewards, rejected rewards).  The outputs are those
    of the decoder for the two answers; ref_*: the reference model's token_log_probs.  avg_type: 'seq' = mean over pairs,
    None = sum."""

    def __init__(self, padding_idx, config, beta=0.1, label_smoothing=0.0, weight=1.0, avg_type="seq"):
        super().__init__()
        if avg_type not in ("seq", None):
            raise NotImplementedError("Unknown avg type")
        self.padding_idx, self.beta, self.label_smoothing = padding_idx, beta, label_smoothing
        self.weight, self.avg_type = weight, avg_type

    def forward(self, chosen_output, chosen_labels, rejected_output, rejected_labels, ref_chosen=None, ref_rejected=None):
        if not isinstance(chosen_output, DeferredLogProbs) and not isinstance(rejected_output, DeferredLogProbs):
            return ops.vocab_preference_loss(chosen_output, chosen_labels, rejected_output, rejected_labels, ref_chosen,
                                             ref_rejected, self.padding_idx, 1.0, self.beta, self.label_smoothing, self.weight,
                                             self.avg_type)
        return ops.preference_loss(token_log_probs(chosen_output, chosen_labels, self.padding_idx), chosen_labels,
                                   token_log_probs(rejected_output, rejected_labels, self.padding_idx), rejected_labels,
                                   ref_chosen, ref_rejected, self.padding_idx, self.beta, self.label_smoothing, self.weight,
                                   self.avg_type)
