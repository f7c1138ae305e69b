"""Losses over rows of a vocabulary softmax in memory (ops.token_logprobs, distill_topk, vocab_policy_loss, policy_loss,
preference_loss and their criterions): what they refuse, without a GPU."""
import ctypes as C

import pytest
import torch

from pevae_amd import _lib, criterions, ops


def rows(B=2, L=3, V=5, dtype=torch.float32):
    return torch.zeros(B, L, V, dtype=dtype)


def ids(*shape):
    return torch.ones(*shape, dtype=torch.int64)


def f(*shape):
    return torch.zeros(*shape)


def test_valid_arguments_on_the_cpu_raise_for_the_device():
    for call in (lambda: ops.token_logprobs(rows(), ids(2, 3)),
                 lambda: ops.distill_topk(rows(), ids(2, 3, 2), f(2, 3, 2), ids(2, 3), 0),
                 lambda: ops.vocab_policy_loss(rows(), ids(2, 3), f(2, 3), f(2)),
                 lambda: ops.policy_loss(f(2, 3), ids(2, 3), f(2, 3), f(2, 3)),
                 lambda: ops.preference_loss(f(2, 3), ids(2, 3), f(2, 4), ids(2, 4)),
                 lambda: ops.vocab_preference_loss(rows(), ids(2, 3), rows(L=4), ids(2, 4)),
                 lambda: ops.projected_distill_topk(f(2, 3, 8), f(5, 8), f(5), ids(2, 3, 2), f(2, 3, 2)),
                 lambda: ops.projected_policy_loss(f(2, 3, 8), f(5, 8), f(5), ids(2, 3), f(2, 3), f(2))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("call", [
    lambda: ops.token_logprobs(rows(dtype=torch.float64), ids(2, 3)),                       # type
    lambda: ops.token_logprobs(rows(V=0), ids(2, 3)),                                       # no words
    lambda: ops.token_logprobs(rows(), ids(3, 2)),                                          # shape
    lambda: ops.token_logprobs(rows(), f(2, 3)),                                            # tokens are no integers
    lambda: ops.token_logprobs(rows(), ids(2, 3), inv_temp=0.0),
    lambda: ops.token_logprobs(rows(), ids(2, 3), inv_temp=float("nan")),
    lambda: ops.distill_topk(rows(), ids(2, 3, 2), f(2, 3, 3)),                             # ids and logits differ
    lambda: ops.distill_topk(rows(), ids(2, 3, 0), f(2, 3, 0)),                             # no entries
    lambda: ops.distill_topk(rows(), ids(2, 3, 257), f(2, 3, 257)),                         # too many
    lambda: ops.distill_topk(rows(), ids(2, 3, 2), f(2, 3, 2).requires_grad_()),            # no gradient for the teacher
    lambda: ops.distill_topk(rows(), ids(2, 3, 2), f(2, 3, 2), ids(2, 4)),
    lambda: ops.distill_topk(rows(), ids(2, 3, 2), f(2, 3, 2), temperature=0.0),
    lambda: ops.distill_topk(rows(), ids(2, 3, 2), f(2, 3, 2), avg_type="real_word"),
    lambda: ops.vocab_policy_loss(rows(), ids(2, 3), f(2, 3), f(3)),                        # advantages
    lambda: ops.vocab_policy_loss(rows(), ids(2, 3), f(2, 2), f(2)),                        # old_logp
    lambda: ops.vocab_policy_loss(rows(), ids(2, 3), f(2, 3), f(2), kl_coef=0.1),           # no reference model
    lambda: ops.vocab_policy_loss(rows(), ids(2, 3), f(2, 3), f(2), clip=-0.1),
    lambda: ops.vocab_policy_loss(rows(), ids(2, 3), f(2, 3).requires_grad_(), f(2)),
    lambda: ops.vocab_policy_loss(rows(), ids(2, 3), f(2, 3), ids(2)),                      # integer advantages
    lambda: ops.vocab_policy_loss(torch.zeros(1, 2, 3, 5), ids(1, 2, 3), f(1, 2, 3), f(1)),
    lambda: ops.policy_loss(f(2, 3).double(), ids(2, 3), f(2, 3), f(2)),
    lambda: ops.policy_loss(f(2, 3), ids(2, 3), f(2, 3), f(2), avg_type="mean"),
    lambda: ops.preference_loss(f(2, 3), ids(2, 3), f(3, 3), ids(3, 3)),                    # not pairs
    lambda: ops.preference_loss(f(6), ids(6), f(6), ids(6)),
    lambda: ops.preference_loss(f(2, 3), ids(2, 3), f(2, 3), ids(2, 3), ref_chosen=f(2, 3)),
    lambda: ops.preference_loss(f(2, 3), ids(2, 3), f(2, 3), ids(2, 3), label_smoothing=1.5),
    lambda: ops.preference_loss(f(2, 3), ids(2, 3), f(2, 3), ids(2, 3), avg_type="word"),
    lambda: ops.vocab_preference_loss(rows(), ids(2, 3), rows(B=3), ids(3, 3)),
    lambda: ops.vocab_preference_loss(rows()[0], ids(3), rows()[0], ids(3)),
    lambda: ops.vocab_preference_loss(rows(), ids(2, 3), rows(), ids(2, 3), f(2, 3)),
    lambda: ops.vocab_preference_loss(rows(), ids(2, 3), rows(), ids(2, 3), f(2, 3).requires_grad_(), f(2, 3)),
])
def test_bad_arguments_raise_value_errors(call):
    with pytest.raises(ValueError):
        call()


def test_registered_operator_has_a_fake_shape():
    import pevae_amd.torch_ops  # noqa: F401
    lp = torch.ops.pevae_amd.token_logprobs(torch.empty(4, 6, 500, device="meta", dtype=torch.bfloat16),
                                            torch.empty(4, 6, device="meta", dtype=torch.int64), 0, 1.0)
    assert lp.shape == (4, 6) and lp.dtype == torch.float32
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        torch.ops.pevae_amd.token_logprobs(rows(), ids(2, 3), 0, 1.0)


@pytest.mark.parametrize("call", [
    lambda h, w, b: ops.projected_distill_topk(h[0], w, b, ids(2, 3, 2), f(2, 3, 2)),
    lambda h, w, b: ops.projected_distill_topk(h.double(), w, b, ids(2, 3, 2), f(2, 3, 2)),
    lambda h, w, b: ops.projected_distill_topk(h, w[:, :4], b, ids(2, 3, 2), f(2, 3, 2)),
    lambda h, w, b: ops.projected_distill_topk(h, w, b[:4], ids(2, 3, 2), f(2, 3, 2)),
    lambda h, w, b: ops.projected_distill_topk(h, w, b, ids(2, 3, 2), f(2, 4, 2)),
    lambda h, w, b: ops.projected_distill_topk(h, w, b, ids(2, 3, 2), f(2, 3, 2), inv_temp=0.0),
    lambda h, w, b: ops.projected_policy_loss(h, w, b, ids(2, 3), f(2, 3), f(3)),
    lambda h, w, b: ops.projected_policy_loss(h, w, b, ids(2, 3), f(2, 3), f(2), kl_coef=0.5),
    lambda h, w, b: ops.projected_distill_topk(f(1, 1, 2), f(81924, 2), f(81924), ids(1, 1, 2), f(1, 1, 2)),         # does not fit
])
def test_bad_projections_raise_value_errors(call):
    with pytest.raises(ValueError):
        call(f(2, 3, 8), f(5, 8), f(5))


def test_criterions_refuse_unknown_averages():
    for cls in (criterions.TopKDistill, criterions.ClippedPolicyLoss, criterions.PreferenceLoss):
        with pytest.raises(NotImplementedError):
            cls(0, None, avg_type="real_word")


def test_entry_points_refuse_on_the_host():
    """Nothing is launched for bad sizes, types, null pointers, or sizes beyond the limits."""
    lib = _lib.load()
    p = C.c_void_p(64)

    def logp(logits=p, dtype=0, n0=1, n1=4, s0=0, s1=5, V=5, tokens=p, temp=1.0, out=p):
        return lib.pv_token_logp_fwd(logits, dtype, n0, n1, s0, s1, V, tokens, 0, temp, out, None, None, None)

    for bad in (dict(logits=None), dict(dtype=3), dict(n0=0), dict(n1=0), dict(V=0), dict(tokens=None), dict(out=None), dict(temp=0.0),
                dict(temp=float("inf")), dict(s1=-5), dict(logits=C.c_void_p(66)), dict(logits=C.c_void_p(65), dtype=1)):
        assert logp(**bad) == -1, bad
        assert b"pv_token_logp_fwd" in lib.pv_last_error()
    assert logp(n0=1 << 16, n1=1 << 15) == -3
    assert logp(V=(1 << 24) + 1) == -3
    assert logp(n0=1 << 13, n1=1 << 13) == -3 and logp(n0=1 << 62) == -3          # 2^26 rows; more than 64 bits count
    assert logp(n0=1 << 22, n1=1, V=16389, s0=0) == -3                            # 2^22 rows of 1024 threads
    assert lib.pv_preference_fwd(p, None, p, 3, p, None, p, 3, 1 << 24, 0, 0.1, 0.0, 1.0, p, p, p, p, None) == -3
    assert lib.pv_preference_bwd(p, 3, p, 3, 1 << 24, 0, p, 1.0, p, p, p, None) == -3
    assert lib.pv_gather_live_rows_bf16(p, p, p, 4, 12, p, None) == -1
    assert lib.pv_gather_live_rows_bf16(C.c_void_p(8), p, p, 4, 16, p, None) == -1
    assert lib.pv_distill_rows_fwd(p, 0, 1, 4, 0, 5, 5, None, 0, 1.0, 1.0, p, p, 0, 257, 1.0, 0, p, p, p, None, 0, None, p, None) == -3
    assert lib.pv_distill_rows_fwd(p, 0, 1, 4, 0, 5, 5, None, 0, 1.0, 1.0, p, p, 7, 4, 1.0, 0, p, p, p, None, 0, None, p, None) == -1
    assert lib.pv_policy_rows_fwd(p, 0, 1, 4, 0, 5, 5, p, 0, 1.0, p, None, p, 0, 1.2, 0.8, 0.0, 0.0, 1.0, 0, p, p, p, None, 0, None, p, None) == -1
    assert lib.pv_policy_tokens_fwd(p, p, 0, 0, 4, p, None, p, 0, 0.8, 1.2, 0.0, 1.0, 0, p, p, p, p, None) == -1
    assert lib.pv_preference_fwd(None, None, None, 3, p, None, p, 3, 2, 0, 0.1, 0.0, 1.0, p, p, p, p, None) == -1
    assert lib.pv_vocab_rows_one_pass(0, 81923) == 1 and lib.pv_vocab_rows_one_pass(0, 81924) == 0     # 20 480 pieces of 16 bytes
    assert lib.pv_vocab_rows_one_pass(1, 163847) == 1 and lib.pv_vocab_rows_one_pass(2, 163848) == 0
    assert lib.pv_distill_rows_fwd(p, 0, 1, 4, 0, 81924, 81924, None, 0, 1.0, 1.0, p, p, 0, 4, 1.0, 0, p, p, p, p, 0, None, p, None) == -1
    for dtype, ld in ((0, 4), (0, 70), (1, 64)):                # shorter than a row, too long, not fp32
        assert lib.pv_distill_rows_fwd(p, dtype, 1, 4, 0, 5, 5, None, 0, 1.0, 1.0, p, p, 0, 4, 1.0, 0, p, p, p, p, ld, None, p, None) == -1
    assert lib.pv_distill_rows_fwd(p, 0, 1, 4, 0, 5, 5, None, 0, 1.0, 0.0, p, p, 0, 4, 1.0, 0, p, p, p, None, 0, None, p, None) == -1
    assert lib.pv_distill_rows_fwd(p, 0, 1, 4, 0, 5, 5, None, 0, 1.0, 1.0, p, p, 0, 4, 1.0, 0, p, p, p, p, 0, p, p, None) == -1
    assert lib.pv_colsum_scaled_bf16(p, 7, 4, 7, p, p, p, None) == -1 and lib.pv_scale_by_f32(p, 6, p, None) == -1
    assert lib.pv_preference_rows_fwd(p, 0, 2, 3, 15, 5, 5, p, None, p, 0, 0, 15, 5, 5, p, None, 0, 1.0, 0.1, 0.0, 1.0, p, p, p, p, p, p,
                                      None) == -1

    def preference_bwd(save_c=p, save_r=p, dc=p, dr=p, Vr=5, dtype_r=0):
        return lib.pv_preference_rows_bwd(p, 0, 2, 3, 15, 5, 5, p, p, dtype_r, 3, 15, 5, Vr, p, 0, 1.0, save_c, save_r, p, 1.0, p, dc, dr,
                                          None)

    for bad in (dict(save_c=None), dict(save_r=None), dict(dc=None, dr=None), dict(Vr=0), dict(dtype_r=4)):
        assert preference_bwd(**bad) == -1, bad
    assert lib.pv_distill_max_entries() == 256 == ops.DISTILL_MAX
    assert lib.pv_vocab_rows_ws_bytes(10) >= 160
