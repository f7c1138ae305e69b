"""One decoder step (forward pass, loss, backward pass) under each loss that a decoder learns from, and the scoring of a batch, at
the Yelp shape: time per step, calls back to back, and the decoder alone.
Usage: python tools/bench_decoder_losses.py [--steps N] [--only "NAME;NAME"]"""
import argparse, os, sys, time
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch
from pevae_amd import criterions
from pevae_amd.enc2dec import decoders as D

ap = argparse.ArgumentParser()
ap.add_argument("--steps", type=int, default=20)
ap.add_argument("--only", default="")
a = ap.parse_args()
dev = torch.device("cuda:0")
V, L, E, H, B, K = 20004, 50, 100, 512, 256, 32
torch.manual_seed(0)
dec = D.DecoderRNN(V, L, E, H, 1, 2, 3, rnn_cell="gru", embedding=torch.nn.Embedding(V, E, padding_idx=0)).to(dev)
ids = torch.randint(4, V, (B, L), device=dev)
y = torch.where(torch.arange(L, device=dev) < torch.randint(1, L + 1, (B, 1), device=dev), ids, torch.zeros_like(ids))
h0 = torch.randn(1, B, H, device=dev) * 0.3
adv, t = torch.randn(B, device=dev), torch.randn(B, L, V, device=dev).topk(K, -1)
half = B // 2
nll, prefer = criterions.NLLEntropy(0, None), criterions.PreferenceLoss(0, None)
distill = criterions.TopKDistill(0, None, temperature=2.0)
policy = criterions.ClippedPolicyLoss(0, None, kl_coef=0.1)
explore = criterions.ClippedPolicyLoss(0, None, kl_coef=0.1, ent_coef=0.01)


def out(rows=slice(0, B)):
    return dec(len(ids[rows]), ids[rows], h0[:, rows].contiguous(), mode=D.TEACH_FORCE)[0]


def score():
    with torch.no_grad():
        return criterions.token_log_probs(out(), y, 0)


def forward():
    with torch.no_grad():
        return out()


old = score() - 0.1
steps = [("decoder forward, no gradients", None, forward),
         ("scoring, no gradients", None, score),
         ("nll", lambda: nll(out(), y), None),
         ("policy", lambda: policy(out(), y, old, adv, old)[0], None),
         ("policy, entropy bonus", lambda: explore(out(), y, old, adv, old)[0], None),
         ("policy, entropy bonus, dense", lambda: explore(out().materialize(), y, old, adv, old)[0], None),
         ("distillation", lambda: distill(out(), y, t.indices, t.values), None),
         ("distillation, dense", lambda: distill(out().materialize(), y, t.indices, t.values), None),
         ("preference, 2 x %d answers" % half, lambda: prefer(out(slice(0, half)), y[:half], out(slice(half, B)), y[half:],
                                                              old[:half], old[half:])[0], None)]
print("%d x %d tokens, V = %d, H = %d, K = %d, %.0f %% of the tokens live" % (B, L, V, H, K, 100.0 * float((y != 0).float().mean())))
for name, loss, call in steps:
    if a.only and name not in a.only.split(";"):
        continue

    def step():
        if loss is None:
            return call()
        dec.zero_grad()
        loss().backward()

    for _ in range(3):
        step()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(a.steps):
        step()
    torch.cuda.synchronize()
    print("%-32s %7.3f ms" % (name, (time.perf_counter() - t0) / a.steps * 1e3), flush=True)
