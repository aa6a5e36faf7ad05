"""Trains an answer head on the GPU: the norm in front of the vocabulary projection,
the projection's cross entropy with its gradients, and the AdamW step that updates
both, over a stream of hidden states and their next tokens.

The hidden states stand for a frozen model's last layer: each is the direction of
the token to come, among noise, through a channel-wise gain that the norm's weight
can learn to undo. A tenth of the rows are prompt tokens and carry no loss.

    python examples/train_head.py --steps 50 --vocab 32003 --dim 1152 --rows 1024
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from gemmaedge_amd import head as H  # noqa: E402


def batches(rows, dim, vocab, seed=1, device="cuda"):
    """Endless (hidden, targets): bfloat16 [rows, dim] and int32 [rows]."""
    gen = torch.Generator(device=device).manual_seed(seed)
    directions = torch.randn(vocab, dim, generator=gen, device=device)
    gain = torch.exp(torch.randn(dim, generator=gen, device=device))
    while True:
        targets = torch.randint(vocab, (rows,), generator=gen, device=device)
        noise = torch.randn(rows, dim, generator=gen, device=device)
        hidden = ((directions[targets] + 0.5 * noise) * gain).bfloat16()
        prompt = torch.rand(rows, generator=gen, device=device) < 0.1
        yield hidden, torch.where(prompt, -1, targets).int()


def train(steps=50, rows=1024, dim=1152, vocab=32003, softcap=30.0, lr=2e-3, state_bits=32, seed=1, log=None):
    """Runs the loop and returns the mean loss of each step."""
    norm_weight = torch.ones(dim, device="cuda")
    weight = (torch.randn(vocab, dim, device="cuda") * 0.02).bfloat16()
    master = weight.float()
    grads = [torch.zeros_like(norm_weight), torch.zeros_like(weight)]
    adamw = H.AdamW([norm_weight, weight], grads, masters=[None, master], lr=lr, weight_decay=0.0, state_bits=state_bits)
    losses = []
    with H.Head(rows, dim, vocab, dtype=torch.bfloat16, train=True) as head:
        source = batches(rows, dim, vocab, seed)
        for step in range(steps):
            hidden, targets = next(source)
            kept = (targets >= 0).sum()
            y, _, rstd = head.norm(hidden, norm_weight, center=False)
            loss, lse = head.loss(y, weight, targets, softcap=softcap)
            each = (1.0 / kept).expand(rows).contiguous()  # the objective is the mean over the rows with a loss
            dy, _ = head.loss_backward(each, y, weight, targets, lse, softcap=softcap, dweight=grads[1])
            head.norm_backward(dy, hidden, norm_weight, None, rstd, dweight=grads[0], need_input=False)
            adamw.step()
            losses.append(loss.sum() / kept)
            if log and step % 10 == 0:
                log(f"step {step}: loss {float(losses[-1]):.4f}")
        losses = torch.stack(losses).tolist()
    if log:
        log(f"step {steps - 1}: loss {losses[-1]:.4f}")
    return losses


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--steps", type=int, default=50)
    p.add_argument("--rows", type=int, default=1024)
    p.add_argument("--dim", type=int, default=1152)
    p.add_argument("--vocab", type=int, default=32003)
    p.add_argument("--softcap", type=float, default=30.0)
    p.add_argument("--lr", type=float, default=2e-3)
    p.add_argument("--state-bits", type=int, choices=(8, 32), default=32)
    a = p.parse_args()
    train(a.steps, a.rows, a.dim, a.vocab, a.softcap, a.lr, a.state_bits, log=print)


if __name__ == "__main__":
    main()
