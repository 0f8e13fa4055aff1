"""Trains a language model's output head from a larger model's top logits, then serves it in 8-bit integers.

The head is layer norm and a projection onto the vocabulary.  Hidden states and the teacher are random here
(a fixed projection of the same states); a program with a model of its own has both from there.

    python examples/lm_head.py [--tokens 512] [--width 256] [--vocab 4096] [--top 32] [--steps 40]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import zpu_b200 as zc  # noqa: E402


class Head:
    def __init__(self, width, vocab, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.gamma = torch.ones(width, device="cuda")
        self.beta = torch.zeros(width, device="cuda")
        self.weight = torch.randn(vocab, width, generator=g, device="cuda") / width ** 0.5

    def value_and_grad(self, x, teacher, indices, temperature):
        """The mean distillation loss of the states x and its gradients (x, gamma, beta, weight)."""
        rows = x.shape[0]
        h, mean, rstd = zc.layer_norm(x, self.gamma, self.beta, stats=True)
        logits = zc.gemm(h, self.weight, trans_b=True)
        each = torch.full((rows,), 1.0 / rows, device="cuda")
        loss, dlogits = zc.distill_value_and_grad(logits, teacher, indices, each, temperature, out=logits)
        dweight = zc.gemm(dlogits, h, trans_a=True)
        dx, dgamma, dbeta = zc.layer_norm_grad(zc.gemm(dlogits, self.weight), x, mean, rstd, self.gamma)
        return loss.mean(), (dx, dgamma, dbeta, dweight)

    def step(self, x, teacher, indices, temperature, rate):
        loss, (_, dgamma, dbeta, dweight) = self.value_and_grad(x, teacher, indices, temperature)
        self.gamma -= rate * dgamma
        self.beta -= rate * dbeta
        self.weight -= rate * dweight
        return loss


class Server:
    """The trained head with int8 weights: states in, tokens out."""

    def __init__(self, head):
        self.gamma, self.beta = head.gamma, head.beta
        self.project = zc.Int8Linear.from_float(head.weight)

    def next_tokens(self, x, uniform, **rules):
        return zc.sample(self.project(zc.layer_norm(x, self.gamma, self.beta)), uniform, **rules)


def main(argv=None):
    p = argparse.ArgumentParser()
    for name, value in (("tokens", 512), ("width", 256), ("vocab", 4096), ("top", 32), ("steps", 40)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args(argv)
    zc.check(zc.lib().zpucuda_init(torch.cuda.current_device()))
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(a.tokens, a.width, generator=g, device="cuda")
    teacher = 4 * zc.gemm(x, torch.randn(a.width, a.vocab, generator=g, device="cuda")) / a.width ** 0.5
    values, indices = teacher.topk(a.top, 1)
    head = Head(a.width, a.vocab)
    losses = [head.step(x, values, indices, 2.0, 3.0) for _ in range(a.steps)]
    losses = torch.stack(losses).tolist()
    print("distillation loss: %.4f -> %.4f in %d steps" % (losses[0], losses[-1], a.steps))
    server = Server(head)
    uniform = zc.rng_uniform(0x5EED, a.tokens)
    best, _ = server.next_tokens(x, uniform, temperature=0.0)
    drawn, logprob = server.next_tokens(x, uniform, temperature=0.8, top_k=40, top_p=0.95, min_p=0.02)
    agree = float((best[:, None] == indices).any(1).float().mean())
    print("the likeliest token is among the teacher's %d for %.1f %% of the states; mean log probability of the drawn "
          "tokens %.3f" % (a.top, 100 * agree, float(logprob.mean())))
    return losses, agree, drawn, logprob


if __name__ == "__main__":
    main()
