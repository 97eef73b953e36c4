"""Trains a transformer's feed-forward block and output layer to follow a
teacher, then serves it in 8 bits.

    python examples/distill_feed_forward.py [--steps 60]

A training step is the library's calls alone:

  norm        MusaAddRmsNorm            h -> n
  up          MusaLinear                n -> a = gelu(n w_up + b_up)
  down        MusaLinear                a -> h2 = a w_down + b_down + h
  norm        MusaAddRmsNorm            h2 -> n2
  logits      MusaLinear                n2 -> l = n2 embedding^T
  loss        MusaTopKDistillation      KL of the teacher's top logits, and dl
  backward    MusaLinearGrad, MusaAddRmsNormGrad
  update      MusaGroupedResourceApplyAdam on float variables

Variables are float; the products use bfloat16 copies of the weights.  The
serving step takes the same block with the norm's output and the weights in 8
bits (MusaAddRmsNormQuantized, MusaLinearQuantized).
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from tensorflow_musa_extension_amd import raw_ops as ops  # noqa: E402

EPS = 1e-5
ACT = "GeluApproximate"
TEMPERATURE = 2.0
TOP = 16


class Block:
    """A feed-forward block of width `width` with a tied output layer of
    `vocab` tokens."""

    def __init__(self, width, inner, vocab, seed, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape, scale):
            return torch.randn(shape, generator=g, device=device) * scale

        self.matrices = {
            "up": normal(width, inner, scale=width ** -0.5),
            "b_up": torch.zeros(inner, device=device),
            "down": normal(inner, width, scale=inner ** -0.5),
            "b_down": torch.zeros(width, device=device),
            "embedding": normal(vocab, width, scale=width ** -0.5),
        }
        self.gammas = {"norm1": torch.ones(width, device=device),
                       "norm2": torch.ones(width, device=device)}
        self.half = {k: v.bfloat16() for k, v in self.matrices.items()}
        self.state = {k: (torch.zeros_like(v), torch.zeros_like(v))
                      for k, v in {**self.matrices, **self.gammas}.items()}
        self.steps = 0

    def forward(self, h):
        """Logits of h [tokens, width] and what the backward pass needs."""
        w, s = self.half, {"h": h}
        s["n1"] = ops.MusaAddRmsNorm(h, self.gammas["norm1"], epsilon=EPS)
        s["up"] = ops.MusaLinear(s["n1"].y, w["up"], bias=w["b_up"], activation=ACT,
                                 keep_pre_activation=True)
        s["down"] = ops.MusaLinear(s["up"].y, w["down"], bias=w["b_down"], residual=h).y
        s["n2"] = ops.MusaAddRmsNorm(s["down"], self.gammas["norm2"], epsilon=EPS)
        return ops.MusaLinear(s["n2"].y, w["embedding"], transpose_b=True).y, s

    def backward(self, dlogits, s):
        """Gradients of all variables, by name."""
        w = self.half
        out = ops.MusaLinearGrad(dlogits, s["n2"].y, w["embedding"], transpose_b=True,
                                 has_bias=False)
        n2 = ops.MusaAddRmsNormGrad(out.x_backprop, s["down"], self.gammas["norm2"], s["n2"].rstd)
        down = ops.MusaLinearGrad(n2.x_backprop, s["up"].y, w["down"])
        up = ops.MusaLinearGrad(down.x_backprop, s["n1"].y, w["up"],
                                pre_activation=s["up"].pre_activation, activation=ACT)
        # The residual path brings n2's gradient to h; h is the input here.
        n1 = ops.MusaAddRmsNormGrad(up.x_backprop, s["h"], self.gammas["norm1"], s["n1"].rstd,
                                    sum_backprop=n2.x_backprop)
        return {"up": up.weight_backprop, "b_up": up.bias_backprop, "down": down.weight_backprop,
                "b_down": down.bias_backprop, "embedding": out.weight_backprop,
                "norm1": n1.gamma_backprop, "norm2": n2.gamma_backprop, "h": n1.x_backprop}

    def update(self, grads, lr):
        """One Adam step: float variables, bfloat16 gradients (the norms'
        are float)."""
        self.steps += 1
        for names in (list(self.matrices), list(self.gammas)):
            var = {**self.matrices, **self.gammas}
            ops.MusaGroupedResourceApplyAdam(
                [var[n] for n in names], [self.state[n][0] for n in names],
                [self.state[n][1] for n in names], [grads[n] for n in names],
                0.9 ** self.steps, 0.999 ** self.steps, lr, 0.9, 0.999, 1e-8)
        for n, v in self.matrices.items():
            self.half[n].copy_(v)

    def quantized(self):
        """The weights that take a norm's 8-bit output, for serving: e4m3 rows
        [outputs, inputs] and scales."""
        packed = {}
        for name in ("up", "embedding"):
            rows = self.matrices[name] if name == "embedding" else self.matrices[name].t()
            scale = rows.abs().amax(1) / 448
            packed[name] = ((rows / scale[:, None]).to(torch.float8_e4m3fn).contiguous(), scale)
        return packed

    def serve(self, h, packed):
        """Logits of h with 8-bit norms and weights; the inner activation
        stays bfloat16."""
        n1 = ops.MusaAddRmsNormQuantized(h, self.gammas["norm1"], epsilon=EPS)
        up = ops.MusaLinearQuantized(n1.y, n1.scale, *packed["up"], bias=self.half["b_up"],
                                     activation=ACT)
        down = ops.MusaLinear(up, self.half["down"], bias=self.half["b_down"])
        n2 = ops.MusaAddRmsNormQuantized(down.y, self.gammas["norm2"], residual=h, epsilon=EPS)
        return ops.MusaLinearQuantized(n2.y, n2.scale, *packed["embedding"])


def train(steps=60, tokens=512, width=256, inner=1024, vocab=1000, lr=3e-3, seed=0):
    """Trains a student on a teacher of the same shape; returns (losses,
    student, teacher, the last batch)."""
    teacher = Block(width, inner, vocab, seed + 1)
    student = Block(width, inner, vocab, seed + 2)
    g = torch.Generator(device="cuda").manual_seed(seed + 3)
    weights = torch.full((tokens,), 1.0 / tokens, device="cuda")
    losses = []
    for _ in range(steps):
        h = torch.randn((tokens, width), generator=g, device="cuda").bfloat16()
        top = torch.topk(teacher.forward(h)[0].float(), TOP, dim=1)
        logits, saved = student.forward(h)
        loss = ops.MusaTopKDistillation(logits, top.indices, top.values, row_weights=weights,
                                        temperature=TEMPERATURE)
        student.update(student.backward(loss.backprop, saved), lr)
        losses.append(loss.loss.sum())
    return [float(v) for v in losses], student, teacher, h


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--steps", type=int, default=60)
    args = p.parse_args()
    losses, student, _, h = train(args.steps)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.4f}")
    print(f"step {len(losses) - 1:4d}  loss {losses[-1]:.4f}")
    full = student.forward(h)[0].float()
    low = student.serve(h, student.quantized()).float()
    print(f"served in 8 bits: logits off by {float((low - full).norm() / full.norm()):.3f}, "
          f"the first choice kept for {float((low.argmax(1) == full.argmax(1)).float().mean()):.1%}")


if __name__ == "__main__":
    main()
