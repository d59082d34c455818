"""A small recurrent language model of DNA, trained on a resident cohort's windows and asked for bases one by one.

    python examples/train_recurrent.py COHORT_DIR --steps 200

Everything between the windows and the updated weights that is not a matrix product runs in panvram_amd.ops: each block is
the residual stream's norm, a projection to gate and value, the gated scan over the window and a projection back; the head
and loss come in one call; the gradients are clipped before the update. Windows are packed two to a row here, with a reset
at the second one's first base. (The reference's examples/train_small.py:1-12 trains a convolutional net on such windows.)
"""
import argparse
import math
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import panvram_amd  # noqa: E402
from panvram_amd import ops  # noqa: E402

BASES = "ACGTN"


class Model(torch.nn.Module):
    """Weights in float32, activations in bfloat16."""

    def __init__(self, width=256, depth=2):
        super().__init__()
        p = lambda *s: torch.nn.Parameter(torch.randn(*s) * s[-1] ** -0.5)  # noqa: E731
        self.embed = torch.nn.Parameter(torch.randn(len(BASES), width) * 0.5)
        self.norms = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(width)) for _ in range(depth + 1))
        self.inward = torch.nn.ParameterList(p(2 * width, width) for _ in range(depth))
        self.outward = torch.nn.ParameterList(p(width, width) for _ in range(depth))
        self.head = p(4, width)
        # gates that begin by keeping the state for tens of bases
        self.bias = torch.nn.ParameterList(torch.nn.Parameter(torch.cat([torch.full((width,), -3.0), torch.zeros(width)])) for _ in range(depth))

    def forward(self, tokens, states=None, reset=None):
        """tokens uint8 [B, T] -> (hidden [B, T, width], each block's state after the last token)"""
        stream = F.embedding(tokens.long(), self.embed.bfloat16())
        step, last = None, []
        for k, (inward, outward, bias) in enumerate(zip(self.inward, self.outward, self.bias)):
            y, stream = ops.add_rms_norm(stream, None, self.norms[k]) if step is None else ops.add_rms_norm(step, stream, self.norms[k])
            gate, value = F.linear(y, inward.bfloat16(), bias.bfloat16()).chunk(2, -1)
            h, state = ops.gated_scan(gate, value, state=None if states is None else states[k], reset=reset)
            step = F.linear(h, outward.bfloat16())
            last.append(state)
        return ops.add_rms_norm(step, stream, self.norms[-1])[0], last


def batch(cohort, rows, window, generator):
    """Rows of two windows each, and where the second ones begin"""
    tokens = cohort.sample(2 * rows, window, generator=generator, reverse_complement=0.5, tokens=True, check=False).view(rows, 2 * window)
    reset = torch.zeros(rows, 2 * window, dtype=torch.bool, device=tokens.device)
    reset[:, window] = True
    return tokens, reset


def train(cohort, model, steps, rows=16, window=2048, rate=2e-3, seed=0, tell=None):
    """The loss of each step, in bits per base"""
    generator = torch.Generator(device=cohort.device).manual_seed(seed)
    optimizer = torch.optim.AdamW(model.parameters(), lr=rate, betas=(0.9, 0.98))
    losses = []
    for k in range(steps):
        tokens, reset = batch(cohort, rows, window, generator)
        hidden, _ = model(tokens, reset=reset)
        # a row for each window, so that no window's last place predicts another one's first base
        loss = ops.next_base_loss(hidden.view(2 * rows, window, -1), model.head, tokens.view(2 * rows, window))
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        norm = ops.clip_gradients([p.grad for p in model.parameters()], 1.0)
        optimizer.step()
        losses.append(loss.detach())
        if tell and k % 20 == 0:
            tell(f"step {k}: {float(loss) / math.log(2):.4f} bits a base, gradient norm {float(norm):.3f}")
    return [x / math.log(2) for x in torch.stack(losses).tolist()] if losses else []


@torch.no_grad()
def score(model, tokens):
    """Bits that each next base takes, float32 [B, T]"""
    return ops.next_base_loss(model(tokens)[0], model.head, tokens, reduction="none") / math.log(2)


@torch.no_grad()
def generate(model, prompt, count, generator):
    """`count` bases after each row of `prompt` (uint8 [B, T]), drawn one at a time with the states carried along"""
    hidden, states = model(prompt)
    made = []
    for _ in range(count):
        p = torch.softmax(hidden[:, -1].float() @ model.head.T, -1)
        made.append(torch.multinomial(p, 1, generator=generator).to(torch.uint8))
        hidden, states = model(made[-1], states=states)
    return torch.cat(made, 1)


def main():
    a = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    a.add_argument("cohort", help="directory of archives, with their reference")
    a.add_argument("--dataset", default="q4k")
    a.add_argument("--steps", type=int, default=200)
    a.add_argument("--rows", type=int, default=16)
    a.add_argument("--window", type=int, default=2048)
    a = a.parse_args()
    torch.manual_seed(0)
    cohort = panvram_amd.Cohort.open(a.cohort, device="cuda", dataset=a.dataset)
    model = Model().to(cohort.device)
    train(cohort, model, a.steps, a.rows, a.window, tell=print)
    generator = torch.Generator(device=cohort.device).manual_seed(1)
    prompt = cohort.sample(4, a.window, generator=generator, tokens=True)
    print(f"other windows of the cohort it was trained on: {float(score(model, prompt).mean()):.4f} bits a base")
    for row in generate(model, prompt, 60, generator).tolist():
        print("".join(BASES[b] for b in row))


if __name__ == "__main__":
    main()
