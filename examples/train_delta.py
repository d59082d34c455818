"""A language model of DNA whose layers keep matrices, trained on a resident cohort's windows and asked for bases one by one.

    python examples/train_delta.py COHORT_DIR --steps 200

As examples/train_recurrent.py, with stronger blocks: a layer norm whose residual addition drops some of the block's step, a
projection to queries, keys, values and gates, the gated delta rule over the window and a projection back. Two windows are packed
to a row, with a reset at the second one's first base. One seed on the GPU, counted up once a step, is all that dropout keeps; each
place of the model has a site of its own. (The reference's examples/train_small.py:1-12 trains a convolutional net on such windows.)
"""
import argparse
import math
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import panvram_amd  # noqa: E402
from examples.train_recurrent import BASES, batch  # noqa: E402
from panvram_amd import ops  # noqa: E402


class Model(torch.nn.Module):
    """Weights in float32, activations in bfloat16; `heads` matrices of size x size for each block."""

    def __init__(self, width=256, depth=2, heads=4, size=64, drop=0.1):
        super().__init__()
        p = lambda *s: torch.nn.Parameter(torch.randn(*s) * s[-1] ** -0.5)  # noqa: E731
        self.heads, self.size, self.drop = heads, size, drop
        self.embed = torch.nn.Parameter(torch.randn(len(BASES), width) * 0.5)
        self.norms = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(width)) for _ in range(depth + 1))
        self.shifts = torch.nn.ParameterList(torch.nn.Parameter(torch.zeros(width)) for _ in range(depth + 1))
        self.inward = torch.nn.ParameterList(p(heads * (3 * size + 2), width) for _ in range(depth))
        self.outward = torch.nn.ParameterList(p(width, heads * size) for _ in range(depth))
        self.head = p(4, width)
        # gates that begin by keeping the states for tens to hundreds of bases
        self.keep = torch.nn.ParameterList(torch.nn.Parameter(torch.linspace(-6.0, -3.0, heads)) for _ in range(depth))

    def forward(self, tokens, states=None, reset=None, seed=None):
        """tokens uint8 [B, T] -> (hidden [B, T, width], each block's states after the last token); seed None: nothing is dropped"""
        drop = self.drop if seed is not None else 0.0
        B, T = tokens.shape
        stream = F.embedding(tokens.long(), self.embed.bfloat16())
        if drop:
            stream = ops.dropout(stream, drop, seed)
        step, last = None, []
        for k, (inward, outward, keep) in enumerate(zip(self.inward, self.outward, self.keep)):
            y, stream = self._norm(k, step, stream, drop, seed)
            parts = F.linear(y, inward.bfloat16()).view(B, T, self.heads, 3 * self.size + 2)
            q, key, v, gates = parts.split([self.size, self.size, self.size, 2], -1)
            h, state = ops.gated_delta(q, key, v, gates[..., 0] + keep.bfloat16(), gates[..., 1], state=None if states is None else states[k], reset=reset)
            step = F.linear(h.flatten(2), outward.bfloat16())
            last.append(state)
        return self._norm(len(last), step, stream, drop, seed)[0], last

    def _norm(self, k, step, stream, drop, seed):
        if step is None:
            return ops.add_layer_norm(stream, None, self.norms[k], self.shifts[k])
        return ops.add_layer_norm(step, stream, self.norms[k], self.shifts[k], dropout=drop, seed=seed, site=k)


def train(cohort, model, steps, rows=16, window=2048, rate=2e-3, seed=0, tell=None):
    """The loss of each step, in bits per base"""
    generator = torch.Generator(device=cohort.device).manual_seed(seed)
    drops = torch.randint(1 << 62, (1,), generator=generator, device=cohort.device)
    optimizer = torch.optim.AdamW(model.parameters(), lr=rate, betas=(0.9, 0.98))
    losses = []
    for k in range(steps):
        tokens, reset = batch(cohort, rows, window, generator)
        hidden, _ = model(tokens, reset=reset, seed=drops)
        # a row for each window, so that no window's last place predicts another one's first base
        loss = ops.next_base_loss(hidden.view(2 * rows, window, -1), model.head, tokens.view(2 * rows, window))
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        norm = ops.clip_gradients([p.grad for p in model.parameters()], 1.0)
        optimizer.step()
        drops += 1
        losses.append(loss.detach())
        if tell and k % 20 == 0:
            tell(f"step {k}: {float(loss) / math.log(2):.4f} bits a base, gradient norm {float(norm):.3f}")
    return [x / math.log(2) for x in torch.stack(losses).tolist()] if losses else []


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
    for row in generate(model, prompt, 60, generator).tolist():
        print("".join(BASES[b] for b in row))


if __name__ == "__main__":
    main()
