"""A student learns from a teacher's top logits, in half precision under the dynamic loss scale.

The operators of the package as a training program uses them, one after another:

* ``norm_rotate_qk`` in every attention layer of teacher and student: norms of queries and keys and the rotation by the position
  (here on three axes, as for frames of a video) in one pass, with its gradient in the student;
* ``top_logits`` on the teacher's output: what is kept of it for the student;
* ``distill_loss`` on the student's, with the loss scale told ahead, so that its gradient comes out of the forward pass at that scale;
* ``engine.backward`` and ``optimizer.step()``: the chunk-wise Adam step on the fp16 gradients.

    python examples/distill_student.py --steps 40
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import patrickstar_amd as ps  # noqa: E402


class Attention(torch.nn.Module):
    """Causal attention with normed, rotated queries and keys.  The products are torch's, in 32 bits."""

    def __init__(self, hidden, heads):
        super().__init__()
        self.heads = heads
        self.qkv = torch.nn.Linear(hidden, 3 * hidden)
        self.out = torch.nn.Linear(hidden, hidden)
        self.q_norm = torch.nn.Parameter(torch.ones(hidden // heads))
        self.k_norm = torch.nn.Parameter(torch.ones(hidden // heads))

    def forward(self, x, positions, plan):
        q, k, v = self.qkv(x).unflatten(-1, (3, self.heads, -1)).unbind(-3)  # views: their strides are the operator's business
        q, k = ps.norm_rotate_qk(q, k, self.q_norm, self.k_norm, positions, plan)
        q, k, v = (t.float().transpose(1, 2) for t in (q, k, v))
        scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) / q.shape[-1] ** 0.5
        later = torch.ones(x.shape[1], x.shape[1], dtype=torch.bool, device=x.device).triu(1)
        mixed = torch.matmul(scores.masked_fill(later, float("-inf")).softmax(-1), v)
        return self.out(mixed.transpose(1, 2).flatten(-2).to(x.dtype))


class Layer(torch.nn.Module):
    def __init__(self, hidden, heads):
        super().__init__()
        self.norm1, self.norm2 = torch.nn.LayerNorm(hidden), torch.nn.LayerNorm(hidden)
        self.attention = Attention(hidden, heads)
        self.up, self.down = torch.nn.Linear(hidden, 4 * hidden), torch.nn.Linear(4 * hidden, hidden)

    def forward(self, x, positions, plan):
        x = x + self.attention(self.norm1(x), positions, plan)
        return x + self.down(torch.nn.functional.gelu(self.up(self.norm2(x))))


class Model(torch.nn.Module):
    def __init__(self, vocab, hidden, heads, layers):
        super().__init__()
        self.embedding = torch.nn.Embedding(vocab, hidden)
        self.layers = torch.nn.ModuleList([Layer(hidden, heads) for _ in range(layers)])
        self.norm = torch.nn.LayerNorm(hidden)
        self.head = torch.nn.Linear(hidden, vocab, bias=False)

    def logits(self, ids, positions, plan):
        x = self.embedding(ids)
        for layer in self.layers:
            x = layer(x, positions, plan)
        return self.head(self.norm(x))

    def forward(self, ids, positions, plan, taught, labels, temperature, grad_scale):
        return ps.distill_loss(self.logits(ids, positions, plan), taught.ids, taught.values, teacher_lse=taught.logsumexp, labels=labels,
                               label_weight=0.1, temperature=temperature, grad_scale=grad_scale)


def places(batch, tokens, width, height):
    """Time, height and width of tokens that are the patches of frames."""
    n = torch.arange(tokens, device="cuda").expand(batch, tokens)
    return torch.stack([n // (width * height), n // width % height, n % width])


def train(steps, vocab=8192, hidden=256, heads=4, tokens=96, batch=8, k=32, temperature=2.0, ahead=True, seed=0, report=lambda step, loss: None):
    """Losses of the steps.  ``ahead``: whether the loss scale is told to the forward pass."""
    torch.manual_seed(seed)
    plan = ps.RotaryPlan(hidden // heads, sections=(8, 12, 12))
    positions = places(batch, tokens, width=6, height=4)
    with torch.device("cuda"):
        teacher = Model(vocab, hidden, heads, 2)
        teacher.head.weight.data.mul_(8)  # an untrained teacher that is sure of something
    teacher = teacher.half().eval().requires_grad_(False)

    def student():
        with torch.device("cuda"):
            return Model(vocab, hidden, heads, 2)

    config = {
        "optimizer": {"type": "AdamW", "params": {"lr": 2e-3, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.01}},
        "fp16": {"enabled": True, "loss_scale": 0, "initial_scale_power": 14, "loss_scale_window": 200},
        "default_chunk_size": 4 << 20,
    }
    engine, optimizer = ps.initialize_engine(student, 0, config)
    losses = []
    ids = torch.randint(vocab, (batch, tokens), device="cuda")
    labels = torch.roll(ids, -1, 1)
    labels[:, -1] = -100  # nothing follows
    with torch.no_grad():
        taught = ps.top_logits(teacher.logits(ids, positions, plan), k, temperature)
    for step in range(steps):
        scale = optimizer.loss_scaler.scale_tensor if ahead else None  # on the device: nobody waits for it
        loss = engine(ids, positions, plan, taught, labels, temperature, scale)
        engine.backward(loss)
        optimizer.step()
        losses.append(loss.detach())
        report(step, losses[-1])
    return torch.stack(losses)


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=40)
    args = parser.parse_args()
    train(args.steps, report=lambda step, loss: print(f"step {step}: loss {float(loss):.4f}", flush=True) if step % 5 == 0 else None)


if __name__ == "__main__":
    main()
