"""Distils a small language model from a teacher's top logits on the xdna device.

The student embeds the tokens (``lm.embedding``), mixes each position with its
predecessors' mean, passes gated feed-forward blocks (``lm.gated_mlp``) and a
head tied to the embedding (the device's GEMM), and is trained with fused Adam
on ``lm.distill_loss`` against the teacher's largest logits for every position.
Teacher and text are synthetic: a random bigram table whose rows' top entries
are the teacher, and text drawn from it.

    python examples/distill_lm.py [--steps 200] [--graph] [--device cpu]

prints the loss as it falls.  ``--graph`` captures the whole step in a CUDA
graph; ``--device cpu`` runs the operators' plain CPU path.
"""
import argparse
import sys
from pathlib import Path

import torch
import torch.nn as nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "pytorch-xdna2_b200"))
import xdna_train  # noqa: E402
from xdna_train import graphs, lm  # noqa: E402


class Student(nn.Module):
    def __init__(self, vocab: int, width: int, hidden: int, blocks: int):
        super().__init__()
        self.embed = nn.Parameter(torch.randn(vocab, width) * width ** -0.5)
        self.mix = nn.Linear(width, width, bias=False)
        self.blocks = nn.ModuleList(
            nn.ParameterDict({"gate": torch.randn(hidden, width) * width ** -0.5,
                              "up": torch.randn(hidden, width) * width ** -0.5,
                              "down": torch.randn(width, hidden) * hidden ** -0.5}) for _ in range(blocks))
        self.scale = width ** 0.5

    def forward(self, ids):
        batch, length = ids.shape
        h = lm.embedding(ids, self.embed, scale=self.scale)
        # the mean of the tokens so far
        count = torch.arange(1, length + 1, device=h.device, dtype=torch.float32).view(1, length, 1)
        past = (h.float().cumsum(1) / count).to(h.dtype)
        h = h + self.mix(past.reshape(batch * length, -1)).view_as(h)
        for b in self.blocks:
            norm = h * torch.rsqrt(h.float().square().mean(-1, keepdim=True) + 1e-6).to(h.dtype)
            h = h + lm.gated_mlp(norm, b["gate"], b["up"], b["down"])
        return (h.reshape(batch * length, -1) @ self.embed.t()).view(batch, length, -1)


def bigram_teacher(vocab: int, top: int, seed: int = 0):
    """A random next-token table: its rows' ``top`` largest logits and their ids."""
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(vocab, vocab, generator=g) * 2
    values, ids = table.topk(top, dim=1)
    return values, ids.int()


def text(ids_of, values, batch: int, length: int, generator):
    """Sequences drawn from the teacher's own distribution."""
    out = torch.empty(batch, length, dtype=torch.int64)
    out[:, 0] = torch.randint(0, len(ids_of), (batch,), generator=generator)
    for i in range(1, length):
        pick = torch.multinomial(torch.softmax(values[out[:, i - 1]], 1), 1, generator=generator)
        out[:, i] = ids_of[out[:, i - 1]].gather(1, pick).squeeze(1).long()
    return out


def train(steps: int = 200, vocab: int = 512, width: int = 128, hidden: int = 384, blocks: int = 2, top: int = 16,
          batch: int = 16, length: int = 32, device: str = "xdna", graph: bool = False, seed: int = 0, report=None):
    """The loss of every step."""
    values, ids_of = bigram_teacher(vocab, top, seed)
    torch.manual_seed(seed)
    native = torch.device(device).type != "cpu"
    if native:
        torch.cuda.init()  # the ops without an xdna kernel run ATen's CUDA kernels
    model = Student(vocab, width, hidden, blocks).bfloat16().to(device)
    opt = torch.optim.Adam(model.parameters(), lr=3e-3, fused=True, capturable=graph)
    g = torch.Generator().manual_seed(seed + 1)
    # every position predicts the token after it; padding (none here) would have weight 0
    weight = torch.ones(batch, length).to(device)
    tokens = torch.zeros(batch, length, dtype=torch.int64).to(device)
    t_values = torch.zeros(batch, length, top).to(device)
    t_ids = torch.zeros(batch, length, top, dtype=torch.int32).to(device)

    def step():
        opt.zero_grad(set_to_none=True)
        loss = lm.distill_loss(model(tokens), t_values, t_ids, temperature=1.0, row_weight=weight)
        loss.backward()
        opt.step()
        return loss.detach()

    run = None
    losses = []
    for i in range(steps):
        seqs = text(ids_of, values, batch, length, g)
        tokens.copy_(seqs)
        t_values.copy_(values[seqs])
        t_ids.copy_(ids_of[seqs])
        if run is None:
            run = graphs.make_graphed_step(step, warmup=1) if graph and native else step
        losses.append(run().item())
        if report and (i % report == 0 or i == steps - 1):
            print(f"step {i:4d}  loss {losses[-1]:.4f}", flush=True)
    return losses


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--vocab", type=int, default=512)
    ap.add_argument("--width", type=int, default=128)
    ap.add_argument("--hidden", type=int, default=384)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--graph", action="store_true")
    ap.add_argument("--device", default="xdna")
    a = ap.parse_args()
    train(a.steps, a.vocab, a.width, a.hidden, a.blocks, device=a.device, graph=a.graph, report=20)
    if a.device != "cpu":
        print("launches:", {k: v for k, v in xdna_train.kernel_stats().items() if k.startswith("lm.")})


if __name__ == "__main__":
    main()
