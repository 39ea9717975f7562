"""Recovering what quantisation costs: a frozen, ABFT-protected low-precision
model learns per-task low-rank adapters from its unquantised teacher's top
logits, and then decodes requests of all tasks in one batch.

The student shares the teacher's weights. Every projection of it runs as a
``ProtectedLinear`` (FP8 or NVFP4, checksums on) with adapters beside it;
queries and keys are normed per head and turned by position in one pass; the
loss compares the student's logits with the teacher's top 32.

    python examples/distill_adapters.py [--precision nvfp4] [--steps 30]
"""
import argparse
import sys
from pathlib import Path

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from sdc_b200.gemm.linear import ProtectedLinear, install  # noqa: E402
from sdc_b200.layers import (AdapterBatch, distillation_loss, distillation_loss_and_grad, head_norm_rotary,  # noqa: E402
                             low_rank_adapters, low_rank_adapters_, rotary_table)

DTYPE = torch.bfloat16


class Adapted(nn.Module):
    """A frozen projection and one low-rank adapter a task beside it."""

    def __init__(self, projection, tasks, rank):
        super().__init__()
        self.projection = projection
        n, k = projection.weight.shape
        self.a = nn.Parameter(torch.randn(tasks, rank, k, dtype=DTYPE, device=projection.weight.device) * k ** -0.5)
        self.b = nn.Parameter(torch.zeros(tasks, n, rank, dtype=DTYPE, device=projection.weight.device))
        self.batch = None  # set for every batch by adapt()

    def forward(self, x):
        base = self.projection(x)
        if torch.is_grad_enabled():
            return low_rank_adapters(base, x, self.a, self.b, self.batch)
        return low_rank_adapters_(base, x, self.a, self.b, self.batch)


class Block(nn.Module):
    def __init__(self, hidden, inner, heads, kv_heads):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, hidden // heads
        self.qkv = nn.Linear(hidden, (heads + 2 * kv_heads) * self.dim, bias=False)
        self.o = nn.Linear(hidden, hidden, bias=False)
        self.gate_up = nn.Linear(hidden, 2 * inner, bias=False)
        self.down = nn.Linear(inner, hidden, bias=False)
        self.norm1, self.norm2 = nn.RMSNorm(hidden), nn.RMSNorm(hidden)
        self.q_norm, self.k_norm = nn.Parameter(torch.ones(self.dim)), nn.Parameter(torch.ones(self.dim))

    def forward(self, x, table, positions, cache):
        batch, sequence, hidden = x.shape
        qkv = self.qkv(self.norm1(x).view(-1, hidden)).view(batch, sequence, -1, self.dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 2)  # views: the norm reads them in place
        q, k = head_norm_rotary(q, k, table, positions, self.q_norm.to(DTYPE), self.k_norm.to(DTYPE))
        if cache is not None:
            k, v = (torch.cat(pair, 1) for pair in zip(cache.get(self, (k[:, :0], v[:, :0])), (k, v)))
            cache[self] = k, v
        y = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2),
                                           is_causal=sequence > 1, enable_gqa=True)
        x = x + self.o(y.transpose(1, 2).reshape(-1, hidden)).view_as(x)
        gate, up = self.gate_up(self.norm2(x).view(-1, hidden)).chunk(2, -1)
        return x + self.down(F.silu(gate) * up).view_as(x)


class Model(nn.Module):
    def __init__(self, vocab, hidden, inner, layers, heads, kv_heads):
        super().__init__()
        self.embed = nn.Embedding(vocab, hidden)
        self.blocks = nn.ModuleList(Block(hidden, inner, heads, kv_heads) for _ in range(layers))
        self.norm = nn.RMSNorm(hidden)
        self.head = nn.Linear(hidden, vocab, bias=False)

    def forward(self, tokens, table, positions, cache=None):
        x = self.embed(tokens)
        for block in self.blocks:
            x = block(x, table, positions, cache)
        return self.head(self.norm(x).view(-1, x.shape[-1])).view(*tokens.shape, -1)


def student_of(teacher, config, precision, tasks, rank):
    """The teacher's weights, frozen, on protected low-precision GEMMs, with adapters beside every block's projections."""
    student = Model(**config).to(DTYPE).cuda()
    student.load_state_dict(teacher.state_dict())
    student.requires_grad_(False)
    scaling = {"fp8": "tensorwise", "nvfp4": "block16"}[precision]
    abft = {"method": "classic", "implementation": "native", "reference_mode": "input_fused",
            "reference_layout": "kslice", "on_error": "report", "recovery": "none", "locate": True,
            "atol": 0.0, "rtol": 1e-6}
    install(student, precision, scaling, abft_config=abft, report_max_records=100000)
    for block in student.blocks:
        for name in ("qkv", "o", "gate_up", "down"):
            setattr(block, name, Adapted(getattr(block, name), tasks, rank))
    return student


def adapt(student, batch):
    for module in student.modules():
        if isinstance(module, Adapted):
            module.batch = batch


def train(args):
    """Returns (loss before, loss after, detections, protected GEMMs, tokens decoded for every request)."""
    torch.manual_seed(args.seed)
    config = dict(vocab=args.vocab, hidden=args.hidden, inner=2 * args.hidden, layers=args.layers,
                  heads=args.hidden // 64, kv_heads=max(1, args.hidden // 256))
    teacher = Model(**config).to(DTYPE).cuda().requires_grad_(False)
    student = student_of(teacher, config, args.precision, args.tasks, args.rank)
    table = rotary_table(args.sequence + 8, 64, 1e6)
    positions = torch.arange(args.sequence, device="cuda")
    tokens = torch.randint(0, args.vocab, (args.requests, args.sequence), device="cuda")
    requests = [i % args.tasks for i in range(args.requests)]
    adapt(student, AdapterBatch([args.sequence] * args.requests, requests, args.tasks))
    top = teacher(tokens, table, positions).topk(32, -1)
    indices = top.indices.masked_fill(positions[:, None] < 4, -1)  # the first positions are prompt: nothing to learn
    rows = (args.sequence - 4) * args.requests
    scale = torch.full((), 1.0 / rows, device="cuda")
    optimizer = torch.optim.AdamW([p for p in student.parameters() if p.requires_grad], lr=args.lr)
    first = last = None
    for step in range(args.steps):
        optimizer.zero_grad(set_to_none=True)
        logits = student(tokens, table, positions)
        losses, grad = distillation_loss_and_grad(logits.detach(), indices, top.values, grad_loss=scale)
        logits.backward(grad)
        optimizer.step()
        last = losses.sum() * scale
        first = last if first is None else first
        if step % 10 == 0:
            print(f"step {step}: loss {last.item():.4f}")
    with torch.no_grad():
        after = distillation_loss(student(tokens, table, positions), indices, top.values)
        # Decoding: one token a request, each with its task's adapter.
        cache = {}
        chosen = student(tokens, table, positions, cache)[:, -1:].argmax(-1)
        adapt(student, AdapterBatch([1] * args.requests, requests, args.tasks))
        decoded = [chosen]
        for i in range(3):
            at = torch.tensor([args.sequence + i], device="cuda")
            decoded.append(student(decoded[-1], table, at, cache)[:, -1:].argmax(-1))
    protection = next(m.protection for m in student.modules() if isinstance(m, ProtectedLinear))
    detections = sum(bool(report.detected) for report in protection.reports)
    return first.item(), after.item(), detections, protection.call_index, torch.cat(decoded, 1)


def parser():
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--precision", choices=["fp8", "nvfp4"], default="nvfp4")
    p.add_argument("--steps", type=int, default=30)
    p.add_argument("--requests", type=int, default=8)
    p.add_argument("--sequence", type=int, default=128)
    p.add_argument("--tasks", type=int, default=2)
    p.add_argument("--rank", type=int, default=16)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--hidden", type=int, default=512)
    p.add_argument("--vocab", type=int, default=8192)
    p.add_argument("--lr", type=float, default=2e-3)
    p.add_argument("--seed", type=int, default=0)
    return p


def main():
    before, after, detections, gemms, decoded = train(parser().parse_args())
    print(f"loss {before:.4f} -> {after:.4f}; {detections} detections in {gemms} protected GEMMs")
    print("decoded:", decoded.tolist())


if __name__ == "__main__":
    main()
