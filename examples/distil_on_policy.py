"""On-policy distillation of a small student from a FULL-arm teacher, all at the vocabulary end on libsdm_b200.

Each step the student continues a few prompts (sample_logits under a repetition penalty and a mask of allowed tokens),
the teacher (an OneSdmLM) scores what was written and hands over its top logits, and the student learns from them:
distill_loss and its gradient, and the token table's gradient, which comes both from the tied head and from the lookup
(embed_tokens).  The student's body is plain torch, here a perceptron over the last three tokens.

    python examples/distil_on_policy.py --steps 30
"""
import argparse
import math
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import sdmchat_b200 as S  # noqa: E402


class Student(nn.Module):
    """Tied token table and a perceptron over the embeddings of a position and the two before it."""

    def __init__(self, V, d, width):
        super().__init__()
        self.table = nn.Parameter(torch.randn(V, d) * 0.02)
        self.scale = math.sqrt(d)
        self.up = nn.Linear(3 * d, width)
        self.down = nn.Linear(width, d)

    def forward(self, ids):
        """Logits (B * T, V) of ids (B, T)."""
        e = S.embed_tokens(ids, self.table, scale=self.scale)
        back = [F.pad(e, (0, 0, k, 0))[:, : e.shape[1]] for k in (1, 2)]
        h = e + self.down(F.silu(self.up(torch.cat([e, *back], -1))))
        h = F.rms_norm(h, h.shape[-1:])
        return h.reshape(-1, h.shape[-1]) @ self.table.t()


@torch.no_grad()
def roll_out(student, prompt, steps, mask, g):
    """The student's own continuation (B, T + steps) of prompt (B, T)."""
    B, T = prompt.shape
    text = torch.full((B, T + steps), -1, dtype=torch.int32, device=prompt.device)
    text[:, :T] = prompt
    for t in range(T, T + steps):
        logits = student(text[:, max(0, t - 3):t].contiguous()).view(B, -1, student.table.shape[0])[:, -1]
        rules = S.LogitRules(history=text[:, :t].contiguous(), prompt_len=torch.full((B,), T, device=prompt.device),
                             repetition=1.2, mask=mask)
        u = torch.rand(B, generator=g, device=prompt.device)
        text[:, t] = S.sample_logits(logits, rules, u=u, temperature=0.9, top_k=50, top_p=0.95)[0]
    return text


def main(argv=None):
    a = argparse.ArgumentParser()
    a.add_argument("--steps", type=int, default=30)
    a.add_argument("--vocab", type=int, default=4096)
    a.add_argument("--d", type=int, default=256)
    a.add_argument("--layers", type=int, default=2)
    a.add_argument("--batch", type=int, default=16)
    a.add_argument("--prompt", type=int, default=32)
    a.add_argument("--new", type=int, default=32)
    a.add_argument("--top", type=int, default=32, help="teacher logits per position")
    a.add_argument("--temperature", type=float, default=2.0)
    a.add_argument("--lr", type=float, default=1e-2)
    a = a.parse_args(argv)
    dev = "cuda"
    torch.manual_seed(0)
    g = torch.Generator(device=dev).manual_seed(1)
    teacher = S.build_onesdm("onesdm_allsdm", a.vocab, dict(d=a.d, layers=a.layers, mlp_f=S.mlp_width(a.d), heads=4))
    with torch.no_grad():
        teacher.emb.weight.mul_(15)  # random weights: give the logits a language model's spread
        for p in teacher.parameters():
            if p.dim() >= 2 and float(p.abs().max()) == 0:
                nn.init.normal_(p, std=0.05)
    teacher = teacher.to_bf16_stream().to(dev)
    student = Student(a.vocab, a.d, 2 * a.d).to(dev)
    opt = torch.optim.Adam(student.parameters(), lr=a.lr)
    allowed = torch.full((1, -(-a.vocab // 32)), -1, dtype=torch.int32, device=dev)
    allowed[0, 0] &= ~1  # token 0 (a document's end) is not to be written
    prompt = torch.randint(1, a.vocab, (a.batch, a.prompt), generator=g, device=dev, dtype=torch.int32)
    losses = []
    for step in range(a.steps):
        text = roll_out(student, prompt, a.new, allowed, g)
        with torch.no_grad():
            scores = teacher(text).float().flatten(0, 1)
            top = torch.topk(scores, a.top, -1)
            lse = torch.logsumexp(scores / a.temperature, -1)
        loss = S.distill_loss(student(text), top.indices, top.values, temperature=a.temperature, teacher_lse=lse)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
        if step % 5 == 0 or step == a.steps - 1:
            print(f"step {step:3d}  loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    main()
