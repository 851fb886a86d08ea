"""A training step on packed sequences: a small mixture-of-experts decoder with mHC connections.

    python examples/train_packed_moe.py [--steps 20] [--state-bits 8]

Documents of different lengths lie back to back in one row of tokens.  Every sublayer is wrapped in an mHC connection
(``MHCConnection_Fused``); attention sees a token's own document only (``packed_attention``), the router hands out
weights, experts, counts and the balance loss in one pass (``route_topk``), and the optimizer step scales the gradients
to norm 1 and keeps its moments in 32 or 8 bits (``AdamW``).  Synthetic tokens; prints the loss.
"""

import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minimind-mhc_b200"))

from model.mhc_adamw import AdamW  # noqa: E402
from model.mhc_attention import packed_attention  # noqa: E402
from model.mhc_common import MHCHead, StreamExpand  # noqa: E402
from model.mhc_fused import MHCConnection_Fused  # noqa: E402
from model.mhc_router import route_topk  # noqa: E402


class Attention(nn.Module):
    def __init__(self, dim, heads, kv_heads):
        super().__init__()
        self.heads, self.kv_heads, self.hd = heads, kv_heads, dim // heads
        self.qkv = nn.Linear(dim, (heads + 2 * kv_heads) * self.hd, bias=False)
        self.out = nn.Linear(dim, dim, bias=False)

    def forward(self, x, cu):
        t = x.shape[0]
        # q, k and v are slices of one projection's output: read in place
        q, k, v = self.qkv(x).view(t, -1, self.hd).split((self.heads, self.kv_heads, self.kv_heads), 1)
        return self.out(packed_attention(q, k, v, cu).reshape(t, -1))


class MoE(nn.Module):
    def __init__(self, dim, inter, experts, k, aux_coef=5e-4):
        super().__init__()
        self.k, self.aux_coef = k, aux_coef
        self.gate = nn.Linear(dim, experts, bias=False)
        self.up = nn.ParameterList(nn.Parameter(torch.randn(dim, inter) * dim ** -0.5) for _ in range(experts))
        self.down = nn.ParameterList(nn.Parameter(torch.randn(inter, dim) * inter ** -0.5) for _ in range(experts))

    def forward(self, x):
        weights, experts, counts, self.aux_loss = route_topk(self.gate(x), self.k, self.aux_coef)
        order = experts.flatten().argsort(stable=True)
        token = order // self.k
        rows = x[token].split(counts.tolist())
        y = torch.cat([F.silu(r @ u) @ d for r, u, d in zip(rows, self.up, self.down)])
        y = y * weights.flatten()[order].unsqueeze(1).to(y.dtype)
        return torch.zeros_like(x).index_add(0, token, y)


class Decoder(nn.Module):
    def __init__(self, vocab=512, dim=256, layers=2, heads=4, kv_heads=2, inter=256, experts=8, k=2, streams=4):
        super().__init__()
        self.embed = nn.Embedding(vocab, dim)
        self.expand = StreamExpand(streams, dim)
        self.layers = nn.ModuleList()
        for _ in range(layers):
            self.layers.append(nn.ModuleDict(dict(
                norm1=nn.RMSNorm(dim), attn=Attention(dim, heads, kv_heads), mhc1=MHCConnection_Fused(streams, dim),
                norm2=nn.RMSNorm(dim), moe=MoE(dim, inter, experts, k), mhc2=MHCConnection_Fused(streams, dim))))
        self.head = MHCHead(streams, dim)
        self.lm_head = nn.Linear(dim, vocab, bias=False)

    def forward(self, ids, cu):
        """ids (T,), cu (documents + 1,) int32: logits (T, vocab)"""
        h = self.expand(self.embed(ids)[None])
        for m in self.layers:
            h = m["mhc1"](h, lambda z, m=m: m["attn"](m["norm1"](z)[0], cu)[None])
            h = m["mhc2"](h, lambda z, m=m: m["moe"](m["norm2"](z)[0])[None])
        return self.lm_head(self.head(h)[0])

    def aux_loss(self):
        return sum(m["moe"].aux_loss for m in self.layers)


def make_batch(vocab, lengths, seed, device="cuda"):
    """Documents that count upwards from a random token: what comes next can be learnt."""
    g = torch.Generator().manual_seed(seed)
    docs = [(torch.randint(vocab, (1,), generator=g) + torch.arange(n + 1)) % vocab for n in lengths]
    ids = torch.cat([d[:-1] for d in docs]).to(device)
    labels = torch.cat([d[1:] for d in docs]).to(device)
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(device)
    return ids, labels, cu


def train(steps, state_bits=32, seed=0, lengths=(300, 1, 77, 512, 134)):
    torch.manual_seed(seed)
    model = Decoder().cuda().bfloat16()
    for m in model.modules():  # coefficient math stays in fp32
        if isinstance(m, (MHCConnection_Fused, MHCHead)):
            m.float()
    opt = AdamW(model.parameters(), lr=2e-3, state_bits=state_bits, max_grad_norm=1.0)
    losses = []
    for step in range(steps):
        ids, labels, cu = make_batch(512, list(lengths), seed * 1000 + step)
        loss = F.cross_entropy(model(ids, cu).float(), labels)
        (loss + model.aux_loss()).backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    a = ap.parse_args()
    for i, v in enumerate(train(a.steps, a.state_bits)):
        print(f"step {i:3d}  loss {v:.4f}")
