"""An attention block that trains its head norms, then serves from a quantised
paged cache: a prompt in chunks, single tokens, and a tree of drafted tokens of
which the accepted path is kept.

    PYTHONPATH=. python examples/draft_tree.py [block|mxfp8|nvfp4]

Weights and inputs are random. At the end the cache is read back and the last
step's attention computed from it in plain torch, for comparison.
"""

from __future__ import annotations

import sys

import torch

import breccia_b200 as bb

HEADS, KV_HEADS, DIM, PAGE, PAGES, BATCH = 32, 8, 128, 64, 64, 4
RECIPES = {"block": lambda: bb.Float8BlockScaling(block_k=DIM), "mxfp8": bb.MXFP8BlockScaling,
           "nvfp4": bb.NVFP4BlockScaling}


class Block:
    """Projection, head norm with rotation, cache, attention."""

    def __init__(self, recipe, width=512, positions=4096, device="cuda"):
        g = torch.Generator(device).manual_seed(0)
        self.proj = torch.randn(width, (HEADS + 2 * KV_HEADS) * DIM, generator=g, device=device)
        self.proj = (self.proj * width ** -0.5).bfloat16()
        self.wq = torch.ones(DIM, device=device, requires_grad=True)
        self.wk = torch.ones(DIM, device=device, requires_grad=True)
        angle = torch.arange(positions, device=device)[:, None] * \
            10000.0 ** (-torch.arange(0, DIM, 2, device=device) / DIM)
        self.cos, self.sin = angle.cos(), angle.sin()
        self.cache = bb.QuantizedKVCache(PAGES, PAGE, KV_HEADS, DIM, recipe, device)
        # pages are given out as they come: sequence b's t-th token is in page table[b, t // PAGE]
        self.table = torch.randperm(PAGES, generator=g, device=device).int().view(BATCH, -1)

    def heads(self, x):
        qkv = (x @ self.proj).unflatten(-1, (HEADS + 2 * KV_HEADS, DIM))
        return qkv.split((HEADS, KV_HEADS, KV_HEADS), -2)  # views: the operators read strides

    def train(self, x, positions, lr=1e-2):
        """One step of the norms' weights towards keys that their queries know."""
        q, k, _ = self.heads(x)
        q, k = bb.qk_norm_rope(q, k, self.wq, self.wk, self.cos, self.sin, positions)
        near = q.unflatten(-2, (KV_HEADS, -1)).float() * k.unsqueeze(-2).float()
        loss = -near.sum(-1).mean() * DIM ** -0.5
        loss.backward()
        with torch.no_grad():
            for w in (self.wq, self.wk):
                w -= lr * w.grad
                w.grad = None
        return loss.detach()

    @torch.no_grad()
    def serve(self, x, context, depth, tree=None):
        """``x (batch, n, width)``: the next n tokens of every sequence, or a
        tree of drafted ones, at positions ``context + depth``."""
        n = x.shape[1]
        place = context[:, None] + torch.arange(n, device=x.device)
        slots = self.table.gather(1, place // PAGE) * PAGE + place % PAGE
        q, k, v = self.heads(x)
        q = bb.qk_norm_rope_write(q, k, v, self.wq, self.wk, self.cos, self.sin,
                                  (context[:, None] + depth).flatten(), self.cache, slots.flatten())
        return bb.cache_attention(q, self.cache, self.table, context.int(), tree_mask=tree), q

    @torch.no_grad()
    def keep(self, context, path):
        """The accepted path of a tree moves to the front of its place."""
        for at, node in enumerate(path):
            src, dst = (context + node, context + at)
            a, b = ((self.table.gather(1, (p // PAGE)[:, None])[:, 0].long(), p % PAGE)
                    for p in (src, dst))
            for buf in (self.cache.k_data, self.cache.k_scale, self.cache.v_data, self.cache.v_scale):
                buf[b[0], :, b[1]] = buf[a[0], :, a[1]]
        return context + len(path)


def main(name="mxfp8", device="cuda"):
    torch.manual_seed(1)
    width = 512
    block = Block(RECIPES[name](), width, device=device)
    x, positions = torch.randn(256, width, device=device).bfloat16(), torch.arange(256, device=device)
    losses = [float(block.train(x, positions)) for _ in range(4)]

    context = torch.zeros(BATCH, dtype=torch.int64, device=device)
    for n in (64, 64, 37):  # the prompt, in chunks
        block.serve(torch.randn(BATCH, n, width, device=device).bfloat16(), context,
                    torch.arange(n, device=device))
        context = context + n
    for _ in range(3):  # a token at a time
        out, _ = block.serve(torch.randn(BATCH, 1, width, device=device).bfloat16(), context,
                             torch.zeros(1, dtype=torch.int64, device=device))
        context = context + 1

    # a tree: node i's parent, its depth, and who is an ancestor of whom
    parent = [-1, 0, 0, 1, 1, 2, 3]
    depth, tree = [], torch.eye(len(parent), dtype=torch.bool)
    for i, p in enumerate(parent):
        depth.append(0 if p < 0 else depth[p] + 1)
        if p >= 0:
            tree[i] |= tree[p]
    tree = tree.to(device)
    out, q = block.serve(torch.randn(BATCH, len(parent), width, device=device).bfloat16(), context,
                         torch.tensor(depth, device=device), tree)

    # the same from the cache, read back
    total = int(context[0]) + len(parent)
    k, v = block.cache.read(block.table, context.int() + len(parent), total, torch.float32)
    see = torch.cat([tree.new_ones(len(parent), total - len(parent)), tree], 1)
    s = torch.einsum("bnhgd,bthd->bhgnt", q.unflatten(2, (KV_HEADS, -1)).float(), k) * DIM ** -0.5
    p = s.masked_fill(~see, -torch.inf).softmax(-1)
    want = torch.einsum("bhgnt,bthd->bnhgd", p, v).flatten(2, 3)
    error = float((out.float() - want).norm() / want.norm())

    context = block.keep(context, [0, 1, 4])
    out, _ = block.serve(torch.randn(BATCH, 1, width, device=device).bfloat16(), context,
                         torch.zeros(1, dtype=torch.int64, device=device))
    print(f"{name}: norm losses {losses[0]:.6f} -> {losses[-1]:.6f}; {int(context[0]) + 1} tokens "
          f"cached; tree attention against plain torch: relative difference {error:.1e}")
    return losses, error, out


if __name__ == "__main__":
    main(*sys.argv[1:2])
