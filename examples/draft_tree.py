"""One step of drafted-tree decoding, and one training step, of a layer's attention.

    python -m examples.draft_tree

Serving: the drafted tokens' raw K=V rows and queries go through one launch that
norms them, turns them by their depth in the tree and writes the rows into the
paged cache (``append_shared_kv``); ``tree_attn_sharedkv`` attends over their
ancestors, the window and the compressed cache; ``head_norm_rope`` without the
norm turns the output back (the cache's rows are turned, and are the values
too). Once a path of the tree is accepted, its raw rows are appended again, at
the slots of a chain. What the tree gave for the path is then what
``sparse_attn_sharedkv`` gives for that chain with the same lists. They hold cached
rows alone: a compressed row that ends among the drafted tokens is the chain's to
see, once it is written, and not the tree's.

Training: the same layer on a chain, with the gradients of its raw rows, its
queries and the norms' weights.
"""

from __future__ import annotations

import torch

from dsv4_b200 import (
    append_shared_kv,
    append_shared_kv_backward,
    check_device_status,
    head_norm_rope,
    head_norm_rope_backward,
    sparse_attn_sharedkv,
    sparse_attn_sharedkv_backward,
    tree_attn_sharedkv,
)

D, ROPE, RATIO, WIN = 512, 64, 4, 127


class Layer:
    """A layer's caches, norms and position tables, for requests of the given cached lengths."""

    def __init__(self, cached, heads=64, page=64, topk=256, dtype=torch.bfloat16, room=64, seed=0, device="cuda"):
        g = torch.Generator(device).manual_seed(seed)
        self.dev, self.heads, self.topk, self.dtype, self.g = torch.device(device), heads, topk, dtype, g
        self.cached = torch.tensor(cached, dtype=torch.int32, device=device)
        B = len(cached)
        self.ori, self.obt = self.pool(max(cached) + room, page, B)
        self.cmp, self.cbt = self.pool(max((max(cached) + room) // RATIO, 1), page, B)
        angle = torch.arange(max(cached) + room)[:, None] * 10000.0 ** (-torch.arange(0, ROPE, 2) / ROPE)
        self.rope = dict(cos=angle.cos().to(device), sin=angle.sin().to(device))
        self.q_weight, self.kv_weight = (1 + 0.1 * self.rand(D) for _ in range(2))
        self.sinks = self.rand(heads)

    def rand(self, *shape):
        return torch.randn(shape, generator=self.g, device=self.dev)

    def pool(self, length, page, B):
        n = -(-length // page)
        table = torch.randperm(B * n, generator=self.g, device=self.dev).to(torch.int32).view(B, n)
        return self.rand(B * n, page, 1, D).to(self.dtype), table

    def lists(self, n):
        """Top-k lists of n tokens of every request: random rows of the cached context here,
        an indexer's in a model."""
        out = torch.full((len(self.cached) * n, 1, self.topk), -1, dtype=torch.int32, device=self.dev)
        for b, c in enumerate(self.cached.tolist()):
            for i in range(n):
                ids = torch.randperm(c // RATIO, generator=self.g, device=self.dev)[: self.topk]
                out[b * n + i, 0, : len(ids)] = ids.to(torch.int32)
        return out

    def append(self, kv, cu, used, **kw):
        return append_shared_kv(kv, self.ori, ori_block_table=self.obt, seqused_kv=used, cu_seqlens_q=cu,
                                weight=self.kv_weight, **self.rope, **kw)

    def attention(self, cu, used, idx):
        return dict(ori_kv=self.ori, ori_block_table=self.obt, cmp_kv=self.cmp, cmp_block_table=self.cbt,
                    cmp_sparse_indices=idx, cu_seqlens_q=cu, seqused_kv=used, sinks=self.sinks, softmax_scale=D ** -0.5,
                    cmp_ratio=RATIO)

    def verify(self, q, kv, parents, depth, cu, idx):
        """Attention of drafted tokens: raw queries and rows in, outputs before the projection out."""
        used = self.cached + cu.diff()
        positions = depth + torch.repeat_interleave(self.cached, cu.diff())
        _, q = self.append(kv, cu, used, q=q, q_weight=self.q_weight, positions=positions)
        out = tree_attn_sharedkv(q, tree_parents=parents, **self.attention(cu, used, idx))
        return head_norm_rope(out, positions=positions, **self.rope, norm=False, inverse=True, q_out=out)

    def accept(self, kv, cu):
        """The accepted tokens' rows at the slots of a chain; the rest of the tree is overwritten later."""
        used = self.cached + cu.diff()
        self.append(kv, cu, used)
        return used

    def chain(self, q, kv, cu, idx):
        """The layer on a chain of new tokens."""
        used = self.cached + cu.diff()
        positions = torch.cat([torch.arange(int(u - n), int(u)) for u, n in zip(used, cu.diff())]).to(self.dev)
        _, q = self.append(kv, cu, used, q=q, q_weight=self.q_weight)
        out, lse = sparse_attn_sharedkv(q, return_softmax_lse=True, **self.attention(cu, used, idx))
        return head_norm_rope(out, positions=positions, **self.rope, norm=False, inverse=True), (q, out, lse, positions, used)

    def chain_backward(self, dout, q_raw, kv, cu, idx, saved):
        """Gradients of the raw queries and rows, the two norms' weights and the sinks."""
        q, out, lse, positions, used = saved
        dout = head_norm_rope_backward(dout, out, positions=positions, **self.rope, norm=False, inverse=True)[0]
        dq, d_ori, _, d_sinks = sparse_attn_sharedkv_backward(dout, q, out, lse, **self.attention(cu, used, idx))
        dq, _, dqw, _ = head_norm_rope_backward(dq, q_raw, positions=positions, **self.rope, q_weight=self.q_weight)
        dkv, dkw = append_shared_kv_backward(d_ori, kv, ori_block_table=self.obt, seqused_kv=used, cu_seqlens_q=cu,
                                             weight=self.kv_weight, **self.rope)
        return dq, dkv, dqw, dkw, d_sinks


# Three branches below the cached context; the longest path is tokens 0, 2, 4, 6.
TREE = [-1, -1, 0, 0, 2, 2, 4, 1]
PATH = [0, 2, 4, 6]


def decode(layer):
    """Verifies TREE for every request, accepts PATH and decodes it as a chain: outputs of both,
    and what the chain used."""
    B, n, m = len(layer.cached), len(TREE), len(PATH)
    depth = [0] * n
    for i, p in enumerate(TREE):
        depth[i] = 0 if p < 0 else depth[p] + 1
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=layer.dev)  # noqa: E731
    q, kv = layer.rand(B * n, layer.heads, D).to(layer.dtype), layer.rand(B * n, 1, D).to(layer.dtype)
    idx = layer.lists(n)
    tree = layer.verify(q, kv, ints(TREE * B), ints(depth * B), ints([n * b for b in range(B + 1)]), idx)
    path = torch.tensor([n * b + i for b in range(B) for i in PATH], device=layer.dev)
    cu = ints([m * b for b in range(B + 1)])
    layer.accept(kv[path], cu)
    chain, saved = layer.chain(q[path], kv[path], cu, idx[path])
    return tree[path], chain, idx[path], saved


def train(layer, n=24):
    B = len(layer.cached)
    q, kv = layer.rand(B * n, layer.heads, D).to(layer.dtype), layer.rand(B * n, 1, D).to(layer.dtype)
    cu = torch.tensor([n * b for b in range(B + 1)], dtype=torch.int32, device=layer.dev)
    idx = layer.lists(n)
    out, saved = layer.chain(q, kv, cu, idx)
    dout = layer.rand(*out.shape).to(out.dtype)  # a model's loss gives this
    return (q, kv, idx, dout), out, layer.chain_backward(dout, q, kv, cu, idx, saved)


def main():
    layer = Layer([4096, 1000, 32])
    tree, chain, _, _ = decode(layer)
    print(f"drafted tree, accepted path against the chain: largest difference {(tree.float() - chain.float()).abs().max():.2e} "
          f"of {chain.float().abs().max():.2f}")
    _, _, grads = train(Layer([512, 100], seed=1))
    names = ("queries", "rows", "query norm", "row norm", "sinks")
    print("training step, gradient norms: " + ", ".join(f"{n} {g.float().norm():.3g}" for n, g in zip(names, grads)))
    check_device_status()


if __name__ == "__main__":
    main()
