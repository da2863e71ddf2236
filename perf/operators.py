"""What surrounds ``sparse_attn_sharedkv`` in a decoder layer, as measured cases.

Three operators, in the order a layer runs them:

* ``norm_rope``: RMS norm of every query and key head with the position
  rotation of the last dims in the same pass, and its backward;
* ``append``: the same norm and rotation of the new tokens' shared K=V rows,
  written straight into the paged cache (optionally with the queries in the
  same launch), and the backward that reads the cache's gradient;
* ``tree``: attention of drafted tokens that form a tree over the paged
  window and compressed caches, with the per-head sink.

``run`` computes them with elementary torch operations in 32 bits (``own``
false) or through the package's entry points (``own`` true). ``exact`` gives
the definitions in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
DEV = "cuda"


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 64 requests, 64 heads: a few microseconds, so latency counts
        dict(name="norm_rope_decode", op="norm_rope", dtype="bf16", T=64, H=64, Hk=1, D=512, R=64, interleaved=True,
             qw=False, kw=True, P=65536),
        # prefill of two 8192-token prompts
        dict(name="norm_rope_prefill", op="norm_rope", dtype="bf16", T=16384, H=64, Hk=1, D=512, R=64,
             interleaved=True, qw=False, kw=True, P=8192),
        # odd token count, several key heads, the half-split rotation of the whole head, fp16
        dict(name="norm_rope_odd_fp16", op="norm_rope", dtype="fp16", T=1009, H=40, Hk=8, D=128, R=128,
             interleaved=False, qw=True, kw=True, P=4096),
        # the gradient of a training step of 8192 tokens, both weights learned
        dict(name="norm_rope_backward", op="norm_rope_bwd", dtype="bf16", T=8192, H=64, Hk=1, D=512, R=64,
             interleaved=True, qw=True, kw=True, P=8192),
        # one decode step of 512 requests: 512 cache rows, and their 128 query heads in the same call
        dict(name="append_decode", op="append", dtype="bf16", B=512, n=1, ctx_lo=65, ctx_hi=512, bs=128, D=512, R=64,
             interleaved=True, kw=True, H=128, tree=False, layout="TND"),
        # the cache rows of two 8192-token prompts
        dict(name="append_prefill", op="append", dtype="bf16", B=2, n=8192, ctx_lo=0, ctx_hi=0, bs=128, D=512, R=64,
             interleaved=True, kw=True, H=0, tree=False, layout="TND"),
        # up to 16 drafted tokens for each of 128 requests, rotated by their depth in the tree
        dict(name="append_drafts", op="append", dtype="fp16", B=128, n=16, ctx_lo=100, ctx_hi=700, bs=64, D=512, R=64,
             interleaved=True, kw=True, H=64, tree=True, layout="TND"),
        # the gradient of the raw rows of two 4096-token training sequences out of the paged cache's gradient
        dict(name="append_backward", op="append_bwd", dtype="bf16", B=2, n=4096, ctx_lo=0, ctx_hi=0, bs=128, D=512,
             R=64, interleaved=True, kw=True, H=0, tree=False, layout="TND"),
        # four requests, one token each, 16 heads: the smallest decode step
        dict(name="tree_single", op="tree", dtype="bf16", scenario=3, B=4, n=1, H=16, K=256, ratio=4, win=127,
             ctx_lo=1024, ctx_hi=4096, bs=64, layout="TND", pad=False),
        # a window-only layer verifying 16 drafted tokens for each of 64 requests
        dict(name="tree_window", op="tree", dtype="bf16", scenario=1, B=64, n=16, H=64, K=0, ratio=4, win=127,
             ctx_lo=4096, ctx_hi=16384, bs=128, layout="BSND", pad=True),
        # a top-k layer: every drafted token has its own 512 compressed rows
        dict(name="tree_topk", op="tree", dtype="bf16", scenario=3, B=64, n=8, H=128, K=512, ratio=4, win=127,
             ctx_lo=8192, ctx_hi=32768, bs=128, layout="TND", pad=False),
        # a layer that attends to its whole compressed cache, ratio 128, long contexts
        dict(name="tree_dense", op="tree", dtype="bf16", scenario=2, B=16, n=32, H=128, K=0, ratio=128, win=127,
             ctx_lo=65536, ctx_hi=262144, bs=128, layout="TND", pad=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope_bwd", "append", "append_bwd", "tree", "tree", "tree"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("norm_rope", "norm_rope_bwd"):
        D = rng.choice([64, 128, 192, 512, 512, 512])
        R = rng.choice([r for r in (32, 64, 128) if r <= D])
        H = rng.choice([1, 8, 16, 24, 40, 64, 128])
        most = 16384 * 64 * 512 if op == "norm_rope" else 8192 * 64 * 512
        T = _log_int(rng, 1, min(16384, most // (H * D)))
        return dict(op=op, dtype=dtype, T=T, H=H, Hk=rng.choice([0, 1, 1, 4]), D=D, R=R,
                    interleaved=rng.random() < 0.6, qw=rng.random() < 0.5, kw=rng.random() < 0.7, P=4096)
    if op in ("append", "append_bwd"):
        n = _log_int(rng, 1, 2048)
        B = _log_int(rng, 1, max(1, min(512, 16384 // n)))
        tree = n <= 64 and rng.random() < 0.5
        hi = _log_int(rng, 64, 700)
        H = 0 if op == "append_bwd" else rng.choice([0, 16, 64, 128])
        if n * B * H > 512 * 128 * 8:
            H = 0
        return dict(op=op, dtype=dtype, B=B, n=n, ctx_lo=rng.randint(0, hi), ctx_hi=hi, bs=rng.choice([16, 48, 64, 128]),
                    D=512, R=rng.choice([32, 64]), interleaved=rng.random() < 0.7, kw=rng.random() < 0.8, H=H,
                    tree=tree, layout=rng.choice(["TND", "TND", "BSND"]))
    scenario = rng.choice([1, 2, 3])
    H = rng.choice([8, 16, 24, 40, 64, 128])
    ratio = rng.choice([4, 16, 128]) if scenario == 2 else 4
    n = _log_int(rng, 1, 32)
    most = {1: 64 * 16 * 64, 2: 16 * 32 * 64, 3: 64 * 8 * 64}[scenario]
    B = _log_int(rng, 1, max(1, min(64, most // (n * H))))
    lo = _log_int(rng, 16, 8192)
    hi = _log_int(rng, lo, min(8 * lo, 65536 if ratio == 128 else 8192))
    return dict(op="tree", dtype=dtype, scenario=scenario, B=B, n=n, H=H,
                K=rng.choice([64, 200, 256, 512]) if scenario == 3 else 0, ratio=ratio, win=rng.choice([63, 127, 127, 200, 500]),
                ctx_lo=lo, ctx_hi=max(lo, hi), bs=rng.choice([16, 48, 64, 128]), layout=rng.choice(["TND", "BSND"]),
                pad=rng.random() < 0.4)


# ------------------------------------------------------------------- lengths
def _lens(c):
    """Drafted or new tokens of each request and the rows cached before them; they belong to the case."""
    B, n = c["B"], c["n"]
    ragged = c["layout"] == "TND" and n <= 64
    r = np.random.default_rng([B, n, c["ctx_hi"]])
    q = r.integers(max(1, n // 2), n + 1, B) if ragged else np.full(B, n)
    q[0] = n
    ctx = r.integers(c["ctx_lo"], c["ctx_hi"] + 1, B)
    return [int(x) for x in q], [int(x) for x in ctx]


def _pages(lens, bs, g):
    nb = [max(1, -(-x // bs)) for x in lens]
    total = sum(nb) + 1
    perm = torch.randperm(total, generator=g, device=DEV, dtype=torch.int64)
    width = max(nb)
    start = torch.tensor([0] + nb[:-1], device=DEV).cumsum(0)
    col = torch.arange(width, device=DEV)
    have = col[None] < torch.tensor(nb, device=DEV)[:, None]
    table = torch.where(have, perm[(start[:, None] + col).clamp(max=total - 1)], torch.full((), -1, device=DEV))
    return table.to(torch.int32).contiguous(), total


def _randn(shape, g, dt, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dt)


def _rope_table(P, R):
    inv = 10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
    a = torch.arange(P, device=DEV, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _trees(lens, n, seed, pad):
    """A random tree for each request, parents before children; with `pad`, some requests' last slots stay unused (-2)."""
    r = np.random.default_rng(seed)
    rows = []
    for m in lens:
        par = np.array([-1 if i == 0 else int(r.integers(max(-1, i - 6), i)) for i in range(m)], np.int32)
        if pad and m > 2 and r.random() < 0.5:
            par[m - int(r.integers(1, m // 2 + 1)):] = -2
        rows.append(par)
    return rows


def _depths(par):
    d = np.zeros(len(par), np.int32)
    for i, p in enumerate(par):
        d[i] = d[p] + 1 if p >= 0 else 0
    return d


# ------------------------------------------------------------------- prepare
def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = dict(case=c)
    if c["op"] in ("norm_rope", "norm_rope_bwd"):
        T, D = c["T"], c["D"]
        s["q"] = _randn((T, c["H"], D), g, dt, 2.0)
        s["k"] = _randn((T, c["Hk"], D), g, dt, 2.0) if c["Hk"] else None
        s["positions"] = torch.randint(0, c["P"], (T,), generator=g, device=DEV, dtype=torch.int32)
        s["cos"], s["sin"] = _rope_table(c["P"], c["R"])
        s["q_weight"] = 1 + 0.1 * torch.randn(D, generator=g, device=DEV) if c["qw"] else None
        s["k_weight"] = 1 + 0.1 * torch.randn(D, generator=g, device=DEV) if c["kw"] and c["Hk"] else None
        if c["op"] == "norm_rope_bwd":
            s["dq"] = _randn((T, c["H"], D), g, dt)
            s["dk"] = _randn((T, c["Hk"], D), g, dt) if c["Hk"] else None
        return s
    lens, ctx = _lens(c)
    s["lens"], s["ctx"] = lens, ctx
    used = [a + b for a, b in zip(lens, ctx)]
    T = sum(lens)
    s["T"] = T
    s["seqused_kv"] = torch.tensor(used, dtype=torch.int32, device=DEV)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    s["cu_seqlens_q"] = torch.from_numpy(cu).to(DEV)
    table, total = _pages(used, c["bs"], g)
    s["ori_block_table"] = table
    if c["op"] in ("append", "append_bwd"):
        pool = _randn((total, c["bs"], 1, c["D"]), g, dt)
        s["ori_kv"] = pool  # the cache, or the gradient of it
        s["kv"] = _randn((T, 1, c["D"]), g, dt, 2.0)
        s["q"] = _randn((T, c["H"], c["D"]), g, dt, 2.0) if c["H"] else None
        s["cos"], s["sin"] = _rope_table(max(used) + 64, c["R"])
        s["weight"] = 1 + 0.1 * torch.randn(c["D"], generator=g, device=DEV) if c["kw"] else None
        s["positions"] = None
        if c["tree"]:
            dep = np.concatenate([x + _depths(p) for x, p in zip(ctx, _trees(lens, c["n"], seed, False))])
            s["positions"] = torch.from_numpy(dep.astype(np.int32)).to(DEV)
        if c["layout"] == "BSND":
            for k in ("kv", "q", "positions"):
                s[k] = s[k].view(c["B"], c["n"], *s[k].shape[1:]) if s[k] is not None else None
        return s
    H = c["H"]
    s["q"] = _randn((T, H, 512), g, dt)
    s["ori_kv"] = _randn((total, c["bs"], 1, 512), g, dt)
    s["tree_parents"] = torch.from_numpy(np.concatenate(_trees(lens, c["n"], seed, c["pad"]))).to(DEV)
    s["sinks"] = torch.randn(H, generator=g, device=DEV)
    s["softmax_scale"] = 512 ** -0.5
    s["cmp_kv"] = s["cmp_block_table"] = s["idx"] = None
    if c["scenario"] >= 2:
        s["cmp_block_table"], total = _pages([x // c["ratio"] for x in ctx], c["bs"], g)
        s["cmp_kv"] = _randn((total, c["bs"], 1, 512), g, dt)
    if c["scenario"] == 3:
        # distinct ids of each token's valid range in random order, -1 where there are fewer
        K, lim = c["K"], torch.tensor([x // c["ratio"] for x in ctx], device=DEV)
        lim = torch.repeat_interleave(lim, torch.tensor(lens, device=DEV))
        most = max(max(ctx) // c["ratio"], K)
        key = torch.rand((T, most), generator=g, device=DEV)
        key = torch.where(torch.arange(most, device=DEV)[None] < lim[:, None], key, torch.full((), -1.0, device=DEV))
        val, ids = key.topk(K, dim=1)
        s["idx"] = torch.where(val >= 0, ids, torch.full((), -1, device=DEV)).to(torch.int32)[:, None].contiguous()
    if c["layout"] == "BSND":
        s["q"] = s["q"].view(c["B"], c["n"], H, 512)
        s["tree_parents"] = s["tree_parents"].view(c["B"], c["n"])
        if s["idx"] is not None:
            s["idx"] = s["idx"].view(c["B"], c["n"], 1, c["K"])
    return s


# --------------------------------------------------------------- plain forms
def _rotate(y, cos, sin, inter, back):
    """The last 2 * cos.shape[-1] dims of y rotated (by the negative angle with `back`); cos, sin [T, 1, R/2]."""
    R = 2 * cos.shape[-1]
    if back:
        sin = -sin
    a = y[..., y.shape[-1] - R:]
    x0, x1 = (a[..., 0::2], a[..., 1::2]) if inter else (a[..., : R // 2], a[..., R // 2:])
    r0, r1 = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    rot = torch.stack([r0, r1], -1).flatten(-2) if inter else torch.cat([r0, r1], -1)
    return torch.cat([y[..., : y.shape[-1] - R], rot], -1)


def _plain_fwd(x, w, cos, sin, inter):
    xf = x.float()
    y = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
    if w is not None:
        y = y * w
    return _rotate(y, cos, sin, inter, False).to(x.dtype)


def _plain_bwd(dy, x, w, cos, sin, inter):
    xf = x.float()
    rstd = torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
    xh = xf * rstd
    d = _rotate(dy.float(), cos, sin, inter, True)
    dw = (d * xh).sum((0, 1)) if w is not None else None
    if w is not None:
        d = d * w
    dx = rstd * (d - xh * (d * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw


def _cs(s, pos):
    return s["cos"][pos.long()][:, None], s["sin"][pos.long()][:, None]


def _slots(s, c):
    """Cache row (page * page size + offset) and position of every new token."""
    cu, bs = s["cu_seqlens_q"].long(), c["bs"]
    t = torch.arange(s["T"], device=DEV)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = s["seqused_kv"].long()[b] - (cu[b + 1] - cu[b]) + t - cu[b]
    return s["ori_block_table"].long()[b, pos // bs] * bs + pos % bs, pos


def _plain_tree(s, c):
    B, N, H = c["B"], c["n"], c["H"]
    cu = s["cu_seqlens_q"].long()
    n = cu[1:] - cu[:-1]
    ctx = s["seqused_kv"].long() - n
    i = torch.arange(N, device=DEV)
    have = i[None] < n[:, None]
    tok = (cu[:-1, None] + i).clamp(max=s["T"] - 1)
    par = torch.where(have, s["tree_parents"].reshape(-1).long()[tok], torch.full((), -2, device=DEV))
    live = par >= -1
    # which drafted tokens each one descends from, itself among them: paths of doubling length
    anc = ((i[None, None] == par[..., None]) | (i[:, None] == i)).float()
    for _ in range(max(1, (N - 1).bit_length())):
        anc = ((anc @ anc) > 0).float()
    anc = (anc > 0) & live[..., None]
    at = ctx[:, None] + anc.sum(-1) - 1  # position of each token
    W = c["win"]
    pos = ctx[:, None] - W + torch.arange(W + N, device=DEV)  # window rows, then the drafted ones
    real = (pos >= 0) & (pos < s["seqused_kv"].long()[:, None])
    p0 = pos.clamp(min=0, max=s["ori_block_table"].shape[1] * c["bs"] - 1)
    page = s["ori_block_table"].long().gather(1, p0 // c["bs"]).clamp(min=0)
    kv = s["ori_kv"].reshape(-1, 512)[page * c["bs"] + p0 % c["bs"]].float()
    q = s["q"].reshape(-1, H, 512)[tok].float()
    sc = (q.reshape(B, N * H, 512) @ kv.transpose(1, 2)).view(B, N, H, W + N) * s["softmax_scale"]
    see = real[:, None] & live[..., None] & torch.cat([pos[:, None, :W] >= at[..., None] - W, anc], -1)
    dep = anc.sum(-1) - 1
    see[..., W:] &= dep[..., None] - dep[:, None] <= W
    sc = sc.masked_fill(~see[:, :, None], -math.inf)
    parts = [(sc, kv)]
    if c["scenario"] == 2:
        L = max(1, max(x // c["ratio"] for x in s["ctx"]))
        j = torch.arange(L, device=DEV)
        page = s["cmp_block_table"].long()[:, j // c["bs"]].clamp(min=0)
        kc = s["cmp_kv"].reshape(-1, 512)[page * c["bs"] + j % c["bs"]].float()
        x = (q.reshape(B, N * H, 512) @ kc.transpose(1, 2)).view(B, N, H, L) * s["softmax_scale"]
        ok = (j < ctx[:, None] // c["ratio"])[:, None] & live[..., None]
        parts.append((x.masked_fill(~ok[:, :, None], -math.inf), kc))
    elif c["scenario"] == 3:
        K = c["K"]
        ids = s["idx"].reshape(-1, K)[tok].long()
        ok = (ids >= 0) & (ids < ctx[:, None, None] // c["ratio"]) & live[..., None]
        ids = torch.where(ok, ids, torch.zeros((), dtype=torch.int64, device=DEV))
        bt = s["cmp_block_table"].long()[:, None].expand(B, N, -1)
        kc = s["cmp_kv"].reshape(-1, 512)[bt.gather(2, ids // c["bs"]).clamp(min=0) * c["bs"] + ids % c["bs"]].float()
        x = (q @ kc.transpose(2, 3)) * s["softmax_scale"]
        parts.append((x.masked_fill(~ok[:, :, None], -math.inf), kc))
    sink = s["sinks"][:, None]
    x = torch.cat([p[0] for p in parts], -1)
    m = torch.maximum(x.amax(-1, keepdim=True), sink)
    p = torch.exp(x - m)
    l = p.sum(-1, keepdim=True) + torch.exp(sink - m)
    w = sc.shape[-1]
    o = (p[..., :w].reshape(B, N * H, w) @ kv).view(B, N, H, 512)
    if len(parts) == 2:
        pc, kc = p[..., w:], parts[1][1]
        o = o + ((pc.reshape(B, N * H, -1) @ kc).view(B, N, H, 512) if kc.dim() == 3 else pc @ kc)
    o = torch.where(live[..., None, None], o / l, torch.zeros((), device=DEV)).to(s["q"].dtype)
    lse = torch.where(live[..., None], (m + torch.log(l))[..., 0], torch.zeros((), device=DEV))
    if c["layout"] == "BSND":
        return o, lse
    keep = have.reshape(-1).nonzero()[:, 0]
    return o.reshape(-1, H, 512)[keep], lse.reshape(-1, H)[keep]


def _plain(s):
    c = s["case"]
    inter = c.get("interleaved", True)
    if c["op"] == "norm_rope":
        cos, sin = _cs(s, s["positions"])
        k = _plain_fwd(s["k"], s["k_weight"], cos, sin, inter) if s["k"] is not None else None
        return _plain_fwd(s["q"], s["q_weight"], cos, sin, inter), k
    if c["op"] == "norm_rope_bwd":
        cos, sin = _cs(s, s["positions"])
        dk, dkw = _plain_bwd(s["dk"], s["k"], s["k_weight"], cos, sin, inter) if s["k"] is not None else (None, None)
        dq, dqw = _plain_bwd(s["dq"], s["q"], s["q_weight"], cos, sin, inter)
        return dq, dk, dqw, dkw
    if c["op"] == "tree":
        return _plain_tree(s, c)
    rows, pos = _slots(s, c)
    cos, sin = _cs(s, pos if s["positions"] is None else s["positions"].reshape(-1))
    flat, kv = s["ori_kv"].view(-1, 1, c["D"]), s["kv"].reshape(-1, 1, c["D"])
    if c["op"] == "append_bwd":
        dkv, dw = _plain_bwd(flat[rows], kv, s["weight"], cos, sin, inter)
        return dkv.view(s["kv"].shape), dw
    flat[rows] = _plain_fwd(kv, s["weight"], cos, sin, inter)
    if s["q"] is None:
        return s["ori_kv"], None
    return s["ori_kv"], _plain_fwd(s["q"].reshape(-1, c["H"], c["D"]), None, cos, sin, inter).view(s["q"].shape)


# ----------------------------------------------------------------------- run
def _own(s):
    import dsv4_b200 as M

    c = s["case"]
    if c["op"] in ("norm_rope", "norm_rope_bwd"):
        kw = dict(positions=s["positions"], cos=s["cos"], sin=s["sin"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                  eps=EPS, interleaved=c["interleaved"])
        if c["op"] == "norm_rope":
            r = M.head_norm_rope(s["q"], s["k"], **kw)
            return r if s["k"] is not None else (r, None)
        return M.head_norm_rope_backward(s["dq"], s["q"], s["dk"], s["k"], **kw)
    if c["op"] in ("append", "append_bwd"):
        kw = dict(ori_block_table=s["ori_block_table"], seqused_kv=s["seqused_kv"], layout_q=c["layout"],
                  cu_seqlens_q=s["cu_seqlens_q"] if c["layout"] == "TND" else None, positions=s["positions"], cos=s["cos"], sin=s["sin"], weight=s["weight"], eps=EPS,
                  interleaved=c["interleaved"])
        if c["op"] == "append_bwd":
            return M.append_shared_kv_backward(s["ori_kv"], s["kv"], **kw)
        r = M.append_shared_kv(s["kv"], s["ori_kv"], q=s["q"], **kw)
        return r if s["q"] is not None else (r, None)
    kw = dict(ori_kv=s["ori_kv"], ori_block_table=s["ori_block_table"], tree_parents=s["tree_parents"],
              seqused_kv=s["seqused_kv"], sinks=s["sinks"], softmax_scale=s["softmax_scale"], ori_win_left=c["win"],
              layout_q=c["layout"], return_softmax_lse=True)
    if c["layout"] == "TND":
        kw["cu_seqlens_q"] = s["cu_seqlens_q"]
    if c["scenario"] >= 2:
        kw.update(cmp_kv=s["cmp_kv"], cmp_block_table=s["cmp_block_table"], cmp_ratio=c["ratio"])
    if c["scenario"] == 3:
        kw["cmp_sparse_indices"] = s["idx"]
    return M.tree_attn_sharedkv(s["q"], **kw)


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] in ("norm_rope", "norm_rope_bwd"):
        n = c["T"] * (c["H"] + c["Hk"]) * c["D"]
        table = min(c["T"], c["P"]) * c["R"] * 4 + 4 * c["T"]
        w = 4 * c["D"] * (c["qw"] + (c["kw"] and c["Hk"] > 0))
        if c["op"] == "norm_rope":
            return {"bytes": 4 * n + table + w, "flops": 5 * n}
        return {"bytes": 6 * n + table + 2 * w, "flops": 12 * n}
    lens, ctx = _lens(c)
    T = sum(lens)
    if c["op"] in ("append", "append_bwd"):
        small = T * (c["R"] * 4 + 4) + 4 * sum(-(-(a + b) // c["bs"]) for a, b in zip(lens, ctx)) + 4 * c["D"]
        n = T * (1 + c["H"]) * c["D"]
        if c["op"] == "append":
            return {"bytes": 4 * n + small, "flops": 5 * n}
        return {"bytes": 6 * n + small, "flops": 12 * n}
    H, W = c["H"], c["win"]
    rows = uniq = 0
    for m, x in zip(lens, ctx):
        rows += m * min(x + 1, W + 1)
        uniq += min(x, W) + m
        thr = x // c["ratio"]
        if c["scenario"] == 2:
            rows += m * thr
            uniq += thr
        elif c["scenario"] == 3 and thr:
            k = min(c["K"], thr)
            rows += m * k
            uniq += thr * (1 - (1 - k / thr) ** m)
    bytes_ = uniq * 1024 + T * H * (2 * 1024 + 4) + T * (c["K"] * 4 + 4) + 4 * uniq / c["bs"]
    return {"bytes": bytes_, "flops": 4 * 512 * H * rows}


# --------------------------------------------------------------------- exact
def _exact_fwd(x, w, cos, sin, inter):
    y = x.double()
    y = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    if w is not None:
        y = y * w.double()
    h = cos.shape[-1]
    D = y.shape[-1]
    a = torch.arange(h, device=DEV)
    i0, i1 = (D - 2 * h + 2 * a, D - 2 * h + 2 * a + 1) if inter else (D - 2 * h + a, D - h + a)
    z = torch.complex(y[..., i0], y[..., i1]) * torch.complex(cos.double(), sin.double())
    y[..., i0], y[..., i1] = z.real, z.imag
    return y


def _exact_bwd(dy, x, w, cos, sin, inter):
    # by differentiation of the definition, a slice of the tokens at a time
    dxs, dw = [], torch.zeros(x.shape[-1], dtype=torch.float64, device=DEV)
    for t in range(0, x.shape[0], 1024):
        xs = x[t:t + 1024].double().requires_grad_()
        ws = (w.double() if w is not None else torch.ones_like(dw)).requires_grad_()
        y = xs / (xs.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * ws
        h, D = cos.shape[-1], x.shape[-1]
        tail = y[..., D - 2 * h:].unflatten(-1, (h, 2) if inter else (2, h))
        tail = tail if inter else tail.transpose(-1, -2)
        z = torch.view_as_complex(tail.contiguous()) * torch.complex(cos[t:t + 1024].double(), sin[t:t + 1024].double())
        r = torch.view_as_real(z)
        r = (r if inter else r.transpose(-1, -2)).flatten(-2)
        gx, gw = torch.autograd.grad(torch.cat([y[..., : D - 2 * h], r], -1), (xs, ws), dy[t:t + 1024].double())
        dxs.append(gx)
        dw += gw
    return torch.cat(dxs), dw if w is not None else None


def _exact_tree(s, c):
    H, bs = c["H"], c["bs"]
    q = s["q"].reshape(-1, H, 512)
    par = s["tree_parents"].reshape(-1).tolist()
    ori, cmp = s["ori_kv"].reshape(-1, 512), s["cmp_kv"].reshape(-1, 512) if s["cmp_kv"] is not None else None
    obt = s["ori_block_table"].tolist()
    out = torch.zeros((s["T"], H, 512), dtype=torch.float64, device=DEV)
    lse = torch.zeros((s["T"], H), dtype=torch.float64, device=DEV)
    sink = s["sinks"].double()
    t = 0
    for b, (m, x) in enumerate(zip(s["lens"], s["ctx"])):
        thr = x // c["ratio"]
        cbt = s["cmp_block_table"][b].long() if cmp is not None else None
        for i in range(m):
            if par[t + i] >= -1:
                path, j = [], i
                while j >= 0:
                    path.append(j)
                    j = par[t + j]
                at = x + len(path) - 1
                pos = list(range(max(0, at - c["win"]), x)) + [x + j for d, j in enumerate(path) if d <= c["win"]]
                rows = ori[torch.tensor([obt[b][p // bs] * bs + p % bs for p in pos], device=DEV)].double()
                if c["scenario"] == 2:
                    j = torch.arange(thr, device=DEV)
                    rows = torch.cat([rows, cmp[cbt[j // bs] * bs + j % bs].double()])
                elif c["scenario"] == 3:
                    j = s["idx"].reshape(-1, c["K"])[t + i].long()
                    j = j[(j >= 0) & (j < thr)]
                    rows = torch.cat([rows, cmp[cbt[j // bs] * bs + j % bs].double()])
                a = torch.cat([q[t + i].double() @ rows.T * s["softmax_scale"], sink[:, None]], 1)
                lse[t + i] = torch.logsumexp(a, 1)
                out[t + i] = torch.softmax(a, 1)[:, :-1] @ rows
        t += m
    return out.view(s["q"].shape), lse.view(s["q"].shape[:-1])


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    inter = c.get("interleaved", True)
    if c["op"] == "tree":
        return _exact_tree(s, c)
    if c["op"] in ("norm_rope", "norm_rope_bwd"):
        p = s["positions"].long()
        cos, sin = s["cos"][p][:, None], s["sin"][p][:, None]
        if c["op"] == "norm_rope":
            k = _exact_fwd(s["k"], s["k_weight"], cos, sin, inter) if s["k"] is not None else None
            return _exact_fwd(s["q"], s["q_weight"], cos, sin, inter), k
        dq, dqw = _exact_bwd(s["dq"], s["q"], s["q_weight"], cos, sin, inter)
        dk, dkw = _exact_bwd(s["dk"], s["k"], s["k_weight"], cos, sin, inter) if s["k"] is not None else (None, None)
        return dq, dk, dqw, dkw
    bt, rows, pos = s["ori_block_table"].tolist(), [], []
    for b, (m, x) in enumerate(zip(s["lens"], s["ctx"])):
        pos += range(x, x + m)
        rows += [bt[b][p // c["bs"]] * c["bs"] + p % c["bs"] for p in range(x, x + m)]
    rows = torch.tensor(rows, device=DEV)
    p = s["positions"].reshape(-1).long() if s["positions"] is not None else torch.tensor(pos, device=DEV)
    cos, sin = s["cos"][p][:, None], s["sin"][p][:, None]
    flat, kv = s["ori_kv"].view(-1, 1, c["D"]), s["kv"].reshape(-1, 1, c["D"])
    if c["op"] == "append_bwd":
        dkv, dw = _exact_bwd(flat[rows], kv, s["weight"], cos, sin, inter)
        return dkv.view(s["kv"].shape), dw
    pool = flat.double()
    pool[rows] = _exact_fwd(kv, s["weight"], cos, sin, inter)
    if s["q"] is None:
        return pool.view(s["ori_kv"].shape), None
    return pool.view(s["ori_kv"].shape), _exact_fwd(s["q"].reshape(-1, c["H"], c["D"]), None, cos, sin, inter).view(s["q"].shape)
