"""Attention of drafted trees against a 64-bit definition, its masks, edges and refusals.

Bounds, from the arithmetic (u = 2^-8 for bf16, 2^-11 for fp16): the output is
rounded once (u * |out|); every P_j is rounded to the I/O type before the
product (u * sum_j p_j |v_j|; for fp16 also half a subnormal spacing, 2^-25,
relative to the largest P of at least 2^-8: 2^-17 * mean |v|, within the next
term); scores are fp32 sums of 512 exact products, off by at most
512 * 2^-24 * scale * sum_d |q_d k_d| =: e, which moves p by a factor e^(+-2e),
and the fp32 sums and exponentials add 1e-5. LSE: e + 1e-6 * (1 + |lse|).
"""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

D = 512
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Case:
    def __init__(self, lens, ctx, *, H=16, dt=torch.bfloat16, scenario=1, K=64, ratio=4, win=127, bs=64, layout="TND",
                 trees=None, seed=0, pad=0, lead=0):
        g = torch.Generator().manual_seed(seed)
        r = np.random.default_rng(seed)
        self.lens, self.ctx, self.H, self.dt, self.scenario, self.K = lens, ctx, H, dt, scenario, K
        self.ratio, self.win, self.bs, self.layout = ratio, win, bs, layout
        self.S = max(lens) if layout == "BSND" else 0
        self.base = [b * self.S for b in range(len(lens))] if layout == "BSND" else list(lead + np.cumsum([0] + lens[:-1]))
        self.T = len(lens) * self.S if layout == "BSND" else lead + sum(lens) + pad
        self.q = torch.randn((self.T, H, D), generator=g).to(dt)
        if trees is None:
            trees = [[-1 if i == 0 else int(r.integers(max(-1, i - 5), i)) for i in range(n)] for n in lens]
        self.parents = torch.full((self.T,), -2, dtype=torch.int32)
        for b, t in enumerate(trees):
            self.parents[self.base[b]:self.base[b] + len(t)] = torch.tensor(t, dtype=torch.int32)
        used = [a + b for a, b in zip(lens, ctx)]
        self.used = torch.tensor(used, dtype=torch.int32)
        self.ori, self.obt = self.pages(used, g)
        self.cmp = self.cbt = self.idx = None
        if scenario >= 2:
            self.cmp, self.cbt = self.pages([x // ratio for x in ctx], g)
        if scenario == 3:
            self.idx = torch.full((self.T, 1, K), -1, dtype=torch.int32)
            for b, n in enumerate(lens):
                thr = ctx[b] // ratio
                for i in range(n):
                    k = min(K, thr)
                    self.idx[self.base[b] + i, 0, :k] = torch.from_numpy(r.choice(thr, k, replace=False).astype(np.int32)) if k else -1
        self.sinks = torch.randn(H, generator=g)
        self.scale = D ** -0.5

    def pages(self, lens, g):
        nb = [max(1, -(-x // self.bs)) for x in lens]
        perm = torch.randperm(sum(nb) + 1, generator=g)
        table = torch.full((len(lens), max(nb)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(nb):
            table[b, :n] = perm[at:at + n]
            at += n
        return torch.randn((sum(nb) + 1, self.bs, 1, D), generator=g).to(self.dt), table

    def call(self, **over):
        from dsv4_b200 import tree_attn_sharedkv

        shape = (lambda t: t.view(len(self.lens), self.S, *t.shape[1:])) if self.layout == "BSND" else (lambda t: t)
        kw = dict(ori_kv=self.ori.cuda(), ori_block_table=self.obt.cuda(), tree_parents=shape(self.parents).cuda(),
                  seqused_kv=self.used.cuda(), sinks=self.sinks.cuda(), softmax_scale=self.scale, ori_win_left=self.win,
                  layout_q=self.layout, return_softmax_lse=True)
        ragged = self.layout == "BSND" and any(n != self.S for n in self.lens)
        if self.layout == "TND" or ragged:
            at = self.base + [self.base[-1] + self.lens[-1]] if self.layout == "TND" else [0] + list(np.cumsum(self.lens))
            kw["cu_seqlens_q"] = torch.tensor(at, dtype=torch.int32).cuda()
        if self.scenario >= 2:
            kw.update(cmp_kv=self.cmp.cuda(), cmp_block_table=self.cbt.cuda(), cmp_ratio=self.ratio)
        if self.scenario == 3:
            kw["cmp_sparse_indices"] = shape(self.idx).cuda()
        kw.update(over)
        o, lse = tree_attn_sharedkv(kw.pop("q", shape(self.q).cuda()), **kw)
        return o.reshape(self.T, self.H, D), lse.reshape(self.T, self.H)

    def row(self, pool, table, b, pos):
        blk = int(table[b, pos // self.bs])
        return None if blk < 0 else pool[blk, pos % self.bs, 0].double()

    def rows(self, b, i):
        """The KV rows that token i of request b sees, in float64; None for an unused token."""
        par = self.parents[self.base[b]:self.base[b] + self.lens[b]].tolist()
        if par[i] < -1:
            return None
        path, j = [], i
        while j >= 0:
            path.append(j)
            j = par[j]
        s = self.ctx[b] + len(path) - 1
        pos = list(range(max(0, s - self.win), self.ctx[b])) + [self.ctx[b] + j for d, j in enumerate(path) if d <= self.win]
        rows = [self.row(self.ori, self.obt, b, p) for p in pos]
        thr = self.ctx[b] // self.ratio
        if self.scenario == 2:
            rows += [self.row(self.cmp, self.cbt, b, p) for p in range(thr)]
        elif self.scenario == 3:
            rows += [self.row(self.cmp, self.cbt, b, p) for p in self.idx[self.base[b] + i, 0].tolist() if 0 <= p < thr]
        rows = [r for r in rows if r is not None]
        return torch.stack(rows) if rows else torch.zeros(0, D, dtype=torch.float64)

    def check(self, out, lse, skip=()):
        out, lse, u = out.double().cpu(), lse.double().cpu(), U[self.dt]
        held = set()
        for b, n in enumerate(self.lens):
            for i in range(n):
                t = self.base[b] + i
                held.add(t)
                if t in skip:
                    continue
                kv = self.rows(b, i)
                if kv is None:
                    held.discard(t)
                    continue
                q = self.q[t].double()
                x = q @ kv.T * self.scale
                e = (512 * 2.0 ** -24 * self.scale * (q.abs() @ kv.abs().T)).amax(-1, keepdim=True) if len(kv) else torch.zeros(self.H, 1)
                full = torch.cat([x, self.sinks.double()[:, None]], 1)
                ref = torch.logsumexp(full, 1)
                p = torch.softmax(full, 1)[:, :-1] if len(kv) or torch.isfinite(self.sinks).all() else torch.zeros(self.H, 0, dtype=torch.float64)
                o, mag = p @ kv, p @ kv.abs()
                lim = u * o.abs() + (u * 1.01 + 2 * e + 1e-5) * mag + 2.0 ** -25
                over = (out[t] - o).abs() - lim
                assert over.max() <= 0, f"token {t}: {(out[t] - o).abs().max():.3e}, {over.max():.3e} over the bound"
                dl = torch.where(lse[t] == ref, torch.zeros_like(ref), (lse[t] - ref).abs())  # -inf where nothing is seen
                assert (dl <= e[:, 0] + 1e-6 * (1 + ref.abs().clamp(max=1e6))).all(), f"token {t}: LSE off by {dl.max():.3e}"
        for t in set(range(self.T)) - held:
            assert not out[t].any() and not lse[t].any(), f"unused token {t} is not zero"


# ------------------------------------------------------------------ refusals
def _call(**over):
    from dsv4_b200 import tree_attn_sharedkv

    T, H = over.pop("T", 3), over.pop("H", 16)
    dt = over.pop("dtype", torch.bfloat16)
    kv = torch.zeros(4, 16, 1, D, dtype=dt)
    kw = dict(q=torch.zeros(T, H, D, dtype=dt), ori_kv=kv, ori_block_table=torch.zeros(2, 2, dtype=torch.int32),
              tree_parents=torch.zeros(T, dtype=torch.int32), seqused_kv=torch.tensor([9, 9], dtype=torch.int32),
              sinks=torch.zeros(H), softmax_scale=1.0, cu_seqlens_q=torch.tensor([0, 1, 3], dtype=torch.int32),
              cmp_kv=kv, cmp_block_table=torch.zeros(2, 2, dtype=torch.int32),
              cmp_sparse_indices=torch.zeros(T, 1, 8, dtype=torch.int32))
    kw.update(over)
    return tree_attn_sharedkv(kw.pop("q"), **kw)


@pytest.mark.parametrize("over", [
    dict(H=12), dict(dtype=torch.float32), dict(q=torch.zeros(3, 16, 256, dtype=torch.bfloat16)),
    dict(q=torch.zeros(1, 3, 16, D, dtype=torch.bfloat16)), dict(tree_parents=torch.zeros(2, dtype=torch.int32)),
    dict(sinks=torch.zeros(8)), dict(seqused_kv=torch.zeros(1, dtype=torch.int32)), dict(ori_win_left=-1),
    dict(cmp_ratio=0), dict(ori_kv=torch.zeros(4, 16, 1, D).half()), dict(ori_kv=torch.zeros(4, 16, D).bfloat16()),
    dict(ori_block_table=torch.zeros(3, 2, dtype=torch.int32)), dict(cmp_sparse_indices=torch.zeros(2, 1, 8, dtype=torch.int32)),
    dict(out=torch.zeros(3, 16, D)), dict(lse_out=torch.zeros(3, 8)),
], ids=lambda o: next(iter(o)))
def test_value_errors(over):
    with pytest.raises(ValueError):
        _call(**over)


@pytest.mark.parametrize("over", [dict(layout_q="BSH"), dict(layout_kv="TND"), dict(cu_seqlens_q=None),
                                  dict(cmp_block_table=None), dict(cmp_kv=None)], ids=lambda o: next(iter(o)))
def test_assertions(over):
    with pytest.raises(AssertionError):
        _call(**over)


def test_cpu_tensors_have_no_fallback():
    with pytest.raises(RuntimeError, match="CUDA"):
        _call()


# ----------------------------------------------------------------------- GPU
@pytest.fixture
def gpu(sas_lib):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from dsv4_b200 import check_device_status, reset_device_status

    reset_device_status()
    yield
    check_device_status()


BF, FP = torch.bfloat16, torch.float16
CASES = {
    "first token": dict(lens=[1], ctx=[0], H=8),
    "one cached": dict(lens=[1, 1], ctx=[1, 128], H=64, bs=1),
    "no context": dict(lens=[16, 3], ctx=[0, 0], H=24, bs=16),
    "short windows": dict(lens=[5, 9], ctx=[40, 127], H=40, bs=48, dt=FP),
    "window 0": dict(lens=[7], ctx=[50], H=8, win=0),
    "window past a tile": dict(lens=[6, 2], ctx=[900, 300], H=16, win=300, bs=48),
    "whole context": dict(lens=[4], ctx=[2500], H=16, win=1 << 40, bs=128),
    "heads over 128": dict(lens=[3], ctx=[200], H=200),
    "chain past its window": dict(lens=[60], ctx=[33], H=8, win=7, trees=[list(range(-1, 59))], bs=16),
    "wide tree": dict(lens=[300], ctx=[70], H=8, bs=16),
    "empty requests": dict(lens=[0, 2, 0, 0, 3, 0], ctx=[5, 70, 0, 9, 200, 1], H=16, scenario=2),
    "rows of no request": dict(lens=[2, 2], ctx=[70, 10], H=16, pad=5, lead=3),
    "padded": dict(lens=[4, 4, 4], ctx=[30, 300, 128], H=64, layout="BSND", trees=[[-1, 0], [-2, -1, -2, 1], [-2] * 4]),
    "long runs of unused slots": dict(lens=[24] * 6, ctx=[30, 300, 128, 2, 400, 260], H=64, layout="BSND", scenario=2,
                                      trees=[[-1] + [-2] * 23, [-2] * 20 + [-1, -1, 20, -2], [-2] * 24, [-1, 0] + [-2] * 22,
                                             [-2] * 23 + [-1], [-1] * 24]),
    "padding past 64 slots": dict(lens=[150] * 3, ctx=[70, 300, 9], H=8, layout="BSND", scenario=2,
                                  trees=[[-1] + [-2] * 149, [-2] * 140 + [-1, 140, -2, 141] + [-2] * 6, [-2] * 150]),
    "padded top-k": dict(lens=[20] * 3, ctx=[70, 300, 900], H=136, layout="BSND", scenario=3, K=70,
                         trees=[[-2] * 20, [-1, 0] + [-2] * 18, [-2] * 9 + [-1] + [-2] * 10]),
    "ragged bsnd": dict(lens=[2, 5, 0], ctx=[30, 300, 128], H=16, layout="BSND", scenario=2, ratio=16),
    "dense": dict(lens=[5, 1], ctx=[1000, 37], H=64, scenario=2),
    "dense odd": dict(lens=[3, 8, 2], ctx=[515, 4099, 3], H=24, scenario=2, ratio=4, bs=48, dt=FP, win=63),
    "one long request": dict(lens=[1], ctx=[60000], H=16, scenario=2, bs=128),
    "many requests": dict(lens=[1] * 500, ctx=[i % 150 for i in range(500)], H=8, bs=32),
    "top-k": dict(lens=[3, 1, 6], ctx=[2000, 9, 400], H=64, scenario=3, K=256),
    "top-k odd": dict(lens=[2, 5], ctx=[900, 2], H=40, scenario=3, K=200, bs=16, dt=FP),
    "top-k 3 head groups": dict(lens=[2, 2], ctx=[900, 1500], H=136, scenario=3, K=130),
    "top-k bsnd": dict(lens=[4, 4], ctx=[3, 700], H=16, scenario=3, K=64, layout="BSND", trees=[[-1, 0, -2, -2], [-1, -1, 0, 0]]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
def test_against_the_definition(gpu, name):
    c = Case(**CASES[name])
    out, lse = c.call()
    c.check(out, lse)
    again = c.call()
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1]), "a repeat differs"


@pytest.mark.gpu
@pytest.mark.parametrize("scenario", [1, 3])
def test_no_sinks_and_large_sinks(gpu, scenario):
    c = Case([3, 2], [150, 0], H=16, scenario=scenario, K=64)
    c.sinks[:] = float("-inf")
    c.check(*c.call())
    c.sinks[::2] = 90.0
    c.sinks[1::2] = -90.0
    c.check(*c.call())


@pytest.mark.gpu
def test_scores_that_rise_and_fall(gpu):
    """Maxima that move from tile to tile by far more than the running maximum may lag, up and down."""
    for seed, order in ((1, 1), (2, -1)):
        c = Case([2], [1500], H=16, scenario=2, ratio=2, seed=seed)
        k = torch.arange(c.cmp.shape[0] * c.bs).view(-1, c.bs, 1, 1).double() / (c.cmp.shape[0] * c.bs)
        c.cmp = (c.cmp.double() * (0.05 + 6 * (k if order > 0 else 1 - k))).to(c.dt)
        c.check(*c.call())


@pytest.mark.gpu
def test_odd_ids_in_the_lists(gpu):
    """Ids past the committed rows, negative ones anywhere and repeated ones."""
    c = Case([4, 3], [400, 1600], H=16, scenario=3, K=96)
    c.idx[0, 0, ::3] = -1
    c.idx[1, 0, 5:50] = 100  # 400 // 4: one past
    c.idx[2, 0] = 7
    c.idx[3, 0] = -5
    c.idx[4, 0, 10] = 2 ** 31 - 1
    c.check(*c.call())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
def test_rows_that_are_not_finite(gpu, bad, dt):
    """They reach the tokens that see them and no others, in one branch, in the
    window's edge and in rows that nobody sees."""
    c = Case([4], [140], H=16, dt=dt, win=100, trees=[[-1, 0, 0, 2]])
    rows = c.ori.view(-1, D)
    at = lambda p: int(c.obt[0, p // c.bs]) * c.bs + p % c.bs  # noqa: E731
    rows[at(141), 3] = bad           # token 1: seen by itself alone
    rows[at(40), 100] = bad          # seen from position 140, token 0, alone (depths 1 and 2 start at 41, 42)
    rows[at(30)] = bad               # before every window
    for p in range(144, c.obt.shape[1] * c.bs):
        rows[at(p)] = bad            # past the last token
    out, lse = c.call()
    assert torch.isnan(out[:2].float()).all(-1).all()
    c.check(out, lse, skip=(0, 1))
    # a query that is not finite spoils its own heads alone
    c = Case([3], [200], H=16, dt=dt, trees=[[-1, 0, 0]])
    c.q[1, 5, 17] = bad
    out, lse = c.call()
    assert torch.isnan(out[1, 5].float()).any()
    c.check(out, lse, skip=(1,))
    good = Case([3], [200], H=16, dt=dt, trees=[[-1, 0, 0]]).call()[0]
    keep = [h for h in range(16) if h != 5]
    assert torch.equal(out[1, keep], good[1, keep])


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [64, 48, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_past_the_committed_ones_are_not_finite(gpu, bad, bs):
    """What a page of the compressed cache holds past its request's last row reaches nobody."""
    c = Case([3, 1, 2], [1000, 514, 5], H=16, scenario=2, bs=bs)
    for b, ctx in enumerate(c.ctx):
        for p in range(ctx // c.ratio, (ctx // c.ratio + bs - 1) // bs * bs):
            c.cmp[c.cbt[b, p // bs], p % bs] = bad
    c.check(*c.call())


@pytest.mark.gpu
def test_weightless_rows_that_are_not_finite(gpu):
    """Scores of -inf alone in a part of a cut unit: the joined result is still NaN for the tokens that see the rows."""
    c = Case([1], [40000], H=8, scenario=1, win=1 << 20)
    c.q[..., 7] = -1.0
    for p in range(40001):
        c.ori[c.obt[0, p // c.bs], p % c.bs, 0, 7] = float("inf")
    c.sinks[:] = float("-inf")
    out, lse = c.call()
    assert torch.isnan(out[..., 7].float()).all() and torch.isnan(lse).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scenario", [1, 2, 3])
def test_chain_is_the_frameworks_decode(gpu, scenario):
    """A tree that is a chain, with no compressed row ending among its tokens, is sparse_attn_sharedkv's case."""
    from dsv4_b200 import sparse_attn_sharedkv

    c = Case([2, 3, 1], [804, 128, 1600], H=16, scenario=scenario, ratio=4, trees=[[-1, 0], [-1, 0, 1], [-1]])
    out, lse = c.call()
    kw = dict(ori_kv=c.ori.cuda(), ori_block_table=c.obt.cuda(), seqused_kv=c.used.cuda(), sinks=c.sinks.cuda(),
              cu_seqlens_q=torch.tensor([0, 2, 5, 6], dtype=torch.int32).cuda(), softmax_scale=c.scale)
    if scenario >= 2:
        kw.update(cmp_kv=c.cmp.cuda(), cmp_block_table=c.cbt.cuda(), cmp_ratio=4)
    if scenario == 3:
        kw["cmp_sparse_indices"] = c.idx.cuda()
    o, l = sparse_attn_sharedkv(c.q.cuda(), return_softmax_lse=True, **kw)
    c.check(out, lse)
    c.check(o, l)


@pytest.mark.gpu
def test_bad_block_entries_are_dropped(gpu):
    """Like -1 entries; the pool is declared smaller than its allocation, so an unchecked read would stay inside it."""
    from dsv4_b200 import device_status, reset_device_status

    c = Case([2, 2], [300, 260], H=16, scenario=2, win=200)
    c.obt[0, 2] = -1
    c.cbt[1, 0] = -1
    ref = c.call()
    c.check(*ref)
    assert device_status() == 0
    n, m = c.ori.shape[0], c.cmp.shape[0]
    c.obt[0, 2], c.cbt[1, 0] = n, m + 5
    got = c.call(ori_kv=torch.cat([c.ori, c.ori]).cuda()[:n], cmp_kv=torch.cat([c.cmp] * 8).cuda()[:m])
    assert device_status() == 7
    reset_device_status()
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    c.obt = c.obt[:, :4].contiguous()  # request 0's drafted rows lie past the table
    c.call()
    assert device_status() == 7
    reset_device_status()


@pytest.mark.gpu
def test_bad_trees_are_recorded(gpu):
    from dsv4_b200 import device_status, reset_device_status

    for trees, skip in (([[-1, 1, 0], [-1, 0, 0]], 1), ([[-1, 0, 7], [-1, 0, 0]], 2), ([[-1, -2, 1], [-1, 0, 0]], 2)):
        c = Case([3, 3], [90, 400], H=16, trees=trees)
        out, lse = c.call()
        assert device_status() == 9
        reset_device_status()
        assert not out[skip].any() and not lse[skip].any()
        c.check(out, lse, skip=(skip, 1))
    c = Case([2, 2], [50, 60], H=16)
    c.used[0] = 1  # fewer rows than tokens
    out, lse = c.call()
    assert device_status() == 9 and not out[:2].any() and not lse[:2].any()
    reset_device_status()
    c.check(out, lse, skip=(0, 1))
    c = Case([1025, 2], [0, 60], H=8, trees=[[-1] * 1025, [-1, 0]])
    out, lse = c.call()
    assert device_status() == 9 and not out[:1025].any() and not lse[:1025].any()
    reset_device_status()
    c.check(out, lse, skip=range(1025))


@pytest.mark.gpu
def test_strides_streams_and_graphs(gpu):
    c = Case([3, 4], [500, 90], H=16, scenario=3, K=128)
    ref = c.call()
    wide = torch.zeros(c.T, 32, D + 8, dtype=c.dt, device="cuda")
    wide[:, 8:24, 8:] = c.q.cuda()
    odd = torch.empty(c.q.numel() + 1, dtype=c.dt, device="cuda")[1:].view(c.q.shape).copy_(c.q)
    for q in (wide[:, 8:24, 8:], odd):
        assert torch.equal(c.call(q=q)[0], ref[0])
    assert torch.equal(c.call(tree_parents=c.parents.cuda().long(), sinks=c.sinks.cuda().double())[0], ref[0])
    out, lse = torch.empty_like(ref[0]), torch.empty_like(ref[1])
    assert c.call(out=out, lse_out=lse)[0].data_ptr() == out.data_ptr() and torch.equal(out, ref[0])
    from dsv4_b200 import tree_attn_sharedkv

    kw = dict(ori_kv=c.ori.cuda(), ori_block_table=c.obt.cuda(), tree_parents=c.parents.cuda(), seqused_kv=c.used.cuda(),
              sinks=c.sinks.cuda(), softmax_scale=c.scale, cu_seqlens_q=torch.tensor([0, 3, 7], dtype=torch.int32).cuda(),
              cmp_kv=c.cmp.cuda(), cmp_block_table=c.cbt.cuda(), cmp_ratio=4, cmp_sparse_indices=c.idx.cuda())
    q = c.q.cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 3:  # two streams at once do not share a workspace
        with torch.cuda.stream(s):
            got.append(tree_attn_sharedkv(q, **kw))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(streams[0]), torch.cuda.graph(graph, stream=streams[0]):
        got.append(tree_attn_sharedkv(q, **kw))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o, ref[0])


@pytest.mark.gpu
def test_past_32_bit_offsets(gpu):
    """Pages at the end of a pool of over 2^31 values."""
    c = Case([2], [150], H=16, scenario=2, bs=128, ratio=2)
    pages = (1 << 22) // 128 + 20
    far = torch.empty((pages, 128, 1, D), dtype=c.dt, device="cuda")
    n, m = c.ori.shape[0], c.cmp.shape[0]
    far[-n:] = c.ori.cuda()
    far[-n - m:-n] = c.cmp.cuda()
    c.check(*c.call(ori_kv=far, cmp_kv=far, ori_block_table=(c.obt + (pages - n)).cuda(),
                    cmp_block_table=(c.cbt + (pages - n - m)).cuda()))


@pytest.mark.gpu
def test_no_tokens(gpu):
    c = Case([1], [10], H=16)
    from dsv4_b200 import tree_attn_sharedkv

    o = tree_attn_sharedkv(c.q[:0].cuda(), ori_kv=c.ori.cuda(), ori_block_table=c.obt.cuda(), seqused_kv=c.used.cuda(),
                           tree_parents=c.parents[:0].cuda(), sinks=c.sinks.cuda(), softmax_scale=c.scale,
                           cu_seqlens_q=torch.zeros(2, dtype=torch.int32).cuda())
    assert o.shape == (0, 16, D)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["dense", "top-k odd", "padded", "whole context", "top-k 3 head groups", "many requests", "one long request"])
@pytest.mark.parametrize("limit", [1000, 20000])
def test_waits_that_run_out(gpu, name, limit):
    """A limit that real waits miss: the call returns with the id of one in the status word and the next call is right.
    Pages in boxes and rows by themselves, one tile and many, cut units and whole ones."""
    from dsv4_b200 import _lib, device_status, reset_device_status

    set_limit = lambda ns: _lib.check(_lib.lib().sas_fwd_set_option(_lib.OPT_WAIT_LIMIT_NS, float(ns), None), "option")  # noqa: E731
    c = Case(**CASES[name])
    for _ in range(3):
        try:
            set_limit(limit)
            c.call()
            torch.cuda.synchronize()
        finally:
            set_limit(0)
        status = device_status()
        assert status == 0 and limit > 1000 or _lib.STATUS_TIMEOUT_BASE + 20 <= status < _lib.STATUS_TIMEOUT_BASE + 49, status
        reset_device_status()
        c.check(*c.call())
        assert device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["BSND", "TND"])
def test_more_tokens_named_than_there_are(gpu, layout):
    """cu_seqlens_q that counts more tokens than q has: the slots are still those of the append and of the framework's
    decode, seqused_kv - n on."""
    from dsv4_b200 import append_shared_kv

    c = Case([3], [40], H=8, layout=layout, trees=[[-1, 0, 1]])
    cu, used = torch.tensor([0, 5], dtype=torch.int32).cuda(), torch.tensor([45], dtype=torch.int32).cuda()
    c.check(*c.call(cu_seqlens_q=cu, seqused_kv=used))
    rows = c.ori.view(-1, D)[[int(c.obt[0, p // c.bs]) * c.bs + p % c.bs for p in (40, 41, 42)]]
    pool = torch.zeros_like(c.ori).cuda()
    kv = rows.view(1, 3, 1, D) if layout == "BSND" else rows.view(3, 1, D)
    append_shared_kv(kv.cuda(), pool, ori_block_table=c.obt.cuda(), seqused_kv=used, cu_seqlens_q=cu, layout_q=layout, norm=False)
    assert torch.equal(pool.view(-1, D).cpu().nonzero()[:, 0].unique(),
                       torch.tensor(sorted(int(c.obt[0, p // c.bs]) * c.bs + p % c.bs for p in (40, 41, 42))))


@pytest.mark.gpu
def test_writes_are_seen_by_autograd(gpu):
    c = Case([2], [30], H=8)
    out, lse = torch.empty_like(c.q, device="cuda"), torch.empty(c.T, 8, device="cuda")
    before = out._version, lse._version
    c.call(out=out, lse_out=lse)
    assert out._version > before[0] and lse._version > before[1]


@pytest.mark.gpu
@pytest.mark.parametrize("scenario", [2, 3])
def test_compressed_rows_that_end_in_the_tree(gpu, scenario):
    """The limit of the compressed rows is ctx // ratio for every token of a tree; a chain of sparse_attn_sharedkv goes to
    (position + 1) // ratio. The two agree where a chain's list or cache ends with the cached context."""
    from dsv4_b200 import sparse_attn_sharedkv

    c = Case([6], [802], H=8, scenario=scenario, ratio=4, K=256, trees=[[-1, 0, 1, 2, 3, 4]])
    full, used = c.cmp.clone(), 808
    assert 802 // 4 == 200 and (802 + 5 + 1) // 4 == 202
    if scenario == 3:
        c.idx[0, 0, :202] = torch.randperm(202, generator=torch.Generator().manual_seed(0)).to(torch.int32)
        c.idx[1:] = c.idx[0]
    out, lse = c.call()
    c.check(out, lse)  # the rows below 200
    kw = dict(ori_kv=c.ori.cuda(), ori_block_table=c.obt.cuda(), cmp_kv=full.cuda(), cmp_block_table=c.cbt.cuda(), cmp_ratio=4,
              seqused_kv=torch.tensor([used], dtype=torch.int32).cuda(), sinks=c.sinks.cuda(), softmax_scale=c.scale,
              cu_seqlens_q=torch.tensor([0, 6], dtype=torch.int32).cuda())
    if scenario == 3:
        kw["cmp_sparse_indices"] = torch.where(c.idx < 200, c.idx, -1).sort(-1, descending=True).values.contiguous().cuda()
    o, l = sparse_attn_sharedkv(c.q.cuda(), return_softmax_lse=True, **kw)
    if scenario == 3:  # lists of cached rows: the same rows in both
        c.check(o, l)
    else:  # the whole cache: the first token sees the same, the last two rows more
        c.check(o, l, skip=range(1, 6))
        assert (l[5].cpu() > lse[5].cpu()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [512, 1024])
def test_long_lists_of_many_requests(gpu, K):
    r = np.random.default_rng(K)
    lens = [int(x) for x in r.integers(0, 3, 130)]
    ctx = [int(x) for x in r.integers(0, 6000, 130)]
    lens[0], ctx[0] = 3, 6000
    c = Case(lens, ctx, H=8, scenario=3, K=K)
    c.check(*c.call())
