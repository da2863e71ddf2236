"""Head norm with rotation and the paged append, forward and backward, against 64-bit definitions.

Bounds, from the arithmetic: a value is computed in fp32 from exact 16-bit
inputs and rounded once, so it is off by at most u * |value| (u = 2^-8 for
bf16, 2^-11 for fp16; the half spacing of fp16 subnormals, 2^-25, beside it)
plus the fp32 work before it, which for D <= 1024 terms and a rotation is
below 1e-5 of the row's largest value. A weight gradient sums at most a few
hundred fp32 terms in a chain: 1e-5 of the sum of their magnitudes. A
directional derivative is compared with central differences of the 64-bit
definition (h = 1e-5: error below 1e-6 of the terms) and may be off by the
rounding of the gradient's values.
"""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 1e-5


def definition(x, w, cos, sin, inter, eps=1e-6, norm=True, inverse=False):
    """y [T, H, D] in float64; cos, sin [T, R/2] or None."""
    y = x.double()
    if norm:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w.double()
    if cos is None:
        return y
    c, s = cos.double()[:, None], sin.double()[:, None]
    s = -s if inverse else s
    h = c.shape[-1]
    a = y[..., y.shape[-1] - 2 * h:]
    x0, x1 = (a[..., 0::2], a[..., 1::2]) if inter else (a[..., :h], a[..., h:])
    r0, r1 = x0 * c - x1 * s, x0 * s + x1 * c
    rot = torch.stack([r0, r1], -1).flatten(-2) if inter else torch.cat([r0, r1], -1)
    return torch.cat([y[..., : y.shape[-1] - 2 * h], rot], -1)


def formula_bwd(dy, x, w, cos, sin, inter, eps=1e-6, norm=True, inverse=False):
    """(dx, dw, magnitude of dw's terms) in float64."""
    x = x.double()
    d = definition(dy, None, cos, sin, inter, norm=False, inverse=not inverse)
    rstd = 1 / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() if norm else torch.ones_like(x[..., :1])
    xh = x * rstd
    g = d * w.double() if w is not None else d
    dx = rstd * (g - xh * (g * xh).mean(-1, keepdim=True)) if norm else g
    return dx, (d * xh).sum((0, 1)), (d * xh).abs().sum((0, 1))


def close(got, ref, scale=None):
    got, ref = got.double().cpu(), ref.cpu()
    assert got.shape == ref.shape
    u = U[torch.bfloat16] if close.dtype is torch.bfloat16 else U[torch.float16]
    big = ref.abs().amax(-1, keepdim=True) if scale is None else scale.cpu()
    lim = u * ref.abs() + F32 * big + 2.0 ** -25
    over = (got - ref).abs() - lim
    assert not torch.isnan(got).any()
    assert over.max() <= 0, f"off by {(got - ref).abs().max():.3e}, {over.max():.3e} over the bound"


def tables(P, R, dev="cpu"):
    if R == 0:
        return None, None
    a = torch.arange(P, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return a.cos().float().to(dev), a.sin().float().to(dev)


# --------------------------------------------------------------- definitions
@pytest.mark.parametrize("inter", [True, False])
def test_formula_matches_differences(inter):
    g = torch.Generator().manual_seed(0)
    x = torch.randn((3, 2, 32), generator=g, dtype=torch.float64)
    w = 1 + 0.1 * torch.randn(32, generator=g, dtype=torch.float64)
    dy = torch.randn((3, 2, 32), generator=g, dtype=torch.float64)
    cos, sin = (t[[5, 0, 9]] for t in tables(10, 16))
    dx, dw, _ = formula_bwd(dy, x, w, cos, sin, inter)
    h = 1e-5
    for _ in range(4):
        v, vw = torch.randn(x.shape, generator=g, dtype=torch.float64), torch.randn(32, generator=g, dtype=torch.float64)
        f = lambda s: (dy * definition(x + s * h * v, w + s * h * vw, cos, sin, inter)).sum()  # noqa: E731
        num = (f(1) - f(-1)) / (2 * h)
        assert abs(num - (dx * v).sum() - (dw * vw).sum()) <= 1e-6 * (dx.abs().sum() + dw.abs().sum())


# ------------------------------------------------------------------ refusals
def _qk(T=2, H=4, D=64, dtype=torch.bfloat16):
    return torch.zeros(T, H, D, dtype=dtype), torch.zeros(T, 1, D, dtype=dtype)


def test_norm_rope_refusals():
    from dsv4_b200 import head_norm_rope, head_norm_rope_backward, head_norm_rope_train

    q, k = _qk()
    cos, sin = tables(8, 32)
    pos = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        head_norm_rope(q.float())
    with pytest.raises(ValueError):
        head_norm_rope(torch.zeros(2, 4, 60, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        head_norm_rope(torch.zeros(2, 4, 1032, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        head_norm_rope(q, k.half())
    with pytest.raises(ValueError):
        head_norm_rope(q, k[:1])
    with pytest.raises(ValueError):
        head_norm_rope(q, cos=cos, sin=sin)  # no positions
    with pytest.raises(ValueError):
        head_norm_rope(q, cos=cos, positions=pos)
    with pytest.raises(ValueError):
        head_norm_rope(q, cos=cos, sin=sin, positions=pos[:1])
    with pytest.raises(ValueError):
        head_norm_rope(q, cos=cos, sin=sin, positions=pos.float())
    with pytest.raises(ValueError):
        head_norm_rope(q, cos=cos[:, :6], sin=sin[:, :6], positions=pos)
    with pytest.raises(ValueError):
        head_norm_rope(q, cos=cos[:, :12], sin=sin[:, :12], positions=pos, interleaved=False)
    with pytest.raises(ValueError):
        head_norm_rope(q, q_weight=torch.ones(32))
    with pytest.raises(ValueError):
        head_norm_rope(q, q_out=torch.zeros(2, 4, 32, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        head_norm_rope_backward(q[:1], q)
    with pytest.raises(AssertionError):
        head_norm_rope(q, q_weight=torch.ones(64), norm=False)
    with pytest.raises(AssertionError):
        head_norm_rope_train(q, q_out=q)
    with pytest.raises(RuntimeError, match="CUDA"):
        head_norm_rope(q, k, cos=cos, sin=sin, positions=pos)


def test_append_refusals():
    from dsv4_b200 import append_shared_kv, append_shared_kv_backward

    kv = torch.zeros(3, 1, 64, dtype=torch.bfloat16)
    pool = torch.zeros(4, 16, 1, 64, dtype=torch.bfloat16)
    kw = dict(ori_block_table=torch.zeros(2, 2, dtype=torch.int32), seqused_kv=torch.tensor([4, 9], dtype=torch.int32),
              cu_seqlens_q=torch.tensor([0, 1, 3], dtype=torch.int32))
    for fn in (lambda **o: append_shared_kv(o.pop("kv", kv), o.pop("pool", pool), **{**kw, **o}),
               lambda **o: append_shared_kv_backward(o.pop("pool", pool), o.pop("kv", kv), **{**kw, **o})):
        with pytest.raises(ValueError):
            fn(pool=pool.half())
        with pytest.raises(ValueError):
            fn(pool=pool[:, :, 0])
        with pytest.raises(ValueError):
            fn(pool=pool.transpose(0, 1))
        with pytest.raises(ValueError):
            fn(kv=kv[..., :32])
        with pytest.raises(ValueError):
            fn(seqused_kv=torch.tensor([4], dtype=torch.int32))
        with pytest.raises(ValueError):
            fn(ori_block_table=torch.zeros(3, 2, dtype=torch.int32))
        with pytest.raises(ValueError):
            fn(layout_q="BSND")
        with pytest.raises(AssertionError):
            fn(cu_seqlens_q=None)
        with pytest.raises(AssertionError):
            fn(layout_q="BSH")
        with pytest.raises(AssertionError):
            fn(weight=torch.ones(64), norm=False)
        with pytest.raises(RuntimeError, match="CUDA"):
            fn()
    with pytest.raises(ValueError):
        append_shared_kv(kv, pool, q=torch.zeros(2, 4, 64, dtype=torch.bfloat16), **kw)


# ----------------------------------------------------------------------- GPU
@pytest.fixture
def gpu(sas_lib):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from dsv4_b200 import check_device_status, reset_device_status

    reset_device_status()
    yield
    check_device_status()


CASES = [  # T, H, Hk, D, R, interleaved, q weight, k weight
    (1, 1, 0, 64, 64, True, False, False),
    (1, 64, 1, 512, 64, True, False, True),
    (7, 5, 3, 128, 32, False, True, True),
    (33, 24, 1, 192, 64, True, True, False),
    (17, 3, 2, 1024, 128, False, True, True),
    (5, 128, 1, 512, 512, True, True, True),
    (40, 7, 1, 64, 16, False, False, False),
    (129, 16, 4, 128, 0, True, True, True),
    (9, 2, 1, 8, 8, True, True, True),
    (700, 56, 1, 512, 64, True, True, True),  # several rows in flight, many partial sums
    (701, 57, 1, 512, 64, False, True, True),
    (3, 1, 1, 768, 96, False, False, True),
    (310, 40, 8, 128, 128, False, True, True),
    (2, 3, 1, 1024, 1024, False, True, True),  # the most shared memory
    (50, 9, 2, 256, 64, True, True, False),
    (4, 2, 0, 320, 48, True, True, False),
]


def _case(T, H, Hk, D, R, qw, kw, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = lambda h: (2 * torch.randn((T, h, D), generator=g)).to(dt) if h else None  # noqa: E731
    q, k = x(H), x(Hk)
    cos, sin = tables(300, R)
    pos = torch.randint(0, 300, (T,), generator=g, dtype=torch.int32)
    w = lambda on: 1 + 0.1 * torch.randn(D, generator=g) if on else None  # noqa: E731
    return q, k, cos, sin, pos if R else None, w(qw), w(kw and Hk), (x(H), x(Hk))


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _rows(cos, sin, pos):
    return (None, None) if cos is None else (cos[pos.long()], sin[pos.long()])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("cfg", CASES, ids=lambda c: "-".join(map(str, c)))
def test_norm_rope_and_backward(gpu, cfg, dt):
    from dsv4_b200 import head_norm_rope, head_norm_rope_backward

    close.dtype = dt
    T, H, Hk, D, R, inter, qwo, kwo = cfg
    q, k, cos, sin, pos, qw, kw, (dq, dk) = _case(T, H, Hk, D, R, qwo, kwo, dt)
    c, s = _rows(cos, sin, pos)
    dev = _cuda(q, k, cos, sin, pos, qw, kw, dq, dk)
    args = dict(positions=dev[4], cos=dev[2], sin=dev[3], q_weight=dev[5], k_weight=dev[6], interleaved=inter)
    r = head_norm_rope(dev[0], dev[1], **args)
    yq, yk = r if k is not None else (r, None)
    close(yq, definition(q, qw, c, s, inter))
    if k is not None:
        close(yk, definition(k, kw, c, s, inter))
    gq, gk, gqw, gkw = head_norm_rope_backward(dev[7], dev[0], dev[8], dev[1], **args)
    for got, gw, x, w, dy in ((gq, gqw, q, qw, dq), (gk, gkw, k, kw, dk)):
        if x is None:
            assert got is None and gw is None
            continue
        dx, dw, mag = formula_bwd(dy, x, w, c, s, inter)
        rstd = 1 / (x.double().pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        close(got, dx, dx.abs().amax(-1, keepdim=True) + 4 * rstd * dy.double().abs().amax(-1, keepdim=True))
        assert (gw is None) == (w is None)
        if w is not None:
            assert gw.dtype == torch.float32
            assert ((gw.double().cpu() - dw).abs() <= F32 * mag).all()
    again = head_norm_rope_backward(dev[7], dev[0], dev[8], dev[1], **args)
    for a, b in zip((gq, gk, gqw, gkw), again):
        assert a is None and b is None or torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [True, False])
def test_gradient_against_differences(gpu, inter):
    from dsv4_b200 import head_norm_rope_backward

    dt = torch.float16
    q, _, cos, sin, pos, w, _, (dy, _) = _case(6, 4, 0, 128, 64, True, False, dt, seed=3)
    c, s = _rows(cos, sin, pos)
    dev = _cuda(dy, q, pos, cos, sin, w)
    dx, _, dw, _ = head_norm_rope_backward(dev[0], dev[1], positions=dev[2], cos=dev[3], sin=dev[4], q_weight=dev[5],
                                           interleaved=inter)
    dx, dw = dx.double().cpu(), dw.double().cpu()
    g = torch.Generator().manual_seed(1)
    h = 1e-5
    for _ in range(3):
        v, vw = torch.randn(q.shape, generator=g, dtype=torch.float64), torch.randn(128, generator=g, dtype=torch.float64)
        f = lambda t: (dy.double() * definition(q.double() + t * h * v, w.double() + t * h * vw, c, s, inter)).sum()  # noqa: E731
        num = (f(1) - f(-1)) / (2 * h)
        lim = U[dt] * (dx * v).abs().sum() + F32 * ((dw * vw).abs().sum() + dx.abs().sum())
        assert abs(num - (dx * v).sum() - (dw * vw).sum()) <= lim


@pytest.mark.gpu
def test_norm_rope_layouts_and_modes(gpu):
    """Strided inputs and results, in place, BSND, int64 positions, no norm, turning back, another stream, a graph."""
    from dsv4_b200 import head_norm_rope

    close.dtype = dt = torch.bfloat16
    T, H, D, R = 24, 6, 128, 64
    fused = (2 * torch.randn(T, H + 2, D + 8)).to(dt).cuda()
    q, k = fused[:, :H, :D], fused[:, H:, :D]  # a slice of a fused projection
    cos, sin = tables(64, R, "cuda")
    pos = torch.randint(0, 64, (T,)).cuda()
    for inter in (True, False):
        kw = dict(positions=pos, cos=cos, sin=sin, interleaved=inter)
        cpu = lambda x, **o: definition(x.cpu(), None, cos[pos].cpu(), sin[pos].cpu(), inter, **o)  # noqa: E731
        store = torch.zeros(T, H, D + 16, dtype=dt, device="cuda")
        yq, yk = head_norm_rope(q, k, q_out=store[..., :D], **kw)
        assert yq.data_ptr() == store.data_ptr() and not store[..., D:].any()
        close(yq, cpu(q))
        close(yk, cpu(k))
        odd = torch.randn(T * H * D + 1).to(dt).cuda()[1:].view(T, H, D)  # not 16-byte aligned: copied
        close(head_norm_rope(odd, **kw), cpu(odd))
        y4 = head_norm_rope(q.reshape(4, 6, H, D), **{**kw, "positions": pos.view(4, 6).int()})
        assert torch.equal(y4.view(T, H, D), yq)
        mine = q.contiguous()
        head_norm_rope(mine, q_out=mine, **kw)
        assert torch.equal(mine, yq)
        back = head_norm_rope(yq, norm=False, inverse=True, **kw)
        close(back, cpu(yq, norm=False, inverse=True))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = head_norm_rope(q, k, **kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = head_norm_rope(q, k, **kw)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for got in (other, held):
        assert torch.equal(got[0], yq) and torch.equal(got[1], yk)
    assert head_norm_rope(q[:0], positions=pos[:0], cos=cos, sin=sin).shape == (0, H, D)


@pytest.mark.gpu
def test_norm_of_extreme_rows(gpu):
    """Zero rows, rows whose squares leave bf16's range, infinities and NaN: as the definition in fp32 gives."""
    from dsv4_b200 import head_norm_rope, head_norm_rope_backward

    close.dtype = dt = torch.bfloat16
    x = torch.randn(5, 1, 64).to(dt)
    x[0] = 0
    x[1] *= 1e-18
    x[2] *= 1e15
    y = head_norm_rope(x[:3].cuda())
    close(y, definition(x[:3], None, None, None, True))
    x[3, 0, 5] = float("nan")
    x[4, 0, 5] = float("inf")
    y = head_norm_rope(x.cuda()).float().cpu()
    assert torch.isnan(y[3]).all() and torch.isnan(y[4, 0, 5]) and not torch.isnan(y[:3]).any()
    d = head_norm_rope_backward(torch.randn(5, 1, 64).to(dt).cuda(), x.cuda())[0]
    assert not torch.isnan(d[:3]).any()


@pytest.mark.gpu
def test_position_outside_the_tables_is_recorded(gpu):
    from dsv4_b200 import device_status, head_norm_rope, reset_device_status

    cos, sin = tables(8, 32, "cuda")
    q = torch.randn(3, 2, 64).bfloat16().cuda()
    near = head_norm_rope(q, positions=torch.tensor([0, 7, 7], device="cuda"), cos=cos, sin=sin)
    got = head_norm_rope(q, positions=torch.tensor([-4, 8, 1 << 40], device="cuda"), cos=cos, sin=sin)
    assert device_status() == 8
    reset_device_status()
    assert torch.equal(got, near)


@pytest.mark.gpu
def test_train_matches_backward(gpu):
    from dsv4_b200 import head_norm_rope_backward, head_norm_rope_train

    q, k, cos, sin, pos, qw, kw, (dq, dk) = _case(12, 4, 1, 64, 32, True, True, torch.bfloat16)
    q, k, cos, sin, pos, qw, kw, dq, dk = _cuda(q, k, cos, sin, pos, qw, kw, dq, dk)
    args = dict(positions=pos, cos=cos, sin=sin)
    ref = head_norm_rope_backward(dq, q, dk, k, q_weight=qw, k_weight=kw, **args)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    yq, yk = head_norm_rope_train(q, k, q_weight=qw, k_weight=kw, **args)
    torch.autograd.backward([yq, yk], [dq, dk])
    for leaf, r in zip(leaves, ref):
        assert torch.equal(leaf.grad, r)
    y = head_norm_rope_train(q.detach().requires_grad_(), **args)
    y.backward(dq)


def _paged(lens, ctx, bs, D, dt, seed, spare=2, blocks=None):
    g = torch.Generator().manual_seed(seed)
    used = [a + b for a, b in zip(lens, ctx)]
    nb = [max(1, -(-u // bs)) for u in used]
    total = sum(nb) + spare
    perm = torch.randperm(total, generator=g)
    table = torch.full((len(lens), max(nb) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(nb):
        table[b, :n] = perm[at:at + n]
        at += n
    pool = torch.randn((total, bs, 1, D), generator=g).to(dt)
    rows = [int(table[b, p // bs]) * bs + p % bs for b, (n, x) in enumerate(zip(lens, ctx)) for p in range(x, x + n)]
    slots = [p for n, x in zip(lens, ctx) for p in range(x, x + n)]
    return pool, table, torch.tensor(used, dtype=torch.int32), torch.tensor(rows), torch.tensor(slots)


APPENDS = [  # tokens of each request, rows before them, page size, q heads, interleaved, layout
    ([1], [0], 1, 0, True, "TND"),
    ([1, 1, 1], [5, 0, 127], 16, 8, True, "TND"),
    ([3, 0, 9, 1], [0, 7, 61, 200], 48, 3, False, "TND"),
    ([5, 5], [11, 123], 64, 16, True, "BSND"),
    ([1] * 1100, [i % 70 for i in range(1100)], 32, 0, True, "TND"),  # more requests than one search round
    ([700, 1], [3, 3], 128, 64, True, "TND"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("cfg", APPENDS, ids=range(len(APPENDS)))
def test_append_and_backward(gpu, cfg, dt):
    from dsv4_b200 import append_shared_kv, append_shared_kv_backward

    close.dtype = dt
    lens, ctx, bs, H, inter, layout = cfg
    D = 128 if bs == 32 else 512
    pool, table, used, rows, slots = _paged(lens, ctx, bs, D, dt, 1)
    T = sum(lens)
    g = torch.Generator().manual_seed(2)
    kv = (2 * torch.randn((T, 1, D), generator=g)).to(dt)
    q = (2 * torch.randn((T, H, D), generator=g)).to(dt) if H else None
    w = 1 + 0.1 * torch.randn(D, generator=g)
    cos, sin = tables(1200, 64)
    given = torch.randint(0, 1200, (T,), generator=g, dtype=torch.int32)
    shape = (lambda t: t.view(len(lens), lens[0], *t.shape[1:])) if layout == "BSND" else (lambda t: t)
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32).cuda() if layout == "TND" else None
    for pos in (None, given):
        at = (slots if pos is None else pos).long()
        args = dict(ori_block_table=table.cuda(), seqused_kv=used.cuda(), cu_seqlens_q=cu, layout_q=layout,
                    positions=None if pos is None else shape(pos).cuda(), cos=cos.cuda(), sin=sin.cuda(),
                    weight=w.cuda(), interleaved=inter)
        dev = pool.cuda()
        r = append_shared_kv(shape(kv).cuda(), dev, q=None if q is None else shape(q).cuda(), **args)
        out, yq = r if q is not None else (r, None)
        assert out is dev
        want = definition(kv, w, cos[at], sin[at], inter)
        flat = dev.view(-1, 1, D)
        close(flat[rows.cuda()], want)
        rest = torch.ones(flat.shape[0], dtype=torch.bool)
        rest[rows] = False
        assert torch.equal(flat.cpu()[rest], pool.view(-1, 1, D)[rest]), "a row that is not the tokens' changed"
        if q is not None:
            close(yq.reshape(T, H, D), definition(q, None, cos[at], sin[at], inter))
        dpool = torch.randn(pool.shape, generator=g).to(dt)
        dkv, dw = append_shared_kv_backward(dpool.cuda(), shape(kv).cuda(), **args)
        dy = dpool.view(-1, 1, D)[rows]
        dx, rw, mag = formula_bwd(dy, kv, w, cos[at], sin[at], inter)
        rstd = 1 / (kv.double().pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        close(dkv.reshape(T, 1, D), dx, dx.abs().amax(-1, keepdim=True) + 4 * rstd * dy.double().abs().amax(-1, keepdim=True))
        assert ((dw.double().cpu() - rw).abs() <= F32 * mag).all()


@pytest.mark.gpu
def test_append_skips_what_has_no_row(gpu):
    """Negative table entries are skipped; entries past the pool and columns past the table are skipped and recorded.
    The pool is declared smaller than its allocation, so that even an unchecked write would stay inside it."""
    from dsv4_b200 import append_shared_kv, append_shared_kv_backward, device_status, reset_device_status

    D, bs = 64, 4
    whole = torch.randn(8, bs, 1, D).bfloat16().cuda()
    kv = torch.randn(6, 1, D).bfloat16().cuda()
    cu = torch.tensor([0, 2, 4, 6], dtype=torch.int32, device="cuda")
    for table, used, code in (([[1], [-1], [2]], [2, 2, 2], 0), ([[1], [6], [2]], [2, 2, 2], 7), ([[1], [3], [2]], [2, 6, 2], 7),
                              ([[1], [3], [2]], [2, 1, 2], 0)):
        pool = whole.clone()
        args = dict(ori_block_table=torch.tensor(table, dtype=torch.int32, device="cuda"),
                    seqused_kv=torch.tensor(used, dtype=torch.int32, device="cuda"), cu_seqlens_q=cu)
        append_shared_kv(kv, pool[:4], **args)
        assert device_status() == code
        reset_device_status()
        good = definition(kv.cpu(), None, None, None, True)
        close.dtype = torch.bfloat16
        close(pool[1, :2], good[:2])
        close(pool[2, :2], good[4:])
        if used[1] == 1:  # its first token lies before slot 0
            close(pool[3, :1], good[3:4])
            pool[3, :1] = whole[3, :1]
        pool[1, :2], pool[2, :2] = whole[1, :2], whole[2, :2]
        assert torch.equal(pool, whole)
        dkv, _ = append_shared_kv_backward(whole[:4], kv, **args)
        reset_device_status()
        assert not dkv[2].any() and dkv[0].any() and dkv[4].any() and dkv[3].any() == (used[1] == 1)


@pytest.mark.gpu
def test_append_past_32_bit_offsets(gpu):
    from dsv4_b200 import append_shared_kv, append_shared_kv_backward

    close.dtype = torch.bfloat16
    blocks, bs, D = (1 << 22) // 128 + 40, 128, 512  # the pool holds over 2^31 values
    pool = torch.empty((blocks, bs, 1, D), dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[blocks - 1], [blocks - 7]], dtype=torch.int32, device="cuda")
    used = torch.tensor([128, 2], dtype=torch.int32, device="cuda")
    kv = torch.randn(3, 1, D).bfloat16().cuda()
    args = dict(ori_block_table=table, seqused_kv=used, cu_seqlens_q=torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"))
    append_shared_kv(kv, pool, **args)
    want = definition(kv.cpu(), None, None, None, True)
    close(torch.cat([pool[-1, 127:], pool[-7, :2]]), want)
    dkv, _ = append_shared_kv_backward(pool, kv, **args)
    assert dkv.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,H,Hk", [(64, 1, 0), (64, 3, 1), (64, 6, 5), (128, 1, 1), (128, 7, 3)])
def test_weight_gradient_without_eps(gpu, D, H, Hk):
    """Heads that do not fill a warp's lanes, with eps 0: the lanes without a row add nothing."""
    from dsv4_b200 import head_norm_rope_backward

    close.dtype = torch.bfloat16
    q, k, cos, sin, pos, qw, kw, (dq, dk) = _case(9, H, Hk, D, 32, True, True, torch.bfloat16, seed=5)
    c, s = _rows(cos, sin, pos)
    dev = _cuda(dq, q, dk, k, pos, cos, sin, qw, kw)
    got = head_norm_rope_backward(*dev[:4], positions=dev[4], cos=dev[5], sin=dev[6], q_weight=dev[7], k_weight=dev[8], eps=0.0)
    for gx, gw, x, w, dy in ((got[0], got[2], q, qw, dq), (got[1], got[3], k, kw, dk)):
        if x is None:
            continue
        dx, dw, mag = formula_bwd(dy, x, w, c, s, True, eps=0.0)
        rstd = 1 / x.double().pow(2).mean(-1, keepdim=True).sqrt()
        close(gx, dx, dx.abs().amax(-1, keepdim=True) + 4 * rstd * dy.double().abs().amax(-1, keepdim=True))
        assert ((gw.double().cpu() - dw).abs() <= F32 * mag).all()


def _unwritten():
    """(name, layout, cu_seqlens_q, tokens, table, seqused_kv, tokens without a row) of appends of 12 tokens."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    full = [[0, 1], [2, 3], [4, 5]]
    return [
        ("padding of BSND", "BSND", i32([0, 4, 5, 8]), (3, 4), i32(full), i32([9, 3, 8]), [5, 6, 7, 11]),
        ("an empty request of BSND", "BSND", i32([0, 4, 4, 6]), (3, 4), i32(full), i32([4, 0, 8]), [4, 5, 6, 7, 10, 11]),
        ("after the last request of TND", "TND", i32([0, 4, 5, 9]), (12,), i32(full), i32([9, 3, 8]), [9, 10, 11]),
        ("without a page", "TND", i32([0, 4, 8, 12]), (12,), i32([[0, 1], [-1, 3], [4, -1]]), i32([9, 10, 9]), [4, 5, 11]),
        ("before slot 0", "TND", i32([0, 4, 8, 12]), (12,), i32(full), i32([9, 2, 8]), [4, 5]),
    ]


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 192, 512])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 0.0])
@pytest.mark.parametrize("which", range(5))
def test_append_backward_of_unwritten_rows(gpu, which, bad, D):
    """They get zero and leave the weight's gradient alone, whatever they hold; zeros with eps 0 too."""
    from dsv4_b200 import append_shared_kv_backward

    close.dtype = torch.bfloat16
    name, layout, cu, lead, table, used, unwritten = _unwritten()[which]
    eps = 1e-6 if bad else 0.0
    g = torch.Generator().manual_seed(7)
    kv = (2 * torch.randn((12, 1, D), generator=g)).bfloat16()
    kv[unwritten] = bad
    w = 1 + 0.1 * torch.randn(D, generator=g)
    dpool = torch.randn((6, 8, 1, D), generator=g).bfloat16()
    dkv, dw = append_shared_kv_backward(dpool.cuda(), kv.view(*lead, 1, D).cuda(), ori_block_table=table, seqused_kv=used,
                                        cu_seqlens_q=cu, layout_q=layout, weight=w.cuda(), eps=eps)
    dkv = dkv.cpu().view(12, 1, D)
    assert not dkv[unwritten].any(), name
    written = [t for t in range(12) if t not in unwritten]
    cu, used, table, S = cu.tolist(), used.tolist(), table.tolist(), lead[-1]
    rows = []
    for t in written:
        b = t // S if layout == "BSND" else max(b for b in range(3) if cu[b] <= t)
        p = used[b] - (cu[b + 1] - cu[b]) + t - (b * S if layout == "BSND" else cu[b])
        rows.append(table[b][p // 8] * 8 + p % 8)
    dy, x = dpool.view(-1, 1, D)[rows], kv[written]
    dx, rw, mag = formula_bwd(dy, x, w, None, None, True, eps=eps)
    rstd = 1 / (x.double().pow(2).mean(-1, keepdim=True) + eps).sqrt()
    close(dkv[written], dx, dx.abs().amax(-1, keepdim=True) + 4 * rstd * dy.double().abs().amax(-1, keepdim=True))
    assert ((dw.double().cpu() - rw).abs() <= F32 * mag).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 512])
def test_append_backward_of_long_padding(gpu, D):
    """Warps that walk over several tokens, runs of padding that hold NaN among them."""
    from dsv4_b200 import append_shared_kv_backward

    close.dtype = torch.bfloat16
    B, S, bs = 40, 400, 16
    r = np.random.default_rng(3)
    lens = [0, S, 1, *(int(x) for x in r.integers(0, S + 1, B - 3))]
    pool, table, used, rows, _ = _paged(lens, [int(x) for x in r.integers(0, 40, B)], bs, D, torch.bfloat16, 3)
    held = torch.zeros(B, S, dtype=torch.bool)
    for b, n in enumerate(lens):
        held[b, :n] = True
    held = held.view(-1)
    g = torch.Generator().manual_seed(5)
    kv = torch.randn((B * S, 1, D), generator=g).bfloat16()
    kv[~held] = float("nan")
    w = 1 + 0.1 * torch.randn(D, generator=g)
    dkv, dw = append_shared_kv_backward(pool.cuda(), kv.view(B, S, 1, D).cuda(), ori_block_table=table.cuda(),
                                        seqused_kv=used.cuda(), layout_q="BSND", weight=w.cuda(),
                                        cu_seqlens_q=torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32).cuda())
    dkv = dkv.cpu().view(-1, 1, D)
    assert not dkv[~held].any()
    dy, x = pool.view(-1, 1, D)[rows], kv[held]
    dx, rw, mag = formula_bwd(dy, x, w, None, None, True)
    rstd = 1 / (x.double().pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
    close(dkv[held], dx, dx.abs().amax(-1, keepdim=True) + 4 * rstd * dy.double().abs().amax(-1, keepdim=True))
    assert ((dw.double().cpu() - rw).abs() <= F32 * mag).all()


@pytest.mark.gpu
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("bad", [None, float("nan"), float("inf")])
def test_backward_without_norm(gpu, bad, inter, inverse):
    """The rotation's transpose of the gradient alone: the inputs, finite or not, have no part in it."""
    from dsv4_b200 import head_norm_rope_backward

    close.dtype = torch.float16
    q, k, cos, sin, pos, _, _, (dq, dk) = _case(11, 5, 2, 128, 64, False, False, torch.float16, seed=6)
    c, s = _rows(cos, sin, pos)
    if bad is not None:
        q[3], k[5, 1, ::3] = bad, -bad
    dev = _cuda(dq, q, dk, k, pos, cos, sin)
    got = head_norm_rope_backward(*dev[:4], positions=dev[4], cos=dev[5], sin=dev[6], norm=False, inverse=inverse, interleaved=inter)
    for gx, dy in ((got[0], dq), (got[1], dk)):
        close(gx, definition(dy, None, c, s, inter, norm=False, inverse=not inverse))
    assert got[2] is None and got[3] is None


@pytest.mark.gpu
@pytest.mark.parametrize("H", [0, 6])
@pytest.mark.parametrize("which", [0, 1, 2, 4])
def test_positions_of_tokens_without_a_slot(gpu, which, H):
    """Positions outside the tables are recorded for tokens with a slot alone: padding may hold anything. The nearest row
    of the tables turns it."""
    from dsv4_b200 import append_shared_kv, append_shared_kv_backward, device_status, reset_device_status

    D = 64
    name, layout, cu, lead, table, used, unwritten = _unwritten()[which]
    g = torch.Generator().manual_seed(8)
    kv = torch.randn((12, 1, D), generator=g).bfloat16().view(*lead, 1, D).cuda()
    q = torch.randn((12, H, D), generator=g).bfloat16().view(*lead, H, D).cuda() if H else None
    pool = torch.randn((6, 8, 1, D), generator=g).bfloat16()
    cos, sin = tables(16, 32, "cuda")
    pos = torch.arange(12) + 2
    first = pos.clone()
    first[unwritten] = 0
    args = dict(ori_block_table=table, seqused_kv=used, cu_seqlens_q=cu, layout_q=layout, cos=cos, sin=sin)

    def both(positions):
        args["positions"] = positions.view(lead).cuda()
        r = append_shared_kv(kv, pool.cuda(), q=q, **args)
        return (*(r if H else (r,)), append_shared_kv_backward(pool.cuda(), kv, **args)[0])

    for x in (-1, 16, 1 << 40, -(1 << 40)):
        fill = torch.where(first == 0, torch.tensor(x), first)
        got, want = both(fill), both(fill.clamp(0, 15))
        assert device_status() == 0, name
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    written = next(t for t in range(12) if t not in unwritten)
    fill = first.clone()
    fill[written] = 16
    args["positions"] = fill.view(lead).cuda()
    for call in (lambda: append_shared_kv(kv, pool.cuda(), q=q, **args), lambda: append_shared_kv_backward(pool.cuda(), kv, **args)):
        call()
        assert device_status() == 8
        reset_device_status()


@pytest.mark.gpu
def test_writes_are_seen_by_autograd(gpu):
    """What a call writes in place of a tensor that a backward saved is an error of that backward, as of torch's own."""
    from dsv4_b200 import append_shared_kv, head_norm_rope, sparse_attn_sharedkv_train

    D, dt = 512, torch.bfloat16
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = torch.randn(2, 16, 1, D, device="cuda").to(dt)
    q = torch.randn(3, 8, D, device="cuda").to(dt).requires_grad_()
    table, used = i32(0, 1).view(1, 2), i32(20)
    args = dict(ori_block_table=table, cu_seqlens_q=i32(0, 3))
    out = sparse_attn_sharedkv_train(q, ori_kv=pool, sinks=torch.zeros(8, device="cuda"), softmax_scale=D ** -0.5,
                                     seqused_kv=used, **args)
    append_shared_kv(torch.randn(3, 1, D, device="cuda").to(dt), pool, seqused_kv=used, **args)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    x, y = (torch.randn(3, 8, D, device="cuda").to(dt) for _ in range(2))
    before = [t._version for t in (x, y, pool)]
    head_norm_rope(x, y, q_out=x, k_out=y)
    append_shared_kv(y[:, :1], pool, seqused_kv=used, q=x, q_out=x, **args)
    assert all(t._version > v for t, v in zip((x, y, pool), before)) and x._version == before[0] + 2
    with torch.inference_mode():  # tensors without versions
        z = torch.randn(3, 8, D, device="cuda").to(dt)
        head_norm_rope(z, q_out=z)


def _on_cpu(monkeypatch):
    """``head_norm_rope`` and its backward as far as autograd sees them: a result and gradients that know the positions."""
    from dsv4_b200 import rope

    calls = []

    def fwd(q, k=None, **kw):
        calls.append(("forward", kw))
        return q * 1 if k is None else (q * 1, k * 1)

    def bwd(dq_out, q, dk_out=None, k=None, **kw):
        calls.append(("backward", kw))
        s = 1 if kw.get("positions") is None else int(kw["positions"].sum())
        w = [None if kw.get(n) is None else torch.ones_like(kw[n]) for n in ("q_weight", "k_weight")]
        return dq_out * s, None if k is None else dk_out * s, *w

    monkeypatch.setattr(rope, "head_norm_rope", fwd)
    monkeypatch.setattr(rope, "head_norm_rope_backward", bwd)
    return calls


def test_train_keeps_its_positions(monkeypatch):
    """A buffer of positions or angles that is refilled before the backward is an error, not the wrong gradient."""
    from dsv4_b200 import head_norm_rope_train

    calls = _on_cpu(monkeypatch)
    cos, sin = tables(8, 32)
    pos = torch.tensor([1, 2], dtype=torch.int32)
    args = dict(positions=pos, cos=cos, sin=sin, eps=1e-5, interleaved=False)
    q, k = (t.float().requires_grad_() for t in _qk())
    w = torch.ones(64, requires_grad=True)
    yq, yk = head_norm_rope_train(q, k, q_weight=w, **args)
    torch.autograd.backward([yq, yk], [torch.ones_like(yq), torch.ones_like(yk)])
    assert (q.grad == 3).all() and (k.grad == 3).all() and (w.grad == 1).all()
    (_, f), (_, b) = calls
    for n, x in args.items():
        assert f[n] is x if not torch.is_tensor(x) else f[n].data_ptr() == x.data_ptr() == b[n].data_ptr()
        assert torch.is_tensor(x) or b[n] == x
    assert set(f) == set(b)
    for held in (pos, cos, sin):
        y = head_norm_rope_train(q, **args)
        held += 1
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()
    head_norm_rope_train(q).sum().backward()  # without positions


def test_train_is_once_differentiable(monkeypatch):
    from dsv4_b200 import head_norm_rope_train

    _on_cpu(monkeypatch)
    q = torch.ones(2, 4, 64, requires_grad=True)
    g, = torch.autograd.grad(head_norm_rope_train(q).pow(2).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_train_takes_absent_outputs(monkeypatch):
    from dsv4_b200 import head_norm_rope_train

    q = torch.ones(2, 4, 64, requires_grad=True)
    calls = _on_cpu(monkeypatch)
    head_norm_rope_train(q, q_out=None, k_out=None).sum().backward()
    assert all("q_out" not in kw and "k_out" not in kw for _, kw in calls)  # the backward has no such arguments
    assert (q.grad == 1).all()


def test_overlap_of_rows():
    from dsv4_b200.rope import _overlap

    g = np.random.default_rng(0)
    for _ in range(3000):
        T, H, D = (int(g.integers(1, n)) for n in (6, 6, 5))
        ts, hs = (int(x) for x in g.integers(0, 20, 2))
        at = np.arange(T)[:, None] * ts + np.arange(H) * hs
        values = (at.reshape(-1, 1) + np.arange(D)).reshape(-1)
        assert _overlap(ts, T, hs, H, D) == (len(np.unique(values)) < len(values)), (ts, T, hs, H, D)


@pytest.mark.gpu
def test_outputs_whose_rows_overlap_are_refused(gpu):
    from dsv4_b200 import append_shared_kv, head_norm_rope

    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    base = torch.zeros(3, 4, 64, device="cuda").bfloat16()
    for out in (base[:1].expand(3, 4, 64), base[:, :1].expand(3, 4, 64), base.view(-1).as_strided((3, 4, 64), (256, 32, 1)),
                base.view(-1).as_strided((3, 4, 64), (56, 192, 1)),
                base.view(-1).as_strided((3, 4, 64), (64, 64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            head_norm_rope(q, q_out=out)
    with pytest.raises(ValueError, match="overlap"):
        append_shared_kv(q[:, :1], base[:, :, None], ori_block_table=torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                         seqused_kv=torch.full((1,), 3, dtype=torch.int32, device="cuda"),
                         cu_seqlens_q=torch.tensor([0, 3], dtype=torch.int32, device="cuda"), q=q, q_out=base[:1].expand(3, 4, 64))
    assert not base.any()
    by_head = torch.zeros(4, 3, 72, device="cuda").bfloat16().transpose(0, 1)[..., :64]  # a head's tokens side by side
    assert torch.equal(head_norm_rope(q, q_out=by_head), head_norm_rope(q))


@pytest.mark.gpu
def test_train_without_keys_matches_backward(gpu):
    from dsv4_b200 import head_norm_rope_backward, head_norm_rope_train

    q, _, cos, sin, pos, _, _, (dq, _) = _case(12, 4, 0, 64, 32, False, False, torch.bfloat16)
    q, cos, sin, pos, dq = _cuda(q, cos, sin, pos, dq)
    ref = head_norm_rope_backward(dq, q, positions=pos, cos=cos, sin=sin)[0]
    x = q.clone().requires_grad_()
    head_norm_rope_train(x, positions=pos, cos=cos, sin=sin).backward(dq)
    assert ref.any() and torch.equal(x.grad, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 512])
def test_gradient_has_no_part_along_the_row(gpu, D):
    """The norm does not depend on a row's length, so sum(dx x) is zero (but for eps) where there is no weight: every
    product is off by the rounding of dx, and the term that the norm's projection takes out is far larger."""
    from dsv4_b200 import head_norm_rope_backward

    q, _, cos, sin, pos, _, _, (dq, _) = _case(40, 6, 0, D, 32, False, False, torch.bfloat16, seed=9)
    dev = _cuda(dq, q, pos, cos, sin)
    dx = head_norm_rope_backward(dev[0], dev[1], positions=dev[2], cos=dev[3], sin=dev[4])[0].double().cpu()
    x = q.double()
    dot, mag = (dx * x).sum(-1).abs(), (dx * x).abs().sum(-1)
    assert (dot <= U[torch.bfloat16] * mag).all()
    d = definition(dq, None, *_rows(cos, sin, pos), True, norm=False, inverse=True)  # without the projection
    assert ((d * x).sum(-1).abs() > 4 * U[torch.bfloat16] * (d * x).abs().sum(-1)).double().mean() > 0.5


@pytest.mark.gpu
def test_append_of_padded_bsnd_and_int64_positions(gpu):
    from dsv4_b200 import append_shared_kv

    close.dtype = torch.bfloat16
    B, S, D, H = 3, 5, 128, 3
    lens, ctx = [5, 2, 0], [11, 40, 9]
    pool, table, used, rows, slots = _paged(lens, ctx, 16, D, torch.bfloat16, 4)
    g = torch.Generator().manual_seed(4)
    kv = torch.randn((B, S, 1, D), generator=g).bfloat16()
    q = torch.randn((B, S, H, D), generator=g).bfloat16()
    held = torch.tensor([b * S + i for b, n in enumerate(lens) for i in range(n)])
    cos, sin = tables(64, 64)
    given = torch.randint(0, 64, (B, S), generator=g)
    for pos in (None, given):
        at = slots.long() if pos is None else given.view(-1)[held]
        dev = pool.cuda()
        _, yq = append_shared_kv(kv.cuda(), dev, ori_block_table=table.cuda(), seqused_kv=used.cuda(), layout_q="BSND",
                                 cu_seqlens_q=torch.tensor([0, 5, 7, 7], dtype=torch.int32).cuda(), q=q.cuda(),
                                 positions=None if pos is None else pos.cuda(), cos=cos.cuda(), sin=sin.cuda())
        flat = dev.view(-1, 1, D).cpu()
        close(flat[rows], definition(kv.view(-1, 1, D)[held], None, cos[at], sin[at], True))
        close(yq.view(-1, H, D)[held.cuda()], definition(q.view(-1, H, D)[held], None, cos[at], sin[at], True))
        rest = torch.ones(len(flat), dtype=torch.bool)
        rest[rows] = False
        assert torch.equal(flat[rest], pool.view(-1, 1, D)[rest])
