"""The example's serving and training steps against float64 definitions.

Serving bound: each output is p @ v with one rounding of the result (u |o|) and
of every p (u p), and scores off by at most e = 512 * 2^-24 * scale *
sum_d |q_d k_d|, as fp32 sums are; turning it back mixes two columns, whose
bounds add, and rounds once more. Training bound: six tensors on a gradient's
way are rounded to the I/O type (turned q and rows, output, turned output
gradient, the attention's gradients, the result), each by at most u relative to
its norm; a factor of 2 is left for their way through the softmax.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


@pytest.fixture
def example(sas_lib):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from dsv4_b200 import check_device_status, reset_device_status
    from examples import draft_tree

    reset_device_status()
    yield draft_tree
    check_device_status()


def _turn(x, cos, sin, inverse=False):
    """Interleaved rotation of the last 2 * cos.shape[-1] columns."""
    R = 2 * cos.shape[-1]
    a, b = x[..., -R::2], x[..., 1 - R::2]
    s = -sin if inverse else sin
    y = torch.stack([a * cos - b * s, b * cos + a * s], -1).flatten(-2)
    return torch.cat([x[..., :-R], y], -1)


def _token_rows(layer, b, s, ids, win):
    """Positions in the window pool and rows of the compressed pool that a chain's token at position s sees."""
    page = layer.ori.shape[1]
    at = torch.arange(max(0, s - win), s + 1, device=layer.dev)
    ori = layer.obt[b, at // page].long() * page + at % page
    ids = ids[ids >= 0].long()
    return at, ori, layer.cbt[b, ids // page].long() * page + ids % page


def test_tree_step_gives_the_accepted_chain(example):
    ex = example
    layer = ex.Layer([600, 127, 3], heads=16, page=16, topk=48)
    tree, chain, idx, (q, _, _, positions, _) = ex.decode(layer)
    n, scale = len(ex.PATH), ex.D ** -0.5
    flat, cflat = layer.ori.view(-1, ex.D).double(), layer.cmp.view(-1, ex.D).double()
    for t in range(len(positions)):
        s = int(positions[t])
        _, ori, cmp = _token_rows(layer, t // n, s, idx[t, 0], ex.WIN)
        kv, x = torch.cat([flat[ori], cflat[cmp]]), q[t].double()
        p = torch.softmax(torch.cat([x @ kv.T * scale, layer.sinks.double()[:, None]], 1), 1)[:, :-1]
        e = (512 * 2.0 ** -24 * scale * (x.abs() @ kv.abs().T)).amax(-1, keepdim=True)
        o, mag = p @ kv, p @ kv.abs()
        lim = U * o.abs() + (U * 1.01 + 2 * e + 1e-5) * mag
        c, r = layer.rope["cos"][s].double(), layer.rope["sin"][s].double()
        ref = _turn(o, c, r, inverse=True)
        R = 2 * len(c)
        lim[:, -R:] = (lim[:, -R::2] + lim[:, 1 - R::2]).repeat_interleave(2, -1)
        lim = lim * (1 + U) + U * ref.abs() + 1e-6
        for name, got in (("tree", tree), ("chain", chain)):
            over = (got[t].double() - ref).abs() - lim
            assert over.max() <= 0, f"{name}, token {t}: {over.max():.3e} over the bound"


def test_training_step(example):
    ex = example
    layer = ex.Layer([70, 33], heads=8, page=16, topk=16, seed=3)
    cached = layer.cached.tolist()
    n = 6
    (q, kv, idx, dout), out, grads = ex.train(layer, n=n)
    leaves = [x.double().requires_grad_() for x in (q, kv, layer.q_weight, layer.kv_weight, layer.sinks)]
    xq, xkv, wq, wkv, sinks = leaves
    cos, sin = layer.rope["cos"].double(), layer.rope["sin"].double()
    pos = torch.tensor([c + i for c in cached for i in range(n)], device=layer.dev)

    def norm_turn(x, w):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        return _turn(x, cos[pos][:, None], sin[pos][:, None])

    yq, ykv = norm_turn(xq, wq), norm_turn(xkv, wkv)[:, 0]
    pool = layer.ori.view(-1, ex.D).double()
    cmp = layer.cmp.view(-1, ex.D).double()
    outs = []
    for t in range(len(pos)):
        b, s = t // n, int(pos[t])
        at, ori, crow = _token_rows(layer, b, s, idx[t, 0], ex.WIN)
        new = at >= cached[b]
        rows = torch.cat([pool[ori[~new]], ykv[b * n + at[new] - cached[b]], cmp[crow]])
        p = torch.softmax(torch.cat([yq[t] @ rows.T * ex.D ** -0.5, sinks[:, None]], 1), 1)[:, :-1]
        outs.append(p @ rows)
    ref = _turn(torch.stack(outs), cos[pos][:, None], sin[pos][:, None], inverse=True)
    ref.backward(dout.double())
    for name, got, want in zip(("out", "q", "kv", "q weight", "kv weight", "sinks"), (out, *grads), (ref, *(x.grad for x in leaves))):
        off = (got.double().reshape(want.shape) - want).norm() / want.norm()
        assert off <= 12 * U, f"{name}: {off:.3e}"


def test_main(example, capsys):
    example.main()
    assert "accepted path" in capsys.readouterr().out


def test_training_gradients_have_no_part_along_their_rows(example):
    """A norm takes the part along the row out of its gradient, some 1 / sqrt(512) of it, which the bound on the whole
    gradient lets pass: sum(dx x) is zero but for the rounding of dx."""
    (q, kv, _, _), _, (dq, dkv, *_) = example.train(example.Layer([70, 33], heads=8, page=16, topk=16, seed=3), n=6)
    for x, dx in ((q, dq), (kv, dkv)):
        part = dx.double() * x.double()
        assert dx.any() and (part.sum(-1).abs() <= U * part.abs().sum(-1)).all()
