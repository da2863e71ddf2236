"""What fills q and the caches of ``sparse_attn_sharedkv``: head norm, rotation, paged append.

* ``head_norm_rope``: RMS norm of every query (and key) head with the position
  rotation of its last dims in the same pass; ``head_norm_rope_backward`` and
  the autograd form ``head_norm_rope_train``. With ``norm=False,
  inverse=True`` it turns the attention's output back (the caches hold rotated
  rows as K and as V);
* ``append_shared_kv``: the new tokens' shared K=V rows, normed and rotated,
  written into the paged cache at the slots the attention reads them from,
  optionally with their queries in the same launch;
  ``append_shared_kv_backward`` takes the cache's gradient, as
  ``sparse_attn_sharedkv_backward`` returns it, to the raw rows.

The reference has no counterpart: its op takes a rotated ``q`` and filled
caches (``sparse_attn_sharedkv_tilelang/api.py:129-163``). Each call is one
launch on the current stream (a backward with weight gradients two), without
host synchronisation and without a CPU fallback. Results carry no autograd
graph, whatever requires gradients: ``head_norm_rope_train`` and the
``*_backward`` calls are for training. What is written in place counts as an
in-place change. Shapes are ``ValueError``,
modes ``AssertionError``, as in ``sparse_attn_sharedkv``; what only the device
can see (a bad block-table entry, a position outside the tables) goes to the
status word (``check_device_status``).
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

FLAG_NORM, FLAG_INVERSE, FLAG_INTERLEAVED, FLAG_POS64 = 1, 2, 4, 8
LAYOUTS = {"BSND": 0, "TND": 1}
MAX_DIM = 1024


def _dtype_code(t: torch.dtype) -> int:
    if t == torch.bfloat16:
        return 0
    if t == torch.float16:
        return 1
    raise ValueError(f"unsupported torch dtype {t}")


def _i32(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    if t.dtype is torch.int32 and t.device == dev and t.is_contiguous():
        return t
    return t.to(device=dev, dtype=torch.int32).contiguous()


def _f32(t: Optional[torch.Tensor], dev: torch.device) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.device != dev or not t.is_contiguous():
        t = t.to(device=dev, dtype=torch.float32).contiguous()
    return t if t.data_ptr() & 15 == 0 else t.clone()


def _overlap(ts: int, T: int, hs: int, H: int, D: int) -> bool:
    """Whether two of the rows at t * ts + h * hs, D values each, share one."""
    if T == 1 or H == 1:
        return T * H > 1 and (ts if T > 1 else hs) < D
    (a, na), (b, nb) = sorted(((ts, T), (hs, H)))
    if a < D:
        return True
    if b >= a * (na - 1) + D:
        return False
    # rows of the wider stride among those of the other: the two nearest ones
    return any(abs(j * b - i * a) < D for j in range(1, nb) for i in (j * b // a, j * b // a + 1) if i < na)


_NO_ROWS = (0, 0, 0)


def _rows(t: torch.Tensor, name: str, out: bool = False):
    """``t [..., H, D]`` as the kernel takes it, ``(tensor, (pointer, token stride, head stride))``: copied only
    where a stride or an address does not fit."""
    shape = t.shape
    H, D = shape[-2], shape[-1]
    at = t.data_ptr()
    if at & 15 == 0 and t.is_contiguous():
        return t, (at, H * D, D)
    T = shape[:-2].numel()
    if T == 0:
        return t, (at, H * D, D)
    try:
        r = t.view(T, H, D)
    except RuntimeError:
        if out:
            raise ValueError(f"{name}: the token dims must have one stride") from None
        r = t.reshape(T, H, D)
    ts, hs = (r.stride(0) if T > 1 else H * D), (r.stride(1) if H > 1 else D)
    if out and _overlap(ts, T, hs, H, D):
        raise ValueError(f"the rows of {name} overlap")
    if r.stride(2) != 1 or r.data_ptr() & 15 or (ts | hs) & 7:
        if out:
            raise ValueError(f"{name} must have a contiguous last dim and 16-byte aligned rows")
        r = r.clone(memory_format=torch.contiguous_format)
        ts, hs = H * D, D
    return r, (r.data_ptr(), ts, hs)


def _new(like: torch.Tensor) -> torch.Tensor:
    if like.is_contiguous():  # 0.7 us less than with a memory format given
        return torch.empty_like(like)
    return torch.empty_like(like, memory_format=torch.contiguous_format)


def _out_rows(out: Optional[torch.Tensor], like: torch.Tensor, name: str):
    """The output tensor, a new one without ``out``, and its rows as the kernel takes them."""
    if out is None:
        out = _new(like)
        H, D = like.shape[-2:]
        return out, (out.data_ptr(), H * D, D)
    return out, _rows(out, name, out=True)[1]


def _rope_args(D, T, positions, cos, sin, norm, inverse, interleaved, slots=False):
    """(positions, cos, sin, P, R, flags), checked; the tensors are returned to be kept alive."""
    flags = (FLAG_NORM if norm else 0) | (FLAG_INVERSE if inverse else 0) | (FLAG_INTERLEAVED if interleaved else 0)
    if cos is None and sin is None:
        return None, None, None, 0, 0, flags
    shape = None if cos is None else cos.shape
    if shape is None or sin is None or shape != sin.shape or len(shape) != 2:
        raise ValueError("cos and sin must both be [positions, rotated dims / 2]")
    P, R = shape[0], 2 * shape[1]
    step = 8 if interleaved else 16
    if P < 1 or R < 1 or R > D or R % step:
        raise ValueError(f"the rotated dims must be a multiple of {step} and at most D={D} (got {R})")
    if positions is None:
        if not slots:
            raise ValueError("positions is required with cos and sin")
    else:
        if positions.numel() != T:
            raise ValueError(f"positions must have one entry per token (got {positions.numel()} for {T})")
        dtype = positions.dtype
        if dtype is torch.int64:
            flags |= FLAG_POS64
        elif dtype is not torch.int32:
            raise ValueError(f"positions must be int32 or int64 (got {positions.dtype})")
    return positions, cos, sin, P, R, flags


def _to_dev(dev, positions, cos, sin):
    if positions is not None and (positions.device != dev or not positions.is_contiguous()):
        positions = positions.to(dev).contiguous()
    return positions, _f32(cos, dev), _f32(sin, dev)


def _check_dim(D: int, *weights) -> None:
    if D % 8 or not 0 < D <= MAX_DIM:
        raise ValueError(f"the head dim must be a multiple of 8 and at most {MAX_DIM} (got {D})")
    for w in weights:
        if w is not None and w.shape != (D,):
            raise ValueError(f"a weight must be [{D}] (got {tuple(w.shape)})")


def _check_pair(q, k):
    """(tokens, head dim) of q and k, checked. Shapes are read once: every read of
    a tensor's property costs 0.2-0.3 us, and the smallest calls take longer on the host
    than on the GPU."""
    qs = q.shape
    if len(qs) < 2 or qs[-2] < 1:
        raise ValueError(f"q must be [..., heads, D] (got {tuple(qs)})")
    if k is not None:
        ks = k.shape
        if len(ks) != len(qs) or ks[:-2] != qs[:-2] or ks[-1] != qs[-1] or ks[-2] < 1 or k.dtype != q.dtype \
                or k.device != q.device:
            raise ValueError("k must have q's token dims, head dim, dtype and device")
    return math.prod(qs[:-2]), qs[-1]


def _check_out(out, like, name):
    if out is not None and (out.shape != like.shape or out.dtype != like.dtype or out.device != like.device):
        raise ValueError(f"{name} must have the shape, dtype and device of its input")


def _raise(rc: int, what: str, entry: str) -> None:
    if rc in (1, 2):
        raise ValueError(f"{what}: {_lib.ERRORS[rc]}")
    _lib.check(rc, entry)


def head_norm_rope(
    q: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    *,
    positions: Optional[torch.Tensor] = None,
    cos: Optional[torch.Tensor] = None,
    sin: Optional[torch.Tensor] = None,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    norm: bool = True,
    inverse: bool = False,
    interleaved: bool = True,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
):
    """``Rot(positions) (x * weight / sqrt(mean(x^2) + eps))`` for every head of
    ``q [..., H, D]`` and ``k [..., Hk, D]`` (bf16 or fp16, any token and head
    strides); returns ``q_out``, or ``(q_out, k_out)`` with ``k``.

    The last ``2 * cos.shape[1]`` dims are turned by row ``positions[t]`` of
    ``cos`` / ``sin`` (fp32): neighbouring dims as pairs, or with
    ``interleaved=False`` dim i with dim i + half. Without ``cos`` and ``sin``
    there is no rotation; ``norm=False`` leaves out the norm; ``inverse`` turns
    by the negative angle. ``q_out`` / ``k_out`` may be the inputs themselves.
    """
    T, D = _check_pair(q, k)
    _check_dim(D, q_weight, k_weight)
    code = _dtype_code(q.dtype)
    assert norm or (q_weight is None and k_weight is None), "weights need norm=True"
    positions, cos, sin, P, R, flags = _rope_args(D, T, positions, cos, sin, norm, inverse, interleaved)
    _check_out(q_out, q, "q_out")
    _check_out(k_out, k, "k_out")
    dev = q.device
    if dev.type != "cuda":
        raise RuntimeError("head_norm_rope needs CUDA tensors (no CPU path)")
    given = [t for t in (q_out, k_out) if t is not None]
    q_out, qo = _out_rows(q_out, q, "q_out")
    ka = ko = _NO_ROWS
    Hk = 0
    if k is not None:
        k_out, ko = _out_rows(k_out, k, "k_out")
    if T:
        positions, cos, sin = _to_dev(dev, positions, cos, sin)
        qw, kw = _f32(q_weight, dev), _f32(k_weight if k is not None else None, dev)
        q, qa = _rows(q, "q")
        if k is not None:
            Hk = k.shape[-2]
            k, ka = _rows(k, "k")
        rc = _lib.lib().sas_head_norm_rope_fwd(
            *qa, *qo, q.shape[-2], *ka, *ko, Hk, T, D, code, _lib.ptr(positions), _lib.ptr(cos), _lib.ptr(sin), P, R,
            _lib.ptr(qw), _lib.ptr(kw), float(eps), flags, _lib.state(dev).status.data_ptr(), _lib.raw_stream(dev))
        _raise(rc, "head_norm_rope", "sas_head_norm_rope_fwd")
        _lib.written(given)
    return q_out if k is None else (q_out, k_out)


def head_norm_rope_backward(
    dq_out: torch.Tensor,
    q: torch.Tensor,
    dk_out: Optional[torch.Tensor] = None,
    k: Optional[torch.Tensor] = None,
    *,
    positions: Optional[torch.Tensor] = None,
    cos: Optional[torch.Tensor] = None,
    sin: Optional[torch.Tensor] = None,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    norm: bool = True,
    inverse: bool = False,
    interleaved: bool = True,
):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of ``head_norm_rope`` from
    those of its results and its inputs; ``dk`` is None without ``k`` and a
    weight's gradient (fp32, summed in a fixed order) without that weight."""
    T, D = _check_pair(q, k)
    _check_dim(D, q_weight, k_weight)
    code = _dtype_code(q.dtype)
    assert norm or (q_weight is None and k_weight is None), "weights need norm=True"
    positions, cos, sin, P, R, flags = _rope_args(D, T, positions, cos, sin, norm, inverse, interleaved)
    dev = q.device
    for x, dx in ((q, dq_out), (k, dk_out)):
        if x is not None and (dx is None or dx.shape != x.shape):
            raise ValueError("dq_out and dk_out must have the shapes of q and k")
        if x is not None and dx.device != dev:
            raise ValueError("dq_out and dk_out must be on the device of q and k")
    if dev.type != "cuda":
        raise RuntimeError("head_norm_rope_backward needs CUDA tensors (no CPU path)")
    dq = _new(q)
    dk = _new(k) if k is not None else None
    qw = _f32(q_weight, dev)
    kw = _f32(k_weight, dev) if k is not None else None
    dqw = torch.empty(D, dtype=torch.float32, device=dev) if qw is not None else None
    dkw = torch.empty(D, dtype=torch.float32, device=dev) if kw is not None else None
    lib = _lib.lib()
    st = _lib.state(dev)
    positions, cos, sin = _to_dev(dev, positions, cos, sin)
    q, qa = _rows(q, "q")
    dq_out, da = _rows(dq_out.to(q.dtype), "dq_out")
    ka = db = _NO_ROWS
    Hk = 0
    if k is not None:
        Hk = k.shape[-2]
        k, ka = _rows(k, "k")
        dk_out, db = _rows(dk_out.to(q.dtype), "dk_out")
    ws = torch.empty(lib.sas_head_norm_rope_bwd_workspace_bytes(D), dtype=torch.uint8, device=dev) \
        if qw is not None or kw is not None else None
    rc = lib.sas_head_norm_rope_bwd(
        *da, *qa, dq.data_ptr(), q.shape[-2], *db, *ka, _lib.ptr(dk), Hk, T, D, code, _lib.ptr(positions), _lib.ptr(cos),
        _lib.ptr(sin), P, R, _lib.ptr(qw), _lib.ptr(kw), _lib.ptr(dqw), _lib.ptr(dkw), float(eps), flags, st.status.data_ptr(),
        _lib.ptr(ws), ws.numel() if ws is not None else 0, _lib.raw_stream(dev)) if T else 0
    _raise(rc, "head_norm_rope_backward", "sas_head_norm_rope_bwd")
    if not T:
        dqw, dkw = (None if w is None else w.zero_() for w in (dqw, dkw))
    return dq, dk, dqw, dkw


class HeadNormRope(torch.autograd.Function):
    """``head_norm_rope`` as an autograd function of (q, k, q_weight, k_weight), differentiable once."""

    TABLES = ("positions", "cos", "sin")

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, kwargs):
        # positions, cos and sin are saved too, so that one changed before the backward is an error
        held = [kwargs.get(name) for name in HeadNormRope.TABLES]
        ctx.kwargs = {name: x for name, x in kwargs.items() if name not in HeadNormRope.TABLES}
        ctx.save_for_backward(q, k, q_weight, k_weight, *held)
        return head_norm_rope(q, k, q_weight=q_weight, k_weight=k_weight, **kwargs)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out=None):
        q, k, qw, kw, *held = ctx.saved_tensors
        dq, dk, dqw, dkw = head_norm_rope_backward(dq_out, q, dk_out, k, q_weight=qw, k_weight=kw,
                                                   **dict(zip(HeadNormRope.TABLES, held)), **ctx.kwargs)
        return dq, dk, None if dqw is None else dqw.to(qw.dtype), None if dkw is None else dkw.to(kw.dtype), None


def head_norm_rope_train(q, k=None, *, q_weight=None, k_weight=None, **kwargs):
    """``head_norm_rope`` with autograd: gradients flow to ``q``, ``k`` and the weights."""
    for name in ("q_out", "k_out"):
        given = kwargs.pop(name, None)
        assert given is None, f"{name} cannot be given with autograd"
    return HeadNormRope.apply(q, k, q_weight, k_weight, kwargs)


class _Paged:
    """The checked cache arguments of an append: token rows, block table, lengths."""

    def __init__(self, kv, pool, table, seqused, cu, layout):
        assert layout in LAYOUTS, f"unsupported layout_q={layout!r}"
        ps, ks, ts = pool.shape, kv.shape, table.shape
        if len(ps) != 4 or ps[2] != 1:
            raise ValueError(f"the cache must be [blocks, block size, 1, D] (got {tuple(ps)})")
        if pool.dtype != kv.dtype:
            raise ValueError("the cache must have the dtype of kv")
        D = ps[3]
        if not pool.is_contiguous() or pool.data_ptr() % 16:
            raise ValueError("the cache must be contiguous and 16-byte aligned")
        want = 3 if layout == "TND" else 4  # [T, 1, D] or [B, S, 1, D]; the head dim may be left out
        if len(ks) == want - 1:
            kv = kv.unsqueeze(-2)
            ks = kv.shape
        if len(ks) != want or ks[-2] != 1 or ks[-1] != D:
            raise ValueError(f"kv must be [tokens, 1, {D}] in the layout {layout} (got {tuple(ks)})")
        if len(ts) != 2:
            raise ValueError("ori_block_table must be [requests, blocks]")
        if layout == "TND":
            assert cu is not None, "cu_seqlens_q is required for TND"
            self.B, self.S, self.T = cu.numel() - 1, 0, ks[0]
        else:
            self.B, self.S = ks[:2]
            self.T = self.B * self.S
            if cu is not None and cu.numel() != self.B + 1:
                raise ValueError(f"cu_seqlens_q must have {self.B + 1} entries (got {cu.numel()})")
        if self.B < 0 or ts[0] != self.B or seqused.numel() != self.B:
            raise ValueError(f"ori_block_table and seqused_kv must have one entry per request ({self.B})")
        self.kv, self.D, self.layout = kv, D, LAYOUTS[layout]
        self.blocks, self.block_size, self.entries = ps[0], ps[1], ts[1]
        self.table, self.cu, self.seqused = table, cu, seqused

    def put(self, dev):
        self.table, self.seqused = _i32(self.table, dev), _i32(self.seqused, dev)
        self.cu = _i32(self.cu, dev) if self.cu is not None else None

    def args(self):
        return (self.blocks, self.block_size, self.table.data_ptr(), self.entries, _lib.ptr(self.cu),
                self.seqused.data_ptr(), self.B, self.S, self.layout)


def append_shared_kv(
    kv: torch.Tensor,
    ori_kv: torch.Tensor,
    *,
    ori_block_table: torch.Tensor,
    seqused_kv: torch.Tensor,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    layout_q: str = "TND",
    positions: Optional[torch.Tensor] = None,
    cos: Optional[torch.Tensor] = None,
    sin: Optional[torch.Tensor] = None,
    weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    norm: bool = True,
    interleaved: bool = True,
    q: Optional[torch.Tensor] = None,
    q_weight: Optional[torch.Tensor] = None,
    q_out: Optional[torch.Tensor] = None,
):
    """Norms and rotates the new tokens' shared K=V rows ``kv`` (``[T, 1, D]``
    for TND, ``[B, S, 1, D]`` for BSND, any token stride) and writes them into
    the paged cache ``ori_kv [blocks, block size, 1, D]`` in place; returns
    ``ori_kv``, or ``(ori_kv, q_out)`` with ``q``.

    ``seqused_kv`` counts the new tokens, as the attention that follows takes
    it: token i of a request's n goes to slot ``seqused_kv - n + i``, which is
    its position too unless ``positions`` gives one per token (drafted tokens
    are rotated by their depth in the tree). With ``q`` (``[T, H, D]`` or
    ``[B, S, H, D]``) the same launch does ``head_norm_rope`` of the tokens'
    queries. A token whose block-table entry is negative is not written; an
    entry outside the table or the pool is not written and recorded in the
    status word. What padding (slots of BSND past ``cu_seqlens_q``'s count,
    tokens after the last request) holds in ``kv`` and ``positions`` does not
    matter.
    """
    p = _Paged(kv, ori_kv, ori_block_table, seqused_kv, cu_seqlens_q, layout_q)
    D, T = p.D, p.T
    _check_dim(D, weight, q_weight)
    code = _dtype_code(kv.dtype)
    assert norm or (weight is None and q_weight is None), "weights need norm=True"
    positions, cos, sin, P, R, flags = _rope_args(D, T, positions, cos, sin, norm, False, interleaved, slots=True)
    if q is not None:
        _check_pair(q, p.kv)
        _check_out(q_out, q, "q_out")
    dev = kv.device
    if dev.type != "cuda":
        raise RuntimeError("append_shared_kv needs CUDA tensors (no CPU path)")
    if ori_kv.device != dev or (q is not None and q.device != dev):
        raise ValueError("kv, ori_kv and q must be on one device")
    given = [ori_kv] if q is None or q_out is None else [ori_kv, q_out]
    qa = qo = _NO_ROWS
    H = 0
    if q is not None:
        q_out, qo = _out_rows(q_out, q, "q_out")
    if T:
        p.put(dev)
        positions, cos, sin = _to_dev(dev, positions, cos, sin)
        w, qw = _f32(weight, dev), _f32(q_weight if q is not None else None, dev)
        r, ra = _rows(p.kv, "kv")
        if q is not None:
            H = q.shape[-2]
            q, qa = _rows(q, "q")
        rc = _lib.lib().sas_append_sharedkv(
            *ra[:2], ori_kv.data_ptr(), *p.args(), *qa, *qo, H, T, D, code, _lib.ptr(positions), _lib.ptr(cos),
            _lib.ptr(sin), P, R, _lib.ptr(w), _lib.ptr(qw), float(eps), flags, _lib.state(dev).status.data_ptr(),
            _lib.raw_stream(dev))
        _raise(rc, "append_shared_kv", "sas_append_sharedkv")
        _lib.written(given)
    return ori_kv if q is None else (ori_kv, q_out)


def append_shared_kv_backward(
    d_ori_kv: torch.Tensor,
    kv: torch.Tensor,
    *,
    ori_block_table: torch.Tensor,
    seqused_kv: torch.Tensor,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    layout_q: str = "TND",
    positions: Optional[torch.Tensor] = None,
    cos: Optional[torch.Tensor] = None,
    sin: Optional[torch.Tensor] = None,
    weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    norm: bool = True,
    interleaved: bool = True,
):
    """Gradients ``(dkv, dweight)`` of the raw rows and the norm's weight from
    the cache's gradient (shape and dtype of the cache); ``dweight`` is fp32,
    None without ``weight``. Tokens that were not written get zero. The
    queries' part of a fused append is ``head_norm_rope_backward``'s."""
    p = _Paged(kv, d_ori_kv, ori_block_table, seqused_kv, cu_seqlens_q, layout_q)
    D, T = p.D, p.T
    _check_dim(D, weight)
    code = _dtype_code(kv.dtype)
    assert norm or weight is None, "weights need norm=True"
    positions, cos, sin, P, R, flags = _rope_args(D, T, positions, cos, sin, norm, False, interleaved, slots=True)
    dev = kv.device
    if dev.type != "cuda":
        raise RuntimeError("append_shared_kv_backward needs CUDA tensors (no CPU path)")
    if d_ori_kv.device != dev:
        raise ValueError("kv and d_ori_kv must be on one device")
    dkv = _new(kv)
    w = _f32(weight, dev)
    dw = torch.zeros(D, dtype=torch.float32, device=dev) if w is not None and not T else \
        torch.empty(D, dtype=torch.float32, device=dev) if w is not None else None
    if T:
        lib = _lib.lib()
        p.put(dev)
        positions, cos, sin = _to_dev(dev, positions, cos, sin)
        r, ra = _rows(p.kv, "kv")
        ws = torch.empty(lib.sas_head_norm_rope_bwd_workspace_bytes(D), dtype=torch.uint8, device=dev) \
            if w is not None else None
        rc = lib.sas_append_sharedkv_bwd(
            d_ori_kv.data_ptr(), *p.args(), *ra[:2], dkv.data_ptr(), T, D, code, _lib.ptr(positions), _lib.ptr(cos),
            _lib.ptr(sin), P, R, _lib.ptr(w), _lib.ptr(dw), float(eps), flags, _lib.state(dev).status.data_ptr(),
            _lib.ptr(ws), ws.numel() if ws is not None else 0, _lib.raw_stream(dev))
        _raise(rc, "append_shared_kv_backward", "sas_append_sharedkv_bwd")
    return dkv, dw
