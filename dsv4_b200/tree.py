"""Attention of drafted tokens that form a tree over the paged shared-KV caches.

``tree_attn_sharedkv`` is to a drafted tree what ``sparse_attn_sharedkv`` is to
a chain of new tokens: the same caches, tables, lengths, sinks and scenarios
(window only, the whole compressed cache, top-k lists), with each token seeing
its ancestors instead of everything before it. The reference decodes chains
only (``sparse_attn_sharedkv_tilelang/api.py:129-397``). No schedule is needed:
the kernel cuts the work itself. The current stream, no host synchronisation,
no CPU fallback, no autograd graph; errors as in ``sparse_attn_sharedkv``.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from .rope import LAYOUTS, _dtype_code, _f32, _i32

HEAD_DIM = 512
MAX_TREE = 1024


def tree_attn_sharedkv(
    q: torch.Tensor,
    *,
    ori_kv: torch.Tensor,
    ori_block_table: torch.Tensor,
    tree_parents: torch.Tensor,
    seqused_kv: torch.Tensor,
    sinks: torch.Tensor,
    softmax_scale: float,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    cmp_kv: Optional[torch.Tensor] = None,
    cmp_sparse_indices: Optional[torch.Tensor] = None,
    cmp_block_table: Optional[torch.Tensor] = None,
    cmp_ratio: Optional[int] = None,
    ori_win_left: int = 127,
    layout_q: str = "TND",
    layout_kv: str = "PA_ND",
    return_softmax_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    lse_out: Optional[torch.Tensor] = None,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Returns the output in the layout of ``q`` (``[T, H, 512]`` or ``[B, S, H,
    512]``), with ``return_softmax_lse`` also the fp32 log-sum-exp, sinks
    included.

    A request's n drafted tokens are in the window cache at the slots before
    ``seqused_kv`` (``append_shared_kv`` puts them there). ``tree_parents``
    (``[T]`` or ``[B, S]``) names for each the token that it follows, by its
    index among its request's tokens and below its own; -1 follows the cached
    context, anything less marks an unused slot (zero output and LSE). A token
    at depth d has position ``ctx + d``, ``ctx = seqused_kv - n``, and attends
    to its window of ``ori_win_left`` rows before that position (cached rows
    and ancestors), to itself, and to compressed rows below ``ctx //
    cmp_ratio``: with ``cmp_kv`` to all of them, with ``cmp_sparse_indices``
    (``[T, 1, K]`` or ``[B, S, 1, K]``) to its list, where ids outside that
    range are skipped. (A token of ``sparse_attn_sharedkv`` sees those below
    ``(position + 1) // cmp_ratio``: rows that end among the new tokens too, which
    a tree's branches would each have their own of. The two are equal for lists of
    cached rows that end in -1 if they are short, and for tokens with ``(position + 1) // cmp_ratio`` still at
    ``ctx // cmp_ratio``.) A KV row with infinities or NaN makes the output of the
    tokens that see it NaN, at least in the columns where the row is not
    finite; it reaches no other token. A request of over 1024 tokens,
    with more tokens than ``seqused_kv``, or a token whose parent does not
    precede it gives zeros and is recorded in the status word.
    """
    assert layout_kv == "PA_ND", "only layout_kv=PA_ND supported"
    assert layout_q in LAYOUTS, f"unsupported layout_q={layout_q!r}"
    # shapes are read once each: every read of a tensor's property costs 0.2-0.3 us,
    # and the smallest calls take as long on the host as on the GPU
    dtype, shape = q.dtype, q.shape
    code = _dtype_code(dtype)
    if layout_q == "TND":
        assert cu_seqlens_q is not None, "cu_seqlens_q is required for TND"
        if len(shape) != 3:
            raise ValueError(f"q must be [T, heads, {HEAD_DIM}] (got {tuple(shape)})")
        T, H, D = shape
        B, S = cu_seqlens_q.numel() - 1, 0
    else:
        if len(shape) != 4:
            raise ValueError(f"q must be [B, S, heads, {HEAD_DIM}] (got {tuple(shape)})")
        B, S, H, D = shape
        T = B * S
        if cu_seqlens_q is not None and cu_seqlens_q.numel() != B + 1:
            raise ValueError(f"cu_seqlens_q must have {B + 1} entries (got {cu_seqlens_q.numel()})")
    if D != HEAD_DIM or H <= 0 or H % 8:
        raise ValueError(f"only D={HEAD_DIM} and heads a multiple of 8 supported (got {H} heads, D={D})")
    if ori_win_left < 0:
        raise ValueError("ori_win_left must not be negative")
    if tree_parents.numel() != T:
        raise ValueError(f"tree_parents must have one entry per token (got {tree_parents.numel()} for {T})")
    if sinks.numel() != H:
        raise ValueError(f"sinks must have one entry per head (got {sinks.numel()} for {H})")
    scenario, K, ratio = 1, 0, 1
    if cmp_kv is not None:
        scenario, ratio = 2, 4 if cmp_ratio is None else cmp_ratio
        assert cmp_block_table is not None, "cmp_kv needs cmp_block_table"
        if ratio < 1:
            raise ValueError(f"cmp_ratio must be positive (got {ratio})")
    if cmp_sparse_indices is not None:
        assert cmp_kv is not None, "cmp_sparse_indices needs cmp_kv"
        scenario, K = 3, cmp_sparse_indices.shape[-1]
        if K < 1 or cmp_sparse_indices.numel() != T * K:
            raise ValueError(f"cmp_sparse_indices must be [tokens, 1, K] (got {tuple(cmp_sparse_indices.shape)})")
    ori_dims = _check_pool("ori", ori_kv, ori_block_table, B, dtype)
    cmp_dims = (0, 0, 0) if cmp_kv is None else _check_pool("cmp", cmp_kv, cmp_block_table, B, dtype)
    if B < 0 or seqused_kv.numel() != B:
        raise ValueError(f"seqused_kv must have one entry per request (got {seqused_kv.numel()} for {B})")
    dev = q.device
    if out is not None:
        _check_out("out", out, shape, dtype, dev)
    if lse_out is not None:
        _check_out("lse_out", lse_out, shape[:-1], torch.float32, dev)
    if dev.type != "cuda":
        raise RuntimeError("tree_attn_sharedkv needs q on a CUDA device (no CPU path)")
    given = [t for t in (out, lse_out) if t is not None]
    q = _aligned(q, dev)
    if out is None:
        out = torch.empty_like(q)
    if lse_out is None and return_softmax_lse:
        lse_out = torch.empty(shape[:-1], dtype=torch.float32, device=dev)
    if T:
        lib = _lib.lib()
        st = _lib.state(dev)
        cu = _i32(cu_seqlens_q, dev) if cu_seqlens_q is not None else None
        skv, par = _i32(seqused_kv, dev), _i32(tree_parents, dev)
        snk = _f32(sinks, dev)
        ori, obt = _aligned(ori_kv, dev), _i32(ori_block_table, dev)
        cmp = cbt = idx = None
        if scenario >= 2:
            cmp, cbt = _aligned(cmp_kv, dev), _i32(cmp_block_table, dev)
        if scenario == 3:
            idx = _i32(cmp_sparse_indices, dev)
        # from the allocator, so that calls on several streams do not share it
        nws = lib.sas_tree_attn_workspace_bytes(st.num_sms)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        rc = lib.sas_tree_attn_sharedkv(
            q.data_ptr(), T, H, D, code, LAYOUTS[layout_q], B, S, _lib.ptr(cu), skv.data_ptr(), par.data_ptr(),
            ori.data_ptr(), ori_dims[0], ori_dims[1], obt.data_ptr(), ori_dims[2], _lib.ptr(cmp), cmp_dims[0],
            cmp_dims[1], _lib.ptr(cbt), cmp_dims[2], _lib.ptr(idx), K, snk.data_ptr(), float(softmax_scale), int(ratio),
            min(int(ori_win_left), 1 << 30), scenario, out.data_ptr(), _lib.ptr(lse_out), st.num_sms,
            st.status.data_ptr(), ws.data_ptr(), nws, _lib.raw_stream(dev))
        if rc in (1, 2):
            raise ValueError(f"tree_attn_sharedkv: {_lib.ERRORS[rc]}")
        _lib.check(rc, "sas_tree_attn_sharedkv")
        _lib.written(given)
    return (out, lse_out) if return_softmax_lse else out


def _check_pool(name, kv, table, B, dtype) -> Tuple[int, int, int]:
    """Blocks, rows of a block, and entries of a request in the block table."""
    ks, ts = kv.shape, table.shape
    if len(ks) != 4 or ks[2] != 1 or ks[3] != HEAD_DIM or kv.dtype != dtype or ks[1] < 1:
        raise ValueError(f"{name}_kv must be [blocks, block size, 1, {HEAD_DIM}] of q's dtype")
    if len(ts) != 2 or ts[0] != B or ts[1] < 1:
        raise ValueError(f"{name}_block_table must be [{B}, blocks] (got {tuple(ts)})")
    return ks[0], ks[1], ts[1]


def _check_out(name, t, shape, dtype, dev) -> None:
    if t.shape != shape or t.dtype != dtype or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(shape)} tensor of {dtype} beside q")


def _aligned(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    if t.device != dev or not t.is_contiguous():
        t = t.to(dev).contiguous()
    return t if t.data_ptr() & 15 == 0 else t.clone()
