"""B200-native sparse_attn_sharedkv (DeepSeek-V4 style shared-KV sparse attention).

Drop-in replacements for the reference entry points:

* ``sparse_attn_sharedkv`` (``api.py``) -- the fused forward;
* ``sparse_attn_sharedkv_metadata`` (``metadata.py``) -- the scheduler;

and the backward the reference documents but does not ship
(``sparse_attn_sharedkv_backward``, ``sparse_attn_sharedkv_train``).

What fills their inputs is in ``rope``: head norm with rotation
(``head_norm_rope``) and the append to the paged cache (``append_shared_kv``);
``tree`` has the attention of drafted trees (``tree_attn_sharedkv``).

All run hand-written sm_100a kernels from ``libsas_b200.so`` (C ABI in
``include/sas_b200.h``). ``sharding`` holds the request-parallel and
head-sharded multi-GPU drivers; ``synth`` the seeded input generators.
"""

from .api import sparse_attn_sharedkv  # noqa: F401
from .backward import SparseAttnSharedkv, sparse_attn_sharedkv_backward, sparse_attn_sharedkv_train  # noqa: F401
from .rope import (  # noqa: F401
    HeadNormRope,
    append_shared_kv,
    append_shared_kv_backward,
    head_norm_rope,
    head_norm_rope_backward,
    head_norm_rope_train,
)
from .metadata import SAS_META_SIZE, sparse_attn_sharedkv_metadata  # noqa: F401
from .tree import tree_attn_sharedkv  # noqa: F401
from ._lib import check_device_status, device_status, reset_device_status  # noqa: F401

__all__ = [
    "sparse_attn_sharedkv",
    "sparse_attn_sharedkv_backward",
    "sparse_attn_sharedkv_train",
    "SparseAttnSharedkv",
    "sparse_attn_sharedkv_metadata",
    "head_norm_rope",
    "head_norm_rope_backward",
    "head_norm_rope_train",
    "HeadNormRope",
    "append_shared_kv",
    "append_shared_kv_backward",
    "tree_attn_sharedkv",
    "SAS_META_SIZE",
    "check_device_status",
    "device_status",
    "reset_device_status",
]
