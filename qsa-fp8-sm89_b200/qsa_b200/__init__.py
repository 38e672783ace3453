"""qsa_b200 -- B200-native (sm_100a) sparse paged GQA FP8 decode attention.

A drop-in for the decode-attention path of Ammar-Alnagar/QSA-FP8-SM89: the
same torch-callable contract (``run``, ``launch``, ``qsa_decode``), backed by
hand-written sm_100a CUDA kernels behind a C ABI (``include/qsa_b200.h``,
``libqsa_b200.so``) and a thin ``torch.ops.qsa_b200`` extension over it.

Beside it stands the block-scaled cache, with a scale for each block of tokens
and KV head: ``qsa_qk_rope`` norms and rotates the queries (and keys),
``qsa_block_append`` writes new keys and values, ``qsa_block_decode`` attends.
"""

from ._lib import QsaBuildError, load_clib, load_torch_ops
from .block import block_cache, qsa_block_append, qsa_block_decode, qsa_qk_rope, rope_table
from .ops import launch, qsa_cache_write, qsa_decode, qsa_topk_select, run, slots, token_slots, workspace_bytes

__all__ = [
    "QsaBuildError",
    "block_cache",
    "launch",
    "load_clib",
    "load_torch_ops",
    "qsa_block_append",
    "qsa_block_decode",
    "qsa_cache_write",
    "qsa_qk_rope",
    "qsa_topk_select",
    "qsa_decode",
    "rope_table",
    "run",
    "slots",
    "token_slots",
    "workspace_bytes",
]
