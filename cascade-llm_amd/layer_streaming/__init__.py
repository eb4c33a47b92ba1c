"""CPU-resident, HBM-streamed Llama-3.1-8B decode on MI355X (gfx950).

Same public names as the reference package (layer_streaming/__init__.py:
26-45); the device work runs on the hand-written kernels of
libcascade_hip.so (see ``layer_streaming._hip``), which must be built --
nothing here falls back to other device code.
"""

from ._hip import (
    copy_pages,
    gate_up_swiglu_w4,
    linear_w4,
    linear_w4_workspace_bytes,
    paged_append,
    paged_attention_workspace_bytes,
    paged_decode_attention,
    paged_tree_accept,
    paged_tree_attention,
    paged_tree_attention_workspace_bytes,
    sample,
    sample_workspace_bytes,
)
from .graph import DecodeGraph
from .llama31 import (
    LLAMA31_8B_MODEL_ID,
    Llama31Config,
    Llama31DecodeExecutor,
    SimpleKVCache,
)
from .paged import PagedKVCache
from .plan import (
    Granularity,
    HostPlacement,
    ModelPlan,
    TensorSpec,
    TransferUnit,
    VocabPlan,
    build_llama31_8b_plan,
)
from .runtime import DoubleBufferRuntime, ResidentDeviceArena, ResidentTransformerRuntime
from .tree import tree_masks
from .vocab import VocabStreamingRuntime, merge_topk
from .w4 import W4Matrix
from .weight_store import (
    FullPinnedWeightStore,
    PinnedStagingWeightStore,
    WeightStoreMode,
    create_weight_store,
)

__all__ = [
    "DecodeGraph",
    "DoubleBufferRuntime",
    "FullPinnedWeightStore",
    "Granularity",
    "HostPlacement",
    "LLAMA31_8B_MODEL_ID",
    "Llama31Config",
    "Llama31DecodeExecutor",
    "ModelPlan",
    "PagedKVCache",
    "PinnedStagingWeightStore",
    "ResidentDeviceArena",
    "ResidentTransformerRuntime",
    "SimpleKVCache",
    "TensorSpec",
    "TransferUnit",
    "VocabPlan",
    "VocabStreamingRuntime",
    "W4Matrix",
    "WeightStoreMode",
    "build_llama31_8b_plan",
    "copy_pages",
    "create_weight_store",
    "gate_up_swiglu_w4",
    "linear_w4",
    "linear_w4_workspace_bytes",
    "merge_topk",
    "paged_append",
    "paged_attention_workspace_bytes",
    "paged_decode_attention",
    "paged_tree_accept",
    "paged_tree_attention",
    "paged_tree_attention_workspace_bytes",
    "sample",
    "sample_workspace_bytes",
    "tree_masks",
]
