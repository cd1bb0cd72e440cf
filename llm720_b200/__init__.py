"""B200-native (sm_100a) PEER forward: a drop-in for the PEER layer of
wrmedford/llm720 backed by hand-written CUDA kernels behind a C ABI, and the
training operators around it."""
from .peer import PEER, PeerOp  # noqa: F401
from .functional import peer_forward, peer_forward_cutlass  # noqa: F401
from .norm import layer_norm  # noqa: F401
from .checkpoint import pack_rows_e4m3, unpack_rows_e4m3  # noqa: F401
from .token_embedding import embedding  # noqa: F401

__all__ = ["PEER", "PeerOp", "peer_forward", "peer_forward_cutlass", "layer_norm", "pack_rows_e4m3", "unpack_rows_e4m3",
           "embedding"]
