"""Dense attention on MI355X (the dense-others head kind and the dense baseline),
and attention over shared and scored caches."""

from .attention import decode_dense, dense_attention, prefill_dense
from .cached import decode_accumulate, shared_prefix_attention

__all__ = ["dense_attention", "prefill_dense", "decode_dense", "decode_accumulate",
           "shared_prefix_attention"]
