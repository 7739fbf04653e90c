"""glmx: B200-native routed-expert MoE layer over EXL3 trellis-coded experts (drop-in for glm-flash-lite's expert
tier), with the dense operators beside it: the gated feed-forward block, 8-bit linears and sampling. The compute lives in
libglmx.so (include/glmx.h); this package is the PyTorch-side host."""
from ._lib import GlmxError, load  # noqa: F401
from .ffn import GatedFFN, dense_check, gated_ffn  # noqa: F401
from .int8 import Int8Linear, quantize_rows  # noqa: F401
from .layer import MoELayer, decode_tiles  # noqa: F401
from .router import Router  # noqa: F401
from .sampling import sample  # noqa: F401

__all__ = ["MoELayer", "Router", "GatedFFN", "gated_ffn", "Int8Linear", "quantize_rows", "sample", "dense_check", "decode_tiles", "GlmxError",
           "load"]
