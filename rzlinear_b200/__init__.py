"""rzlinear_b200: the RzLinear (ROBE-Z compressed linear layer) hot path on NVIDIA B200.

Same public names as the reference's `rz_linear` package:
    from rzlinear_b200 import RzLinear, RzLinearFunction, controls
and, beside them, layers over the same hashed array for rows picked by an index:
    RzEmbedding (token table), sort_rows (rows by expert)
"""
from .RzLinearFunction import RzLinearFunction, RzConfig, controls  # noqa: F401
from .RzLinear import RzLinear  # noqa: F401
from .RzEmbeddingFunction import RzEmbeddingFunction  # noqa: F401
from .RzEmbedding import RzEmbedding  # noqa: F401
from .rows import sort_rows  # noqa: F401

__all__ = ["RzLinear", "RzLinearFunction", "RzConfig", "controls", "RzEmbedding", "RzEmbeddingFunction", "sort_rows"]
