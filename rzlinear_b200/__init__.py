"""rzlinear_b200: the RzLinear (ROBE-Z compressed linear layer) hot path on NVIDIA B200.

Same public names as the reference's `rz_linear` package:
    from rzlinear_b200 import RzLinear, RzLinearFunction, controls
and, beside them, layers over the same hashed array for rows picked by an index:
    RzEmbedding (token table), RzGroupedLinear (products grouped by expert), sort_rows (rows by expert)
"""
from .RzLinearFunction import RzLinearFunction, RzConfig, controls  # noqa: F401
from .RzLinear import RzLinear  # noqa: F401
from .RzEmbeddingFunction import RzEmbeddingFunction  # noqa: F401
from .RzEmbedding import RzEmbedding  # noqa: F401
from .RzGroupedLinearFunction import RzGroupedLinearFunction  # noqa: F401
from .RzGroupedLinear import RzGroupedLinear  # noqa: F401
from .rows import sort_rows  # noqa: F401

__all__ = ["RzLinear", "RzLinearFunction", "RzConfig", "controls", "RzEmbedding", "RzEmbeddingFunction",
           "RzGroupedLinear", "RzGroupedLinearFunction", "sort_rows"]
