"""B200-native Converse2D / Converse block (drop-in for Yiozolm/ConverseNet's hot path)."""
from .util_converse import (Converse2D, ConverseBlock, ConverseBlockAlphaVariant, Int8Pointwise, LayerNorm,  # noqa: F401
                            ResidualNorm, sequential)
from . import _cabi  # noqa: F401

__all__ = ["Converse2D", "ConverseBlock", "ConverseBlockAlphaVariant", "Int8Pointwise", "LayerNorm",
           "ResidualNorm", "sequential"]
