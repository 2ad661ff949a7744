from .agg import PositionAwareAggregator
from .diff_transformer import DiffTransformerBlock, DiffTransformerLayer
from .linear_transformer import LinearTransformerBlock, LinearTransformerLayer
from .model import SasRec, SasRecBody
from .transformer import SasRecTransformerBlock, SasRecTransformerLayer

__all__ = [
    "DiffTransformerBlock",
    "DiffTransformerLayer",
    "LinearTransformerBlock",
    "LinearTransformerLayer",
    "PositionAwareAggregator",
    "SasRec",
    "SasRecBody",
    "SasRecTransformerBlock",
    "SasRecTransformerLayer",
]
