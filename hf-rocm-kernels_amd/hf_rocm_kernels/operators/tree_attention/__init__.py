from .wrapped import tree_attention
from .reference import reference_tree_attention

__all__ = ["tree_attention", "reference_tree_attention"]
