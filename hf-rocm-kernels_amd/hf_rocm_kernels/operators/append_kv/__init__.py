from .wrapped import append_kv
from .reference import reference_append_kv

__all__ = ["append_kv", "reference_append_kv"]
