from .wrapped import grouped_gemm
from .reference import reference_grouped_gemm

__all__ = ["grouped_gemm", "reference_grouped_gemm"]
