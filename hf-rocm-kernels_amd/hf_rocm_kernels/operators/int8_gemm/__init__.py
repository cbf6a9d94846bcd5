from .wrapped import int8_gemm
from .reference import reference_int8_gemm

__all__ = ["int8_gemm", "reference_int8_gemm"]
