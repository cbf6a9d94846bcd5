from .fp8_linear import Fp8Linear, apply_fp8_linear, convert_linear_layers
from .int8_linear import Int8Linear, apply_int8_linear

__all__ = ["Fp8Linear", "apply_fp8_linear", "convert_linear_layers", "Int8Linear", "apply_int8_linear"]
