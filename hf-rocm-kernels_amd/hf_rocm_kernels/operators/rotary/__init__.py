from .wrapped import rotary
from .frequencies import rotary_frequencies
from .reference import reference_rotary

__all__ = ["rotary", "rotary_frequencies", "reference_rotary"]
