import math
from typing import Optional, Tuple

import torch
from torch import Tensor


def rotary_frequencies(
    rotated: int, base: float = 10000.0, scaling: Optional[dict] = None, device: str = "cuda",
) -> Tuple[Tensor, float]:
    """The frequencies that `rotary` and `append_kv` take, and the magnitude: (float64 tensor of rotated/2 radians per position, float).

    frequency_j = base^(-2j/rotated), for `scaling` changed as a checkpoint's `rope_scaling` entry says (the same keys):
        - None, {"rope_type": "default"}: as they are
        - {"rope_type": "linear", "factor"}: all divided by the factor
        - {"rope_type": "llama3", "factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"}: those that turn fewer
          than low_freq_factor times within the original length divided by the factor, those that turn more than high_freq_factor times kept, a
          linear ramp over the number of turns between
        - {"rope_type": "yarn", "factor", "original_max_position_embeddings", "beta_fast" (32), "beta_slow" (1), "attention_factor"}: the same with a
          ramp that is linear in j, from the pair that turns beta_fast times to the one that turns beta_slow times (both rounded
          outwards), and a magnitude of 0.1 ln(factor) + 1 unless attention_factor is given
    """
    assert rotated > 0 and rotated % 2 == 0, f"Expected a positive even {rotated = }"
    assert base > 0, f"Expected {base = } to be > 0"
    frequencies = base ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)
    magnitude = 1.0
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "linear":
        frequencies = frequencies / scaling["factor"]
    elif kind == "llama3":
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        turns = scaling["original_max_position_embeddings"] * frequencies / (2 * math.pi)
        kept = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        frequencies = frequencies * (kept + (1.0 - kept) / scaling["factor"])
    elif kind == "yarn":
        factor, length = scaling["factor"], scaling["original_max_position_embeddings"]

        def pair(turns):  # the (fractional) pair that turns so often within the original length
            return rotated * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

        first = max(math.floor(pair(scaling.get("beta_fast") or 32)), 0)
        last = min(math.ceil(pair(scaling.get("beta_slow") or 1)), rotated - 1)
        divided = ((torch.arange(rotated // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        frequencies = frequencies * (1.0 - divided + divided / factor)
        magnitude = scaling.get("attention_factor")
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif kind != "default":
        raise ValueError(f"rope_type {kind!r} is not one of default, linear, llama3, yarn")
    return frequencies.to(device), float(magnitude)
