import math
from typing import Optional, Tuple

import torch
from torch import Tensor


# What an entry of each kind may say, and what does not change the frequencies of any (`rotated` is the caller's; a base has to be the same).
_KEYS = {
    "default": {"factor"},
    "linear": {"factor"},
    "llama3": {"factor", "low_freq_factor", "high_freq_factor"},
    "yarn": {"factor", "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate"},
}
_KEYS_OF_ALL = {"rope_type", "type", "original_max_position_embeddings", "finetuned", "partial_rotary_factor", "rope_theta"}


def _yarn_magnitude(factor: float, scaling: dict) -> float:
    def of(m: float) -> float:
        return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

    if "attention_factor" in scaling:
        return scaling["attention_factor"]
    above, below = scaling.get("mscale"), scaling.get("mscale_all_dim")
    if above and below:
        return of(above) / of(below)
    # one of them alone is read differently by different programs, but for a factor of one above the line
    if below or above not in (None, 0, 1):
        raise ValueError(f"mscale and mscale_all_dim come together but the entry has {above} and {below}")
    return of(1.0)


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
        - {"rope_type": "yarn", "factor", "original_max_position_embeddings", "beta_fast" (32), "beta_slow" (1), "truncate" (True), "attention_factor",
          "mscale", "mscale_all_dim"}: the same with a ramp that is linear in j, from the pair that turns beta_fast times to the one that turns
          beta_slow times (both rounded outwards unless truncate is False).  The magnitude is attention_factor; without one
          (0.1 mscale ln(factor) + 1) / (0.1 mscale_all_dim ln(factor) + 1); without these 0.1 ln(factor) + 1.  (Programs that scale
          their scores by mscale_all_dim too do so in the attention's scale.)
    An entry with another key that is set, or with a rope_theta that is not `base`, is refused with a ValueError.
    """
    assert rotated > 0 and rotated % 2 == 0, f"Expected a positive even {rotated = }"
    assert base > 0, f"Expected {base = } to be > 0"
    frequencies = base ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)
    magnitude = 1.0
    scaling = {key: v for key, v in (scaling or {}).items() if v is not None}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _KEYS:
        raise ValueError(f"rope_type {kind!r} is not one of {', '.join(_KEYS)}")
    unknown = sorted(set(scaling) - _KEYS[kind] - _KEYS_OF_ALL)
    if unknown:
        raise ValueError(f"the scaling entry has {', '.join(unknown)}, which rope_type {kind!r} is not known to have")
    if scaling.get("rope_theta", base) != base:
        raise ValueError(f"the scaling entry has rope_theta {scaling['rope_theta']} but base is {base}")
    if kind == "default" and scaling.get("factor", 1) != 1:
        raise ValueError(f"the scaling entry has factor {scaling['factor']}, which rope_type {kind!r} does not use")
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

        first, last = pair(scaling.get("beta_fast") or 32), pair(scaling.get("beta_slow") or 1)
        if scaling.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rotated - 1)
        divided = ((torch.arange(rotated // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        frequencies = frequencies * (1.0 - divided + divided / factor)
        magnitude = _yarn_magnitude(factor, scaling)
    return frequencies.to(device), float(magnitude)
