from .wrapped import ExpertRoute, combine_experts, route_experts
from .reference import reference_combine_experts, reference_route_experts

__all__ = ["ExpertRoute", "combine_experts", "route_experts", "reference_combine_experts", "reference_route_experts"]
