from .history import TokenHistory
from .sampler import Sampler, SamplingParams, pack_allowed, request_seed, sorted_bias, uniform_draw

__all__ = ["Sampler", "SamplingParams", "TokenHistory", "pack_allowed", "request_seed", "sorted_bias", "uniform_draw"]
