from .params import SamplingParams
from .rng import philox4x32, uniform
from .verify import verify_drafts

__all__ = ["SamplingParams", "philox4x32", "uniform", "verify_drafts"]
