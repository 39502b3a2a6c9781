from .params import SamplingParams
from .rules import edit_logits
from .sampler import Sampler, sample_tokens

__all__ = ["SamplingParams", "Sampler", "edit_logits", "sample_tokens"]
