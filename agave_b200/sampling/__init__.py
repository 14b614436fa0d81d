from .sampler import HISTORY_CAP, Sampler, SamplingParams, TokenScore

__all__ = ["HISTORY_CAP", "Sampler", "SamplingParams", "TokenScore"]
