from .sampler import PendingLogprobs, Sampler, SamplingParams, TokenLogprob, check_top, uniform

__all__ = ["PendingLogprobs", "Sampler", "SamplingParams", "TokenLogprob", "check_top", "uniform"]
