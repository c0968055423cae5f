from .sampler import ROW_DTYPE, PendingLogprobs, Sampler, SamplingParams, TokenLogprob, pack_rows

__all__ = ["ROW_DTYPE", "PendingLogprobs", "Sampler", "SamplingParams", "TokenLogprob", "pack_rows"]
