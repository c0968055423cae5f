"""Sampling options and the sampler that turns logits into token ids.

Options and their meaning follow the reference (src/engine/sampling.rs:9-48):
``temperature`` (<= 0: greedy), ``top_k`` (<= 0: off), ``top_p`` (0: greedy,
outside [0, 1]: 1), ``ignore_eos``, ``max_tokens`` (at least 1).  ``logprobs`` is this engine's addition: how many of the
most likely tokens are reported with their log probabilities beside each output token's
own (None: no log probabilities at all); they are those of the model's distribution,
before temperature and cut-offs.  So is ``seed``: the uniform number of a draw is a counter-based random
number keyed by (seed, index of the output token), so a request samples the same
tokens whatever else shares its batch.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..kernels import ops

ROW_DTYPE = np.dtype([("temperature", "<f4"), ("top_k", "<i4"), ("top_p", "<f4"), ("seed_lo", "<u4"),
                      ("seed_hi", "<u4"), ("counter", "<u4"), ("pad0", "<i4"), ("pad1", "<i4")])
assert ROW_DTYPE.itemsize == 32


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.0
    top_k: int = -1
    top_p: float = 1.0
    ignore_eos: bool = False
    max_tokens: int = 1024
    seed: Optional[int] = None
    logprobs: Optional[int] = None

    def normalized(self) -> "SamplingParams":
        top_p = self.top_p if (math.isfinite(self.top_p) and 0.0 <= self.top_p <= 1.0) else 1.0
        if self.logprobs is not None and not 0 <= int(self.logprobs) <= ops.MAX_TOP_LOGPROBS:
            raise ValueError(f"logprobs must be 0 to {ops.MAX_TOP_LOGPROBS} alternatives, or None")
        return SamplingParams(float(self.temperature), int(self.top_k), float(top_p), bool(self.ignore_eos), max(int(self.max_tokens), 1),
                              self.seed, None if self.logprobs is None else int(self.logprobs))

    @property
    def greedy(self) -> bool:
        return not (self.temperature > 0.0) or self.top_p == 0.0


def pack_rows(rows: Sequence[Tuple[SamplingParams, int, int]]) -> np.ndarray:
    """(params, seed, counter) per row -> the 32-byte records that the kernel reads."""
    out = np.zeros(len(rows), dtype=ROW_DTYPE)
    for i, (p, seed, counter) in enumerate(rows):
        seed &= (1 << 64) - 1
        out[i] = (p.temperature, p.top_k, p.top_p, seed & 0xFFFFFFFF, seed >> 32,
                  counter & 0xFFFFFFFF, 0, 0)
    return out


@dataclass(frozen=True)
class TokenLogprob:
    """A token's log probability, the entropy of the distribution that it came from (in nats) and that distribution's most likely
    tokens, (id, log probability) each, most likely first."""
    token: int
    logprob: float
    entropy: float
    top: Tuple[Tuple[int, float], ...] = ()


class PendingLogprobs:
    """Log probabilities on their way to the host.  ``wanted``: of each row how many alternatives, None for a row that wants nothing."""

    def __init__(self, logits: torch.Tensor, ids: torch.Tensor, wanted: Sequence[Optional[int]]):
        most = max((w for w in wanted if w is not None), default=0)
        found = ops.token_logprobs(logits, ids, top=min(most, logits.shape[1]))
        self.wanted = list(wanted)
        self._host = [torch.empty(t.shape, dtype=t.dtype, pin_memory=True) for t in (ids, *found)]
        for host, t in zip(self._host, (ids, *found)):
            host.copy_(t, non_blocking=True)
        self._event = torch.cuda.Event()
        self._event.record(torch.cuda.current_stream(logits.device))

    def finish(self) -> List[Optional[TokenLogprob]]:
        self._event.synchronize()
        tokens, logprobs, entropy, top_ids, top_logprobs = (t.tolist() for t in self._host)
        return [None if w is None else TokenLogprob(tokens[r], logprobs[r], entropy[r], tuple(zip(top_ids[r][:w], top_logprobs[r][:w])))
                for r, w in enumerate(self.wanted)]


class Sampler:
    def __init__(self, device: torch.device):
        self.device = torch.device(device)

    def sample_device(self, logits: torch.Tensor,
                      rows: Sequence[Tuple[SamplingParams, int, int]]) -> torch.Tensor:
        """int32 token ids [rows] on the device."""
        if logits.shape[0] != len(rows):
            raise ValueError(f"{logits.shape[0]} logits rows but {len(rows)} sampling rows")
        if all(p.greedy for p, _, _ in rows):
            return ops.argmax(logits)
        packed = torch.from_numpy(pack_rows(rows).view(np.uint8).reshape(len(rows), 32))
        params = packed.pin_memory().to(self.device, non_blocking=True)
        return ops.sample(logits, params)

    def sample(self, logits: torch.Tensor, rows: Sequence[Tuple[SamplingParams, int, int]]) -> List[int]:
        ids = self.sample_device(logits, rows).cpu().tolist()
        if any(i < 0 for i in ids):
            raise RuntimeError("sampling produced no valid token for a row (were the logits finite?)")
        return ids
