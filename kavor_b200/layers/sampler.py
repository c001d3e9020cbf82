"""Sampler (drop-in for kavor/layers/sampler.py).

Gumbel-max sampling ``argmax(logits / T + Gumbel)`` in one streaming pass per
row, greedy argmax (lowest index on ties) when ``T == 0``. The seed is a
persistent device int32 advanced by one on every call before sampling
(sampler.py:54-59), so a captured CUDA graph advances it on every replay.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import nn

from kavor_b200 import _kernels as K


class Sampler(nn.Module):

    def __init__(self):
        super().__init__()
        self.register_buffer("seed", torch.zeros((), dtype=torch.int32, device="cuda"))

    def forward(self, logits: torch.Tensor, temperatures: torch.Tensor, out: torch.Tensor | None = None):
        assert logits.is_contiguous() and temperatures.is_contiguous()
        self.seed.add_(1)
        return K.sample(logits, temperatures, self.seed, out=out)


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # fp32 [N]: log probability of the given token
    ranks: torch.Tensor         # int64 [N]: entries before it (higher logit, or equal at a lower index); -1 for no token
    entropy: torch.Tensor       # fp32 [N]: entropy of the row, nats
    top_ids: torch.Tensor       # int64 [N, top_k]: most likely entries, in that order
    top_logprobs: torch.Tensor  # fp32 [N, top_k]


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities of given tokens under the logits [N, vocab] (bf16, fp16
    or fp32), their ranks, the rows' entropy and the ``top_k`` (at most 32) most
    likely entries, from one streaming pass. An id of -1 asks for no token
    (logprob 0, rank -1). Banned entries (-inf) have probability 0; a row of
    only -inf has logprobs -inf and entropy 0; a row holding NaN or +inf gives
    NaN, with the NaN entries first in order."""
    return TokenLogprobs(*K.token_logprobs(logits, token_ids, top_k))
