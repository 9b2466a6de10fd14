"""The next tokens from a step's logits, drawn on the device.

Prism's scheduler copies the logits to the host and takes their argmax or samples there (engine/scheduler.py:266-273),
once per step and sequence.  sample_tokens leaves them where they are: the drawn tokens go straight into the next
step's embedding, and a captured decode step can hold its own sampling.
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import _raw_stream, _require_gpu
from .packed import _on


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: float | torch.Tensor = 1.0,
                  top_k: int | torch.Tensor | None = None, top_p: float | torch.Tensor | None = None,
                  min_p: float | torch.Tensor | None = None, return_logprobs: bool = False):
    """Draws a token for every row of ``logits`` [rows, vocab] (bf16, fp16 or fp32) -> int64 [rows].

    With w_i = exp((x_i - max x) / temperature), tokens in the order of descending logits (of equal ones the lowest
    token first): the first ``top_k`` stay (None or 0: all), of those the shortest prefix whose weights sum to
    ``top_p`` of theirs (None or 1: all), of those the ones with w_i >= ``min_p`` (None or 0: all).  The token is the
    first, in the order of the vocabulary, at which the running sum of the weights that stay passes
    ``uniforms[row]`` (fp32 [rows], 0 to 1) times their sum: the same numbers give the same tokens.  ``temperature`` 0
    takes the largest logit.  Each setting is a number (taken as fp32) or a tensor with one for each row (fp32; int32
    for top_k).

    -inf and NaN logits are never drawn; a row that has nothing else gives -1.  With ``return_logprobs`` also the
    logarithm of the drawn token's probability among those that stay, fp32 [rows].  Asynchronous on the current
    stream; can be captured (new numbers are written into ``uniforms`` between replays)."""
    _require_gpu(logits, "logits")
    dev = logits.device
    with _on(dev):
        return _lib.fast().sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, return_logprobs,
                                         _raw_stream(dev.index))
