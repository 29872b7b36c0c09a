"""How likely given tokens were: log probabilities, entropy, alternatives.

``token_logprobs`` goes with ``select.sample_rows`` and ``select.select_step``:
what the served API reports next to the sampled tokens, or the score of a given
text.  It runs one kernel of ``libyapd_select.so`` on the current CUDA stream.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _native as N

_DTYPES = {torch.float32: N.YAPD_DTYPE_F32, torch.bfloat16: N.YAPD_DTYPE_BF16, torch.float16: N.YAPD_DTYPE_F16}


@dataclass
class TokenLogprobs:
    logprob: torch.Tensor | None        # (R,) float32, NaN where the target is outside the vocabulary
    entropy: torch.Tensor               # (R,) float32, in nats
    top_logprobs: torch.Tensor | None   # (R, top_n) float32, most likely first
    top_ids: torch.Tensor | None        # (R, top_n) int32, equal ones in ascending order; -1: none


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, *, top_n: int = 0) -> TokenLogprobs:
    """Log probabilities of ``targets`` ``(R,)`` (int64 or int32) under the
    softmax of each row of ``logits`` ``(R, V)`` (float32, bfloat16 or float16;
    any row stride), the rows' entropies, and the ``top_n <= 32`` most likely
    tokens of each row.

    Arithmetic is in 32 bits; the sum over the tokens leaves out the most likely
    one, so that its log probability keeps its digits near 0.  A target outside ``[0, V)`` (the select step's -1)
    gives NaN.  Masked tokens (-inf) have probability 0 and are no alternatives;
    a row with fewer than ``top_n`` others ends in ids -1 with -inf.  A row with
    NaN or +inf, or with nothing but -inf, gives NaN and ids -1.
    """
    if not logits.is_cuda:
        raise ValueError("token_logprobs runs on CUDA tensors only (no CPU fallback)")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= N.YAPD_LOGPROBS_MAX_V:
        raise ValueError(f"logits must be (R, V) with 1 <= V <= {N.YAPD_LOGPROBS_MAX_V}, got {tuple(logits.shape)}")
    if not 0 <= top_n <= N.YAPD_LOGPROBS_MAX_TOP:
        raise ValueError(f"top_n must be 0 to {N.YAPD_LOGPROBS_MAX_TOP}, got {top_n}")
    R, V = logits.shape
    if R >= 2 ** 31:        # the kernels count rows in 32 bits
        raise ValueError(f"logits must have fewer than 2^31 rows, got {R}")
    if (V > 1 and logits.stride(1) != 1) or (R > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    dev, index = logits.device, logits.get_device()
    a = N.LogprobsArgs()
    a.R, a.V, a.top_n, a.logits_dtype = R, V, top_n, _DTYPES[logits.dtype]
    a.logits, a.stride_row = logits.data_ptr(), logits.stride(0)
    logprob = top = ids = None
    if targets is not None:
        if targets.shape != (R,) or targets.dtype not in (torch.int64, torch.int32) or targets.get_device() != index:
            raise ValueError(f"targets must be an int64 or int32 ({R},) tensor on {dev}")
        if targets.dtype != torch.int64 or not targets.is_contiguous():
            targets = targets.to(torch.int64).contiguous()
        logprob = torch.empty(R, dtype=torch.float32, device=dev)
        a.targets, a.logprob = targets.data_ptr(), logprob.data_ptr()
    entropy = torch.empty(R, dtype=torch.float32, device=dev)
    a.entropy = entropy.data_ptr()
    if top_n:
        top = torch.empty(R, top_n, dtype=torch.float32, device=dev)
        ids = torch.empty(R, top_n, dtype=torch.int32, device=dev)
        a.top_logprobs, a.top_ids = top.data_ptr(), ids.data_ptr()
    if R:
        entry = N.lib().yapd_token_logprobs
        if torch.cuda.current_device() == index:
            rc = entry(a, torch._C._cuda_getCurrentRawStream(index))
        else:
            with torch.cuda.device(dev):
                rc = entry(a, torch._C._cuda_getCurrentRawStream(index))
        if rc:
            N.check(rc)
    return TokenLogprobs(logprob, entropy, top, ids)
