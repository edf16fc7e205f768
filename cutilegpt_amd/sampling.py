"""Choosing the next tokens: temperature, top-k, top-p and min-p from given random numbers.

The reference samples with array operations, temperature and top-k
(``cutile_gpt/models/gpt.py:207-226``); here one kernel takes a batch of rows, with
settings for each row where they differ, and the random numbers are an input: the same
numbers give the same tokens, eagerly or in a captured graph.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib

__all__ = ["sample_tokens"]

_CODE = {torch.float32: _lib.CGPT_F32, torch.bfloat16: _lib.CGPT_BF16, torch.float16: _lib.CGPT_F16}


def _rows_of(name: str, what: str, t: torch.Tensor, B: int, dtype: torch.dtype, dev: int) -> int:
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != B or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{name}: {what} must be {B} contiguous {dtype} values on the logits' GPU, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor, None] = None, top_p: Union[float, torch.Tensor, None] = None,
                  min_p: Union[float, torch.Tensor, None] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token a row (B,) int64 from ``logits`` (B, vocabulary; float32, bfloat16 or
    float16, contiguous rows of any stride) and ``u`` (B,) float32 of [0, 1).

    A token's weight is exp((logit - largest) / temperature).  In the order of the logits,
    equal ones by index, the first ``top_k`` are kept; of these the shortest run that has
    at least ``top_p`` of their weight; of it those of at least ``min_p`` of the largest
    weight.  The draw is the first index, in the order of the vocabulary, at which the
    running sum of the kept weights exceeds u times their sum.  Weights are exact to 2^-44
    of the largest (smaller ones are 0: a mask may be -inf or any number far enough down) and
    their sums exact, so a draw does not depend on how they are added.

    Each setting is a number for all rows or a tensor (B,), float32 (``top_k`` int32), read
    on the device.  None, a ``top_k`` of 0, a ``top_p`` of 1 or a ``min_p`` of 0 cut nothing.
    ``temperature`` 0 takes the largest logit (the first of equals).  NaN logits are skipped
    and -inf never chosen; a row with nothing else gives -1."""
    name = "sample_tokens"
    if not isinstance(logits, torch.Tensor) or not isinstance(u, torch.Tensor) or not logits.is_cuda:
        raise ValueError(f"{name}: logits and u must be torch tensors on one GPU")
    dev, code = logits.get_device(), _CODE.get(logits.dtype)
    if code is None:
        raise ValueError(f"{name}: unsupported dtype {logits.dtype} (float32, bfloat16 or float16)")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"{name}: logits must be (B, vocabulary), got {tuple(logits.shape)}")
    B, V = logits.shape
    ld, one = logits.stride()
    if (one != 1 and V > 1) or (ld < V and B > 1):
        logits = logits.contiguous()
        ld = V
    pu = _rows_of(name, "u", u, B, torch.float32, dev)
    pt = pk = pp = pm = None
    if isinstance(temperature, torch.Tensor):
        pt, temperature = _rows_of(name, "temperature", temperature, B, torch.float32, dev), 0.0
    elif not temperature >= 0.0:
        raise ValueError(f"{name}: temperature must be at least 0, got {temperature}")
    if isinstance(top_k, torch.Tensor):
        pk, top_k = _rows_of(name, "top_k", top_k, B, torch.int32, dev), 0
    elif top_k is None:
        top_k = 0
    elif isinstance(top_k, bool) or not isinstance(top_k, int) or top_k < 0:
        raise ValueError(f"{name}: top_k must be an int of at least 0, got {top_k!r}")
    if isinstance(top_p, torch.Tensor):
        pp, top_p = _rows_of(name, "top_p", top_p, B, torch.float32, dev), 1.0
    elif top_p is None:
        top_p = 1.0
    elif not 0.0 <= top_p <= 1.0:
        raise ValueError(f"{name}: top_p must lie in [0, 1], got {top_p}")
    if isinstance(min_p, torch.Tensor):
        pm, min_p = _rows_of(name, "min_p", min_p, B, torch.float32, dev), 0.0
    elif min_p is None:
        min_p = 0.0
    elif not 0.0 <= min_p <= 1.0:
        raise ValueError(f"{name}: min_p must lie in [0, 1], got {min_p}")
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=logits.device)
    else:
        _rows_of(name, "out", out, B, torch.int64, dev)
    args = (logits.data_ptr(), B, V, max(ld, V), code, pu, pt, pk, pp, pm, temperature, min(top_k, V), top_p, min_p,
            out.data_ptr())
    fn = _lib.load().cgpt_sample
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc, name)
    return out
