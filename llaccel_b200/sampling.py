"""Sampling tokens from the model's integer logits (llx_sample of include/llx.h)."""
from __future__ import annotations

import struct

import torch

from .cuda_backend import _check as _check_code
from .cuda_backend import load_library
from .paged import _cuda, _refuse, _stream, _vector

_SAMPLE = struct.Struct("=13q")


def sample(logits, random, *, exponent, vocab=None, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
    """One token per row of `logits` (int16 `[rows, >= vocab]`, a logit's value is l * 2^exponent;
    `exponent` is the model's E_LOGIT), drawn with `random`, float64 numbers of [0, 1).

    Per-row tensors: `temperature` float32 (default 1; 0 or below: the largest logit), `top_k` int32
    (default and <= 0: all), `top_p` float32 (default and >= 1: all), `min_p` float32 (default 0).
    Tokens are ordered by logit, then by index; the shortest prefix that any of the three allows is
    kept, top_p counting within top_k.  The draw goes through the kept tokens by index.  Everything
    is computed in integers, so the same inputs give the same tokens on any split of the work.
    Returns (tokens int32, probability float32 of each token among the kept ones), in `out` if given."""
    dev = _cuda(logits, "logits")
    if len(logits.shape) != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows, vocabulary] with dense rows")
    R, ld = logits.shape
    V = ld if vocab is None else vocab
    if V > ld:
        raise ValueError(f"vocab {V} exceeds the {ld} columns of logits")
    _refuse(dev, torch.int16, logits=logits)
    _refuse(dev, torch.float32, temperature=temperature, top_p=top_p, min_p=min_p)
    _refuse(dev, torch.int32, top_k=top_k)
    _refuse(dev, torch.float64, random=random)
    ptr = [_vector(t, name, R) if t is not None else 0
           for name, t in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p), ("top_k", top_k))]
    if out is None:
        token, prob = torch.empty(R, dtype=torch.int32, device=logits.device), torch.empty(R, dtype=torch.float32, device=logits.device)
    else:
        token, prob = out
        _refuse(dev, torch.int32, token=token)
        _refuse(dev, torch.float32, prob=prob)
    args = _SAMPLE.pack(logits.data_ptr(), logits.stride(0) if R > 1 else ld, R, V, exponent, *ptr,
                        _vector(random, "random", R), _vector(token, "token", R), _vector(prob, "prob", R), dev)
    lib = load_library()
    code = lib.llx_sample(args, _stream(dev))
    if code:
        _check_code(lib, code)
    return token, prob
