"""Codes drawn from a model's logits, on the GPU through qinco_sample_codes (csrc/sample_kernel.hpp).

A prior over the codes of a residual quantiser answers with K logits per step (or one per inverted list); the codes drawn here are what
`model(codes, step="decode")` and the look-up decoders take, and the list ids what `qinco_amd.lists.group_rows` sorts by.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from . import _lib

_CODES = {np.dtype(np.int64): _lib.CODE_I64, np.dtype(np.int32): _lib.CODE_I32}


_TYPES = {torch.float32: _lib.T_F32, torch.float16: _lib.T_F16, torch.bfloat16: _lib.T_BF16}


def on_device(t, what: str):
    """A torch CUDA tensor, or an error that names the argument."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{what} must be a torch CUDA tensor")
    return t


def row_type(t, what: str) -> int:
    """QINCO_T_* of a tensor of rows."""
    code = _TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    return code


def unit_rows(t):
    """The same 2-D tensor with neighbouring elements of a row next to each other (a copy only where they are not)."""
    return t if t.shape[1] == 1 or t.stride(1) == 1 else t.contiguous()


def on_its_device(dev, call, *args) -> None:
    """One library call on the current stream of `dev` (its last argument), with `dev` current: kernels are launched on a stream of the
    current device."""
    if torch.cuda.current_device() == dev.index:
        rc = call(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = call(*args, torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        _lib.check(rc)


def sample_codes(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, code_dtype=np.int64, return_logp: bool = False):
    """One code per row of `logits` (n, V) float32 / float16 / bfloat16 from the given random numbers `u` (n,) in [0, 1), float32 or
    float64; torch CUDA tensors, asynchronous on the current stream.  Returns codes (n,) of `code_dtype` (int64 or int32) [and the log
    probability of each among the codes that were kept, (n,) float32].

    Codes are ordered by (logit descending, index ascending); with e_i = exp((z_i - max z) / temperature) the kept ones are the first
    `top_k`, of these every one with less than `top_p` of their mass before it (the first always), of these those with e_i >= `min_p`;
    the code is the lowest kept index at which the kept mass, summed in index order, exceeds u times its total.  top_k <= 0 or >= V,
    top_p >= 1 and min_p <= 0 switch a cut off.  temperature 0 takes the largest logit, the lowest index among equals (log probability
    0).  -inf and NaN are never drawn; a row with nothing to draw answers -1 with log probability -inf.  Decisions are taken in 64 bits:
    the same inputs give the same codes, whatever else is in the batch.

    temperature, top_p, min_p (float32) and top_k (int32) may be tensors (n,) with a value per row; there a temperature <= 0 is 0."""
    lib = _lib.load()
    on_device(logits, "logits")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be (n, V) with V >= 1, got {tuple(logits.shape)}")
    dtype = row_type(logits, "logits")
    logits = unit_rows(logits)
    n, V = logits.shape
    dev = logits.device
    if on_device(u, "u").shape != (n,) or u.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"u must be ({n},) float32 or float64, got {tuple(u.shape)} {u.dtype}")
    u = u.contiguous()
    keep = [u]
    params = _lib.QincoSampleParams(struct_bytes=C.sizeof(_lib.QincoSampleParams))
    for name, value, want in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                              ("min_p", min_p, torch.float32)):
        if isinstance(value, torch.Tensor):
            if on_device(value, name).shape != (n,) or value.dtype != want:
                raise ValueError(f"{name} must be a number or ({n},) {want}, got {tuple(value.shape)} {value.dtype}")
            keep.append(value.contiguous())
            setattr(params, name + "_rows", keep[-1].data_ptr())
        elif want is torch.int32:
            params.top_k = min(max(int(value), 0), V)
        else:
            setattr(params, name, float(value))
    if any(t.device != dev for t in keep):
        raise ValueError("logits, u and the settings must be on one device")
    if not isinstance(temperature, torch.Tensor) and not 0.0 <= params.temperature < math.inf:
        raise ValueError(f"temperature must be finite and >= 0, got {temperature}")
    if params.top_p != params.top_p or params.min_p != params.min_p or params.min_p > 1.0:
        raise ValueError(f"top_p must be a number and min_p at most 1, got {top_p} and {min_p}")
    if np.dtype(code_dtype) not in _CODES:
        raise ValueError("code_dtype must be int64 or int32 (a row with nothing to draw answers -1)")
    code = _CODES[np.dtype(code_dtype)]
    codes = torch.empty(n, dtype=torch.int64 if code == _lib.CODE_I64 else torch.int32, device=dev)
    logp = torch.empty(n, dtype=torch.float32, device=dev) if return_logp else None
    need = lib.qinco_sample_workspace(n, V)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    on_its_device(dev, lib.qinco_sample_codes, logits.data_ptr(), dtype, logits.stride(0), n, V, u.data_ptr(), u.dtype == torch.float64,
                  C.byref(params), codes.data_ptr(), code, logp.data_ptr() if return_logp else None,
                  ws.data_ptr() if need else None, need)
    return (codes, logp) if return_logp else codes
