"""Codes drawn from a model's logits, on the GPU through qinco_sample_codes (csrc/sample_kernel.hpp).

A prior over the codes of a residual quantiser answers with K logits per step (or one per inverted list); the codes drawn here are what
`model(codes, step="decode")` and the look-up decoders take, and the list ids what `qinco_amd.lists.group_rows` sorts by.
"""
from __future__ import annotations

import ctypes as C
import functools
import math

import numpy as np
import torch

from . import _lib

_CODES = {np.dtype(np.int64): (_lib.CODE_I64, torch.int64), np.dtype(np.int32): (_lib.CODE_I32, torch.int32)}
_CODES[np.int64], _CODES[np.int32] = _CODES[np.dtype(np.int64)], _CODES[np.dtype(np.int32)]


_RANDOM, _FLOAT, _INT = (torch.float32, torch.float64), (torch.float32,), (torch.int32,)
_PARAMS_BYTES = C.sizeof(_lib.QincoSampleParams)
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


def as_stored(t):
    """The same tensor with its values in memory: a view that torch conjugates or negates on reading is copied."""
    return t.resolve_conj().resolve_neg() if t.is_neg() or t.is_conj() else t


def unit_rows(t):
    """The same 2-D tensor with neighbouring elements of a row next to each other (a copy only where they are not)."""
    t = as_stored(t)
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
# the handle of a device's current stream without a Stream object around it (2 us of a call of 12), where this torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


being_traced = torch.jit.is_tracing
# torch.fx's recorder, None where there is none
recording = functools.partial(torch._C._get_dispatch_mode, torch._C._TorchDispatchModeKey.PROXY)


def refuse_trace(what: str) -> None:
    """torch.fx's recorder (make_fx) and torch.jit.trace see torch's own operators alone: what they make of a call would answer the memory that the
    library fills."""
    raise RuntimeError(f"{what} cannot be recorded by torch.fx" if recording() is not None else f"{what} cannot be traced by torch.jit")


def on_its_device(index: int, call, *args) -> None:
    """One library call on the current stream of device `index` (its last argument), with that device current: kernels are launched on a
    stream of the current device."""
    if _current_device() == index:
        rc = call(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, _raw_stream(index))
    if rc:
        _lib.check(rc)


def _rows(t, n: int, dev, what: str, types):
    """A value per row, on the logits' device."""
    if on_device(t, what).shape != (n,) or t.dtype not in types or t.device != dev:
        raise ValueError(f"{what} must be ({n},) of {' or '.join(map(str, types))} on {dev}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return as_stored(t).contiguous()


def sample_codes(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, code_dtype=np.int64, return_logp: bool = False):
    """One code per row of `logits` (n, V) float32 / float16 / bfloat16 from the given random numbers `u` (n,) in [0, 1), float32 or
    float64; torch CUDA tensors, asynchronous on the current stream.  Returns codes (n,) of `code_dtype` (int64 or int32) [and the log
    probability of each among the codes that were kept, (n,) float32].

    Codes are ordered by (logit descending, index ascending); with e_i = exp((z_i - max z) / temperature) the kept ones are the first
    `top_k`, of these every one with less than `top_p` of their mass before it (the first always), of these those with e_i >= `min_p`;
    the code is the lowest kept index at which the kept mass, summed in index order, exceeds u times its total.  top_k <= 0 or >= V,
    top_p >= 1 and min_p <= 0 switch a cut off.  temperature 0 takes the largest logit, the lowest index among equals (log probability
    0).  -inf and NaN are never drawn; a row with nothing to draw answers -1 with log probability -inf.  The same inputs give the same
    codes, whatever else is in the batch.  Masses and sums are held in 62 bits of the row's total: top_p and u decide as in exact arithmetic
    unless they lie within 2^-43 of a border (V <= 20480; 2^-39 at 2^20 codes, 2^-35 at 2^24).

    temperature, top_p, min_p (float32) and top_k (int32) may be tensors (n,) with a value per row; there a temperature <= 0 or NaN is 0, a
    min_p above 1 is 1, and NaN switches a cut off.

    The log probabilities are values: no derivative goes through them, whether the logits require one or carry a tangent.  For a gradient
    take torch.log_softmax(logits / temperature, 1) at the codes (of what is kept, where something is cut)."""
    lib = _lib.load()
    if being_traced() or recording() is not None:
        refuse_trace("sample_codes")
    shape = on_device(logits, "logits").shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"logits must be (n, V) with V >= 1, got {tuple(shape)}")
    dtype = row_type(logits, "logits")
    logits = unit_rows(logits)
    n, V = shape
    dev = logits.device
    u = _rows(u, n, dev, "u", _RANDOM)
    code = _CODES.get(code_dtype) or _CODES.get(np.dtype(code_dtype))
    if code is None:
        raise ValueError("code_dtype must be int64 or int32 (a row with nothing to draw answers -1)")
    params = _lib.QincoSampleParams(_PARAMS_BYTES)
    keep = []                                          # (arrays made contiguous live until the call is enqueued)
    if isinstance(temperature, torch.Tensor):
        keep.append(_rows(temperature, n, dev, "temperature", _FLOAT))
        params.temperature_rows = keep[-1].data_ptr()
    else:
        params.temperature = temperature = float(temperature)
        if not 0.0 <= temperature < math.inf:
            raise ValueError(f"temperature must be finite and >= 0, got {temperature}")
    if isinstance(top_k, torch.Tensor):
        keep.append(_rows(top_k, n, dev, "top_k", _INT))
        params.top_k_rows = keep[-1].data_ptr()
    else:
        top_k = int(top_k)
        params.top_k = top_k if 0 < top_k < V else 0
    if isinstance(top_p, torch.Tensor):
        keep.append(_rows(top_p, n, dev, "top_p", _FLOAT))
        params.top_p_rows = keep[-1].data_ptr()
    else:
        params.top_p = top_p = float(top_p)
        if top_p != top_p:
            raise ValueError("top_p must be a number")
    if isinstance(min_p, torch.Tensor):
        keep.append(_rows(min_p, n, dev, "min_p", _FLOAT))
        params.min_p_rows = keep[-1].data_ptr()
    else:
        params.min_p = min_p = float(min_p)
        if not min_p <= 1.0:
            raise ValueError(f"min_p must be at most 1, got {min_p}")
    codes = torch.empty(n, dtype=code[1], device=dev)
    logp = torch.empty(n, dtype=torch.float32, device=dev) if return_logp else None
    need = lib.qinco_sample_workspace(n, V)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    on_its_device(dev.index, lib.qinco_sample_codes, logits.data_ptr(), dtype, logits.stride(0), n, V, u.data_ptr(), u.dtype == torch.float64,
                  params, codes.data_ptr(), code[0], logp.data_ptr() if return_logp else None, ws.data_ptr() if need else None, need)
    return (codes, logp) if return_logp else codes
