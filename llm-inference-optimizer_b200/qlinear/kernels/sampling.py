"""Drawing tokens from logits by given random numbers (libqlinear).

The reference's engines decode greedily, by ``argmax`` of the lm_head's logits
(src/engine/paged_engine.py:146-147).  ``sample_tokens`` draws instead, with
temperature, top-k, top-p and min-p for the batch or for each row, in one
launch over the logits as the lm_head leaves them.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._launch import call, call_flags

_DTYPES = {torch.float16: _lib.QL_DTYPE_F16, torch.bfloat16: _lib.QL_DTYPE_BF16, torch.float32: _lib.QL_DTYPE_F32}


def _setting(value, rows: int, dtype: torch.dtype, device: torch.device, what: str):
    """A setting's tensor (kept alive by the caller), its address or 0, and the number for all rows."""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype:
            raise TypeError(f"{what} must be a number or {dtype}, got {value.dtype}")
        assert value.shape == (rows,) and value.device == device, \
            f"{what} must be ({rows},) on {device}, got {tuple(value.shape)} on {value.device}"
        value = value.contiguous()
        return value, value.data_ptr(), 0
    return None, 0, value


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=None, top_p=None, min_p=None,
                  return_logprobs: bool = False, out: torch.Tensor = None):
    """A token for each row of logits (rows, vocab), fp16, bf16 or fp32 with
    unit stride along the vocabulary, drawn by uniform (rows,) fp32 in [0, 1).

    With weights exp((x - max) / temperature), tokens in the order of their
    logits, equal ones by index:

    * top_k: the first top_k are kept (None or 0 and less: all);
    * top_p: of those, the ones before which the weights come to less than
      top_p of their sum (None or 1 and more: all);
    * min_p: of those, the ones whose weight is at least min_p of the largest
      (None or 0: all);
    * the first is always kept.

    The token is the first, by index, at which the running sum of the kept
    weights exceeds uniform times their sum; what is kept and which token it is
    are decided as by sums in fp64.  temperature 0
    (and less) takes the largest logit, the first of equal ones.  Each setting
    is a number, or a tensor (rows,) of fp32 (top_k: int32).  Logits of minus
    infinity or NaN are never drawn; where some are infinite, only those are.

    Returns ids (rows,) int64, in ``out`` if given: -1 for a row with nothing to
    draw, which is no index of an embedding.  With ``return_logprobs``, also the
    log of the probability with which each was drawn, fp32 (0 at temperature 0,
    minus infinity for -1); its sum may be one of fp32 weights, so it is off by up
    to 6e-7 absolute, beside fp32's rounding: more than the value itself where a
    token is all but certain."""
    assert logits.is_cuda and logits.dim() == 2, f"logits must be a CUDA tensor (rows, vocab), got {tuple(logits.shape)}"
    code = _DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"logits must be fp16, bf16 or fp32, got {logits.dtype}")
    rows, vocab = logits.shape
    dev = logits.device
    assert 1 <= vocab <= _lib.QL_SAMPLE_MAX_VOCAB, f"vocab must be from 1 to {_lib.QL_SAMPLE_MAX_VOCAB}, got {vocab}"
    if uniform.dtype != torch.float32:
        raise TypeError(f"uniform must be fp32, got {uniform.dtype}")
    assert uniform.shape == (rows,) and uniform.device == dev, \
        f"uniform must be ({rows},) on {dev}, got {tuple(uniform.shape)} on {uniform.device}"
    stride = logits.stride()
    if stride[1] != 1 and vocab > 1 or stride[0] < vocab and rows > 1:
        logits = logits.contiguous()
        stride = logits.stride()
    if not uniform.is_contiguous():
        uniform = uniform.contiguous()
    heat, heat_ptr, heat_all = _setting(temperature, rows, torch.float32, dev, "temperature")
    k, k_ptr, k_all = _setting(0 if top_k is None else top_k, rows, torch.int32, dev, "top_k")
    p, p_ptr, p_all = _setting(1.0 if top_p is None else top_p, rows, torch.float32, dev, "top_p")
    m, m_ptr, m_all = _setting(0.0 if min_p is None else min_p, rows, torch.float32, dev, "min_p")
    if not isinstance(k_all, int):
        raise TypeError(f"top_k must be a whole number, got {k_all!r}")
    if not 0.0 <= heat_all < float("inf") or not p_all >= 0.0 or not 0.0 <= m_all <= 1.0:
        raise ValueError(f"temperature must be finite and not negative, top_p not negative, min_p from 0 to 1: got "
                         f"{heat_all}, {p_all}, {m_all}")
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=dev)
    else:
        assert out.shape == (rows,) and out.dtype == torch.int64 and out.device == dev and out.is_contiguous(), \
            f"out must be contiguous int64 ({rows},) on {dev}"
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev) if return_logprobs else None
    if rows > 0:
        packed = _lib.SAMPLE_TOKENS_ARGS.pack(
            logits.data_ptr(), uniform.data_ptr(), heat_ptr, k_ptr, p_ptr, m_ptr, out.data_ptr(),
            logprobs.data_ptr() if return_logprobs else 0, rows, vocab, stride[0] if rows > 1 else vocab, code, k_all,
            heat_all, p_all, m_all, call_flags())
        call(_lib.load().ql_sample_tokens, packed, dev)
    return (out, logprobs) if return_logprobs else out


__all__ = ["sample_tokens"]
