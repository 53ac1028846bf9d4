"""Log probabilities of given tokens, entropy and the largest alternatives, of logits or of what the vocabulary's packed weights make of hidden states."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from .experts import _rows, _workspace
from .ops import _DTYPES, _check_rhs, _ptr, _require_gpu, _stream
from .quantization import QuantizationConfig, QuantizationEncoding


class LogProbs(NamedTuple):
    """``logprobs`` float32 of the shape of the tokens, ``entropy`` float32 of the rows; with alternatives, ``top_ids`` int32 and ``top_logprobs`` float32 ``[..., top_k]``."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


def _outputs(tokens, lead, top_k: int, vocab: int, device):
    """The checked tokens of rows of shape ``lead``, how many a row has, and the empty results."""
    _require_gpu(tokens, "tokens")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    if tokens.device != device:
        raise ValueError(f"tokens must live on {device}, got {tokens.device}")
    lead = tuple(lead)
    if tuple(tokens.shape) == lead:
        per_row = 1
    elif tuple(tokens.shape[:-1]) == lead and tokens.shape[-1] > 0:
        per_row = tokens.shape[-1]
    else:
        raise ValueError(f"tokens have shape {tuple(tokens.shape)}; the rows have {lead} (one token each) or {lead} and a number of tokens")
    if not 0 <= top_k <= min(vocab, _lib.QMM_MAX_TOP):
        raise ValueError(f"top_k={top_k} of {vocab} (0 .. {_lib.QMM_MAX_TOP})")
    f32 = {"dtype": torch.float32, "device": device}
    return per_row, LogProbs(torch.empty(tokens.shape, **f32), torch.empty(lead, **f32), torch.empty((*lead, top_k), dtype=torch.int32, device=device) if top_k else None,
                             torch.empty((*lead, top_k), **f32) if top_k else None)


def logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0) -> LogProbs:
    """Log probabilities ``logits[token] - logsumexp(logits)`` of the given tokens, the entropy of each row, and its ``top_k`` (up to 64) largest alternatives.

    ``logits`` is float32 or bfloat16 ``[..., vocab]`` (rows may be a view of wider, padded ones); ``tokens`` int32 or int64, one for each row or ``[..., count]`` of
    them.  A negative token is padding and gets 0, one that is not in the vocabulary NaN.  Alternatives come by falling logit, equal ones by rising index.  Sums are in
    float32, the largest value apart, so that small entropies and log probabilities keep their digits.  A row of ``-inf`` only gives ``-inf`` and an entropy of 0, a
    row with NaN or ``+inf`` NaN.
    """
    done = (_lib._call or _lib.call()).logprobs(logits, tokens, top_k)
    if done is not None:
        return LogProbs(*done)
    stride = _rows(logits, "logits")
    vocab, lead = logits.shape[-1], logits.shape[:-1]
    rows = logits.numel() // vocab
    per_row, out = _outputs(tokens, lead, top_k, vocab, logits.device)
    lib = _lib.load()
    dt = _DTYPES[logits.dtype]
    need = lib.qmm_logprobs_workspace_bytes(dt, rows, vocab, top_k)
    ws = _workspace(need, logits.device)
    with torch.cuda.device(logits.device):
        rc = lib.qmm_logprobs(_ptr(logits), dt, stride, rows, vocab, _ptr(tokens), int(tokens.dtype == torch.int64), per_row, top_k, _ptr(out.logprobs), _ptr(out.entropy),
                              _ptr(out.top_ids), _ptr(out.top_logprobs), _ptr(ws), need, _stream(logits))
    _lib.check(rc, "logprobs")
    return out


def qmatmul_logprobs(encoding: QuantizationEncoding, config: Optional[QuantizationConfig], lhs: torch.Tensor, *rhs: torch.Tensor, tokens: torch.Tensor,
                     top_k: int = 0) -> LogProbs:
    """``logprobs(qmatmul(encoding, config, lhs, *rhs), tokens, top_k)``: a vocabulary product whose logits, kept in the call's workspace some rows at a time,
    nobody else needs (a text scored token by token takes no ``rows x vocab`` tensor)."""
    done = (_lib._call or _lib.call()).matmul_logprobs(encoding, config, lhs, rhs, tokens, top_k)
    if done is not None:
        return LogProbs(*done)
    if not isinstance(encoding, QuantizationEncoding):
        raise TypeError("encoding must be a QuantizationEncoding")
    _require_gpu(lhs, "lhs")
    if lhs.dtype not in _DTYPES:
        raise TypeError(f"lhs must be float32 or bfloat16, got {lhs.dtype}")
    if lhs.dim() < 1 or lhs.numel() == 0:
        raise ValueError("qmatmul_logprobs of an empty tensor")
    k, lead = lhs.shape[-1], lhs.shape[:-1]
    m = lhs.numel() // k
    n, cfg_p = _check_rhs(encoding, config, k, rhs)
    if n == 0:
        raise ValueError("qmatmul_logprobs of an empty tensor")
    if any(t.device != lhs.device for t in rhs):
        raise ValueError("lhs and rhs must be on one device")
    per_row, out = _outputs(tokens, lead, top_k, n, lhs.device)
    lib = _lib.load()
    dt = _DTYPES[lhs.dtype]
    ptrs = (C.c_void_p * len(rhs))(*[t.data_ptr() for t in rhs])
    need = lib.qmm_matmul_logprobs_workspace_bytes(encoding.code, cfg_p, dt, m, n, k, top_k)
    ws = _workspace(need, lhs.device)
    with torch.cuda.device(lhs.device):
        rc = lib.qmm_matmul_logprobs(encoding.code, cfg_p, _ptr(lhs), dt, m, k, ptrs, len(rhs), n, _ptr(tokens), int(tokens.dtype == torch.int64), per_row, top_k,
                                     _ptr(out.logprobs), _ptr(out.entropy), _ptr(out.top_ids), _ptr(out.top_logprobs), _ptr(ws), need, _stream(lhs))
    _lib.check(rc, "qmatmul_logprobs")
    return out
