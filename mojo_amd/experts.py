"""The experts of a mixture-of-experts block on packed weights: the router, and the products grouped by expert.

A GGUF file holds the experts of a layer as one tensor per projection, ``uint8[experts, N, K / epb * bpb]`` (:meth:`GGUFWeights.tensor` hands it out so); these
calls take it as it is.  A block is ::

    routing = route_experts(x @ router.T, top_k)
    h = qmatmul_experts_swiglu(encoding, x, gate, up, routing, out_dtype=x.dtype)
    x = qmatmul_experts_sum(encoding, h, down, routing, residual=x, out_dtype=x.dtype)

Nothing is copied to the host on the way (how many rows an expert has is known on the device only), so a block can be captured into a graph.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from .ops import _DTYPES, _ptr, _require_gpu, _stream
from .quantization import QuantizationEncoding

_SCORING = {"softmax": _lib.QMM_SOFTMAX, "sigmoid": _lib.QMM_SIGMOID}


class ExpertRouting:
    """Which experts each token goes to, and the pairs of a token and an expert sorted by expert.

    ``experts`` int32 ``[..., top]`` (a value outside ``0 .. num_experts - 1``: none), ``weights`` float32 of the same shape, ``offsets`` int32
    ``[num_experts + 1]`` and ``order`` int32 ``[tokens * top]``: the pairs ``top * token + j`` of expert ``e`` are ``order[offsets[e]:offsets[e + 1]]``, those
    without an expert come last.  :func:`route_experts` and :func:`group_experts` make one; their results are not checked again on the device.
    """

    __slots__ = ("experts", "weights", "offsets", "order")

    def __init__(self, experts: torch.Tensor, weights: torch.Tensor, offsets: torch.Tensor, order: torch.Tensor):
        if (_lib._call or _lib.call()).routing_fits(experts, weights, offsets, order):
            self.experts, self.weights, self.offsets, self.order = experts, weights, offsets, order
            return
        for t, name, dtype in ((experts, "experts", torch.int32), (weights, "weights", torch.float32), (offsets, "offsets", torch.int32), (order, "order", torch.int32)):
            _require_gpu(t, name)
            if t.dtype != dtype:
                raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
            if t.device != experts.device:
                raise ValueError(f"{name} must live on {experts.device}, got {t.device}")
        if experts.dim() < 1 or experts.numel() == 0:
            raise ValueError("experts must be [..., top] of at least one token")
        if weights.shape != experts.shape or order.numel() != experts.numel() or order.dim() != 1 or offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError("weights must have the shape of experts, order its number of values, offsets one value more than there are experts")
        self.experts, self.weights, self.offsets, self.order = experts, weights, offsets, order

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1

    @property
    def top(self) -> int:
        return self.experts.shape[-1]

    @property
    def tokens(self) -> int:
        return self.experts.numel() // self.experts.shape[-1]


def _made(experts, weights, offsets, order) -> ExpertRouting:
    r = ExpertRouting.__new__(ExpertRouting)
    r.experts, r.weights, r.offsets, r.order = experts, weights, offsets, order
    return r


def _workspace(need: int, device) -> Optional[torch.Tensor]:
    return torch.empty((need,), dtype=torch.uint8, device=device) if need > 0 else None


def _rows(t: torch.Tensor, name: str) -> int:
    """The values between the rows of a tensor whose last dimension is dense and whose leading ones can be counted through."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU (got device {t.device}); there is no CPU path")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    if t.dim() < 1 or t.numel() == 0:
        raise ValueError(f"{name} must have at least one row")
    if t.is_contiguous():
        return t.shape[-1]
    if (t.stride(-1) != 1 and t.shape[-1] != 1) or any(t.stride(i) != t.stride(i + 1) * t.shape[i + 1] for i in range(t.dim() - 2) if t.shape[i] != 1):
        raise ValueError(f"{name} must have dense rows at equal distances")
    return t.stride(-2) if t.dim() > 1 else t.shape[-1]


def route_experts(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", renormalize: bool = True, bias: Optional[torch.Tensor] = None,
                  scale: float = 1.0) -> ExpertRouting:
    """The ``top_k`` experts of each token from a router's logits, float32 or bfloat16 ``[..., num_experts]`` (rows may be a view of wider ones).

    The scores are ``softmax(logits)`` or ``sigmoid(logits)`` in float32; the largest are chosen, equal ones by rising index, NaN last.  ``bias`` (float32
    ``[num_experts]``) is added to the scores for the choice only.  A chosen expert's weight is its score, divided by the sum of the chosen ones if ``renormalize``, times
    ``scale``.  A token whose logits are all ``-inf`` gets weights of 0.
    """
    done = (_lib._call or _lib.call()).route(logits, top_k, scoring, renormalize, bias, scale)
    if done is not None:
        return _made(*done)
    stride = _rows(logits, "logits")
    experts = logits.shape[-1]
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    if experts > _lib.QMM_MAX_EXPERTS or not 1 <= top_k <= min(experts, _lib.QMM_MAX_TOP):
        raise ValueError(f"top_k={top_k} of {experts} experts (at most {_lib.QMM_MAX_TOP} of {_lib.QMM_MAX_EXPERTS})")
    if bias is not None:
        _require_gpu(bias, "bias")
        if bias.dtype != torch.float32 or tuple(bias.shape) != (experts,) or bias.device != logits.device:
            raise TypeError(f"bias must be float32[{experts}] on the device of the logits")
    lead, dev = logits.shape[:-1], logits.device
    tokens = logits.numel() // experts
    ids = torch.empty((*lead, top_k), dtype=torch.int32, device=dev)
    weights = torch.empty((*lead, top_k), dtype=torch.float32, device=dev)
    offsets = torch.empty((experts + 1,), dtype=torch.int32, device=dev)
    order = torch.empty((tokens * top_k,), dtype=torch.int32, device=dev)
    lib = _lib.load()
    need = lib.qmm_experts_group_workspace_bytes(tokens * top_k, experts, top_k)
    ws = _workspace(need, dev)
    with torch.cuda.device(dev):
        rc = lib.qmm_route_experts(_ptr(logits), _DTYPES[logits.dtype], stride, tokens, experts, top_k, _SCORING[scoring], _ptr(bias), int(bool(renormalize)), float(scale),
                                   _ptr(ids), _ptr(weights), _ptr(offsets), _ptr(order), _ptr(ws), need, _stream(logits))
    _lib.check(rc, "route_experts")
    return _made(ids, weights, offsets, order)


def group_experts(experts: torch.Tensor, weights: torch.Tensor, num_experts: int) -> ExpertRouting:
    """The :class:`ExpertRouting` of experts and weights that come from elsewhere: ``experts`` int32 ``[..., top]``, where a value outside
    ``0 .. num_experts - 1`` stands for none (a padded token, an expert of another rank), ``weights`` float32 of the same shape."""
    _require_gpu(experts, "experts")
    _require_gpu(weights, "weights")
    if experts.dtype != torch.int32 or experts.dim() < 1 or experts.numel() == 0:
        raise TypeError("experts must be a non-empty int32 tensor [..., top]")
    if weights.dtype != torch.float32 or weights.shape != experts.shape or weights.device != experts.device:
        raise TypeError("weights must be float32, of the shape and on the device of experts")
    if not 1 <= num_experts <= _lib.QMM_MAX_EXPERTS or experts.shape[-1] > _lib.QMM_MAX_TOP:
        raise ValueError(f"{experts.shape[-1]} of {num_experts} experts (at most {_lib.QMM_MAX_TOP} of {_lib.QMM_MAX_EXPERTS})")
    dev, pairs = experts.device, experts.numel()
    offsets = torch.empty((num_experts + 1,), dtype=torch.int32, device=dev)
    order = torch.empty((pairs,), dtype=torch.int32, device=dev)
    lib = _lib.load()
    need = lib.qmm_experts_group_workspace_bytes(pairs, num_experts, 1)
    ws = _workspace(need, dev)
    with torch.cuda.device(dev):
        rc = lib.qmm_group_experts(_ptr(experts), pairs, num_experts, _ptr(offsets), _ptr(order), _ptr(ws), need, _stream(experts))
    _lib.check(rc, "group_experts")
    return _made(experts, weights, offsets, order)


def _matrices(encoding: QuantizationEncoding, t: torch.Tensor, name: str, k: int, routing: ExpertRouting):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU (got device {t.device}); there is no CPU path")
    if t.dtype != torch.uint8 or t.dim() != 3 or t.numel() == 0:
        raise TypeError(f"{name} must be a non-empty uint8 tensor [experts, N, row bytes] of packed blocks")
    if t.shape[0] != routing.num_experts:
        raise ValueError(f"{name} holds {t.shape[0]} experts, the routing has {routing.num_experts}")
    if t.shape[2] != encoding.packed_row_bytes(k):
        raise ValueError(f"{name} rows hold {t.shape[2]} bytes; K={k} in {encoding.name} needs {encoding.packed_row_bytes(k)}")
    if t.stride(2) != 1 or (t.stride(1) != t.shape[2] and t.shape[1] != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1] * t.shape[2]):
        raise ValueError(f"the matrix of each expert in {name} must be contiguous")
    if t.device != routing.experts.device:
        raise ValueError(f"{name} must live on {routing.experts.device}, got {t.device}")


def _experts(op: int, what: str, encoding, lhs, mats, routing, residual, out_dtype) -> torch.Tensor:
    done = (_lib._call or _lib.call()).experts(op, encoding, lhs, mats[0][0], mats[-1][0], routing, residual, out_dtype)
    if done is not None:
        return done
    if not isinstance(encoding, QuantizationEncoding) or not encoding.is_gguf:
        raise TypeError(f"{what} takes a GGUF weight encoding")
    if not isinstance(routing, ExpertRouting):
        raise TypeError("routing must be an ExpertRouting (route_experts, group_experts)")
    _require_gpu(lhs, "lhs")
    if lhs.dtype not in _DTYPES:
        raise TypeError(f"lhs must be float32 or bfloat16, got {lhs.dtype}")
    if out_dtype not in _DTYPES:
        raise TypeError("out_dtype must be float32 or bfloat16")
    if lhs.dim() < 1 or lhs.numel() == 0:
        raise ValueError(f"{what} of an empty tensor")
    if lhs.device != routing.experts.device:
        raise ValueError(f"lhs must live on {routing.experts.device}, got {lhs.device}")
    k, tokens, top = lhs.shape[-1], routing.tokens, routing.top
    rows = lhs.numel() // k
    if rows not in (tokens, tokens * top):
        raise ValueError(f"lhs has {rows} rows; the routing has {tokens} tokens with {top} experts each")
    for t, name in mats:
        _matrices(encoding, t, name, k, routing)
    (w, _), (w2, name2) = mats[0], mats[-1]
    n = w.shape[1]
    if w2.shape != w.shape:
        raise ValueError(f"gate {tuple(w.shape)} and up {tuple(w2.shape)} must have the same shape")
    lead = routing.experts.shape[:-1]
    if residual is not None:
        _require_gpu(residual, "residual")
        if residual.dtype not in _DTYPES or residual.numel() != tokens * n or residual.shape[-1] != n or residual.device != lhs.device:
            raise TypeError(f"residual must be a float32 or bfloat16 tensor of {tokens} x {n} values on the device of lhs")
    out = torch.empty((*lead, n) if op == _lib.QMM_EXPERTS_SUM else (*lead, top, n), dtype=out_dtype, device=lhs.device)
    flags = _lib.QMM_FLAG_OUT_BF16 if out_dtype == torch.bfloat16 else 0
    lhs_dt = _DTYPES[lhs.dtype]
    lib = _lib.load()
    need = lib.qmm_matmul_experts_workspace_bytes(op, encoding.code, lhs_dt, rows, tokens, top, routing.num_experts, n, k, flags)
    ws = _workspace(need, lhs.device)
    r = _lib.Routing(routing.offsets.data_ptr(), routing.order.data_ptr(), routing.experts.data_ptr(), routing.weights.data_ptr(), tokens, top, routing.num_experts)
    with torch.cuda.device(lhs.device):
        rc = lib.qmm_matmul_experts(op, encoding.code, C.byref(r), _ptr(lhs), lhs_dt, rows, k, _ptr(w), w.stride(0), _ptr(w2), w2.stride(0), n, _ptr(residual),
                                    _DTYPES[residual.dtype] if residual is not None else 0, _ptr(out), _ptr(ws), need, flags, _stream(lhs))
    _lib.check(rc, what)
    return out


def qmatmul_experts(encoding: QuantizationEncoding, lhs: torch.Tensor, rhs: torch.Tensor, routing: ExpertRouting, *,
                    out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``out[..., j, :] = lhs[row] @ dequantize(rhs[e])^T`` for the ``j``-th expert ``e`` of each token: ``[..., top, N]``, zeros where there is none.

    ``rhs`` is ``uint8[experts, N, K / epb * bpb]`` (the matrix of an expert contiguous, the experts at any distance: a slice of a tensor that holds more).  ``lhs``
    is float32 or bfloat16 ``[..., K]``, a row for each token or one for each of its experts (``[..., top, K]``).  The products are those of :func:`qmatmul` on
    each expert's rows (Q4_0: of the lhs in Q8_0 blocks, whose scale is the largest magnitude times ``1 / 127`` where :func:`qmatmul` divides by 127).
    """
    return _experts(_lib.QMM_EXPERTS_EACH, "qmatmul_experts", encoding, lhs, ((rhs, "rhs"),), routing, None, out_dtype)


def qmatmul_experts_swiglu(encoding: QuantizationEncoding, lhs: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, routing: ExpertRouting, *,
                           out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``silu(lhs @ dequantize(gate[e])^T) * (lhs @ dequantize(up[e])^T)`` for each expert ``e`` of each token: ``[..., top, N]``.

    ``gate`` and ``up`` as ``rhs`` of :func:`qmatmul_experts`, of one shape; of a tensor that holds both, ``t[:, :N]`` and ``t[:, N:]``.
    """
    return _experts(_lib.QMM_EXPERTS_SWIGLU, "qmatmul_experts_swiglu", encoding, lhs, ((gate, "gate"), (up, "up")), routing, None, out_dtype)


def qmatmul_experts_sum(encoding: QuantizationEncoding, lhs: torch.Tensor, rhs: torch.Tensor, routing: ExpertRouting, *,
                        residual: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``residual + sum_j weights[j] * (lhs[row] @ dequantize(rhs[e_j])^T)`` over the experts of each token, in their order: ``[..., N]``.

    ``lhs`` and ``rhs`` as in :func:`qmatmul_experts`; ``residual`` float32 or bfloat16 ``[..., N]``.  The sum is in float32.
    """
    return _experts(_lib.QMM_EXPERTS_SUM, "qmatmul_experts_sum", encoding, lhs, ((rhs, "rhs"),), routing, residual, out_dtype)
