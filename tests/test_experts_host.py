"""What the experts' and log-probability entries refuse without touching a device, and the 64-bit restatement itself."""
import ctypes as C

import numpy as np
import pytest
import torch

import experts_reference as R
from mojo_amd import ExpertRouting, QuantizationEncoding as QE, _lib, logprobs, qmatmul_experts, route_experts

P = C.c_void_p(4096)  # never read: every call here is refused first


@pytest.fixture(scope="module")
def lib():
    try:
        return _lib.load()
    except RuntimeError as e:
        pytest.skip(str(e))


def message(lib):
    return lib.qmm_last_error().decode()


def test_route_and_group_refusals(lib):
    def route(dtype=0, stride=64, tokens=4, experts=64, top=8, scoring=0, ws=None, ws_bytes=0, logits=P):
        return lib.qmm_route_experts(logits, dtype, stride, tokens, experts, top, scoring, None, 1, 1.0, P, P, P, P, ws, ws_bytes, None)

    for kw in ({"logits": None}, {"dtype": 2}, {"stride": 63}, {"tokens": 0}, {"experts": 1025, "stride": 2000}, {"experts": 0}, {"top": 0}, {"top": 65, "experts": 128, "stride": 128}, {"experts": 4},
               {"scoring": 2}, {"tokens": 1 << 60}):
        assert route(**kw) == -1 and "qmm_route_experts" in message(lib), kw
    assert lib.qmm_experts_group_workspace_bytes(64, 64, 8) == 0
    need = lib.qmm_experts_group_workspace_bytes(8 * 1000, 64, 8)
    assert need > 0 and route(tokens=1000, ws=P, ws_bytes=need - 1) == -4
    assert lib.qmm_group_experts(P, 0, 8, P, P, None, 0, None) == -1
    assert lib.qmm_group_experts(P, 5, 1025, P, P, None, 0, None) == -1
    assert lib.qmm_group_experts(None, 5, 8, P, P, None, 0, None) == -1
    assert lib.qmm_group_experts(P, 5000, 8, P, P, None, 0, None) == -4


def test_product_refusals(lib):
    def call(op=0, encoding=1, tokens=4, top=2, experts=8, lhs=P, dtype=0, rows=4, k=512, rhs=P, stride=64 * 288, rhs2=None, stride2=64 * 288, n=64, residual=None, out=P, ws=P, ws_bytes=1 << 40, flags=0,
             weights=4096):
        r = _lib.Routing(4096, 4096, 4096, weights, tokens, top, experts)
        return lib.qmm_matmul_experts(op, encoding, C.byref(r), lhs, dtype, rows, k, rhs, stride, rhs2, stride2, n, residual, 0, out, ws, ws_bytes, flags, None)

    for kw in ({"op": 3}, {"encoding": 3}, {"encoding": 8}, {"tokens": 0}, {"top": 65}, {"experts": 0}, {"experts": 1025}, {"lhs": None}, {"lhs": C.c_void_p(4100)}, {"dtype": 2}, {"rows": 5}, {"k": 500},
               {"k": 0}, {"n": 0}, {"n": (1 << 18) + 1}, {"rhs": None}, {"stride": 64 * 288 - 1}, {"op": 1}, {"op": 1, "rhs2": P, "stride2": 5}, {"residual": P}, {"out": None}, {"flags": 1}, {"flags": 2},
               {"op": 2, "weights": None}):
        assert call(**kw) == -1 and "qmm_matmul_experts" in message(lib), kw
    need = lib.qmm_matmul_experts_workspace_bytes(2, 1, 0, 4, 4, 2, 8, 64, 512, 0)
    assert need >= 4 * 2 * 64 * 4
    assert call(op=2, ws_bytes=need - 1) == -4 and call(op=2, ws=None, ws_bytes=need) == -4 and call(op=2, ws=C.c_void_p(4096 + 64)) == -1


def test_logprobs_refusals(lib):
    def call(logits=P, dtype=0, stride=100, rows=4, vocab=100, tokens=P, per_row=1, top=3, lp=P, h=P, ids=P, values=P, ws=None, ws_bytes=0):
        return lib.qmm_logprobs(logits, dtype, stride, rows, vocab, tokens, 1, per_row, top, lp, h, ids, values, ws, ws_bytes, None)

    for kw in ({"logits": None}, {"dtype": 2}, {"stride": 99}, {"rows": 0}, {"vocab": 0}, {"vocab": (1 << 22) + 1, "stride": 1 << 31}, {"tokens": None}, {"per_row": -1}, {"top": 65}, {"top": -1},
               {"vocab": 2}, {"lp": None}, {"h": None}, {"ids": None}, {"values": None}, {"logits": C.c_void_p(4098)}):
        assert call(**kw) == -1 and "qmm_logprobs" in message(lib), kw
    need = lib.qmm_logprobs_workspace_bytes(0, 1, 128256, 20)
    assert need > 0 and call(rows=1, vocab=128256, stride=128256, top=20, ws=P, ws_bytes=need - 1) == -4
    rhs = (C.c_void_p * 1)(4096)
    def product(lhs=P, m=4, k=512, n=1000, dtype=0, ws=P, ws_bytes=0, top=0):
        return lib.qmm_matmul_logprobs(1, None, lhs, dtype, m, k, rhs, 1, n, P, 1, 1, top, P, P, P, P, ws, ws_bytes, None)

    assert product(lhs=None) == -1 and product(m=0) == -1 and product(k=0) == -1 and product(dtype=2) == -1 and product(top=65) == -1
    assert product() == -4 and product(ws=None, ws_bytes=1 << 40) == -4


def test_no_cpu_path():
    x = torch.zeros(4, 8)
    i = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        route_experts(x, 2)
    with pytest.raises(ValueError, match="GPU"):
        ExpertRouting(i, torch.zeros(4, 2), i[0], i.reshape(-1))
    with pytest.raises(ValueError, match="GPU"):
        logprobs(x, i[:, 0])
    with pytest.raises(TypeError):
        qmatmul_experts(QE.Q4_K, x, x, None)


def test_the_restatement_by_hand():
    ids = torch.tensor([[2, 0], [-1, 2], [5, 0]], dtype=torch.int32)
    offsets, order = R.sorted_pairs(ids, 3)
    assert offsets.tolist() == [0, 2, 2, 4] and order.tolist() == [1, 5, 0, 3, 2, 4]
    chosen, w = R.choose(torch.tensor([[0.0, 2.0, 2.0, -1.0]]), 2, "softmax", True)
    assert chosen.tolist() == [[1, 2]] and w.tolist() == [[0.5, 0.5]]
    lp, h, top, _ = R.log_probabilities(torch.tensor([[1.0, 1.0, -torch.inf]]), torch.tensor([1]), 2)
    assert lp.item() == pytest.approx(-np.log(2)) and h.item() == pytest.approx(np.log(2)) and top.tolist() == [[0, 1]]
    for e in (QE.Q4_0, QE.Q4_K, QE.Q5_K, QE.Q6_K):
        w32 = 0.02 * np.random.default_rng(0).standard_normal((2, 8, 512), dtype=np.float32)
        w = R.weights64(e, R.pack(e, w32))
        assert w.shape == (2, 8, 512) and np.abs(w.numpy() - w32).max() < 0.02
        x = torch.randn(3, 512)
        y, bound = R.products(e, x, w, torch.tensor([[1], [-1], [0]], dtype=torch.int32))
        assert (y[1] == 0).all() and torch.allclose(y[0, 0], w[1] @ R.lhs64(e, x)[0]) and (bound[0] > 0).all()
