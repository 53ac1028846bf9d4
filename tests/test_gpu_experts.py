"""The router, the pairs sorted by expert, and the experts' products against 64 bits."""
import math
import random

import numpy as np
import pytest
import torch

import experts_reference as R
from gguf_writer import write_gguf
from mojo_amd import (ExpertRouting, GGUFWeights, QuantizationEncoding as QE, group_experts, qmatmul_experts, qmatmul_experts_sum, qmatmul_experts_swiglu, route_experts)

pytestmark = pytest.mark.gpu
GGUF = (QE.Q4_0, QE.Q4_K, QE.Q5_K, QE.Q6_K)
DEV = "cuda:0"


def logits_of(seed, tokens, experts, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (2.0 * torch.randn(tokens, experts, generator=g) + torch.randn(1, experts, generator=g)).to(dtype)


def check_routing(r, ids, experts):
    assert torch.equal(r.experts.cpu().reshape(ids.shape), ids)
    offsets, order = R.sorted_pairs(ids, experts)
    assert torch.equal(r.offsets.cpu(), offsets) and torch.equal(r.order.cpu(), order)


@pytest.mark.parametrize("scoring", ("softmax", "sigmoid"))
@pytest.mark.parametrize("renormalize", (True, False))
@pytest.mark.parametrize("tokens,experts,top,dtype", ((1, 64, 8, torch.float32), (1, 8, 2, torch.bfloat16), (3, 1, 1, torch.float32), (128, 60, 4, torch.bfloat16), (129, 128, 8, torch.float32),
                                                      (1025, 256, 8, torch.bfloat16), (70, 1024, 64, torch.float32), (9000, 65, 3, torch.float32)))
def test_route_experts(tokens, experts, top, dtype, scoring, renormalize):
    x = logits_of(tokens + experts, tokens, experts, dtype)
    r = route_experts(x.to(DEV), top, scoring=scoring, renormalize=renormalize, scale=1.5)
    ids, w = R.choose(x, top, scoring, renormalize, scale=1.5)
    check_routing(r, ids, experts)
    # x - m is rounded by u |x - m| (logits within 32 of each other), exp, sums of up to 16 values a lane and six steps, quotients: 2^6 u in all
    assert ((r.weights.cpu().double() - w).abs() <= 2.0 ** 6 * R.U * w).all()


@pytest.mark.parametrize("scoring", ("softmax", "sigmoid"))
def test_route_experts_with_a_bias_for_the_choice(scoring):
    x = logits_of(5, 300, 96)
    bias = 0.3 * torch.randn(96, generator=torch.Generator().manual_seed(6))
    r = route_experts(x.to(DEV), 6, scoring=scoring, bias=bias.to(DEV))
    ids, w = R.choose(x, 6, scoring, True, bias)
    check_routing(r, ids, 96)
    assert ((r.weights.cpu().double() - w).abs() <= 2.0 ** 6 * R.U * w).all()
    assert not torch.equal(ids, R.choose(x, 6, scoring, True)[0])


def test_equal_scores_go_by_rising_index():
    x = torch.zeros(40, 130)
    x[1:, 100] = -0.0
    x[2:, 7] = 1.0
    x[2:, 90] = 1.0
    for bias in (None, torch.zeros(130, device=DEV)):
        r = route_experts(x.to(DEV), 5, bias=bias)
        check_routing(r, R.choose(x, 5, "softmax", True)[0], 130)


def test_masked_empty_and_nan_logits():
    x = torch.randn(6, 70)
    x[0, 3:] = -torch.inf       # three experts for four places
    x[1] = -torch.inf           # none
    x[2, ::2] = torch.finfo(torch.float32).min
    x[3, 5] = torch.nan
    x[4] = torch.nan
    r = route_experts(x.to(DEV), 4)
    ids, w = r.experts.cpu(), r.weights.cpu()
    assert sorted(ids[0, :3].tolist()) == [0, 1, 2] and ids[0, 3] == 3 and w[0, 3] == 0 and abs(w[0].sum() - 1) < 1e-6
    assert ids[1].tolist() == [0, 1, 2, 3] and (w[1] == 0).all()
    assert (ids[2] % 2 == 1).all() and 5 not in ids[3]
    assert ids[4].tolist() == [0, 1, 2, 3] and w[4].isnan().all()
    assert (w[[2, 3, 5]].sum(-1) - 1).abs().max() < 1e-6
    assert (route_experts(x[1:2].to(DEV), 4, renormalize=False).weights == 0).all()


def test_rows_of_wider_logits_and_leading_dimensions():
    wide = logits_of(8, 60, 100)
    x = wide[:, :64]
    r = route_experts(wide.to(DEV)[:, :64], 4)
    check_routing(r, R.choose(x, 4, "softmax", True)[0], 64)
    r = route_experts(x.to(DEV).reshape(3, 20, 64), 4)
    assert r.experts.shape == (3, 20, 4) and r.weights.shape == (3, 20, 4) and r.tokens == 60
    check_routing(r, R.choose(x, 4, "softmax", True)[0], 64)
    with pytest.raises(ValueError, match="equal distances"):
        route_experts(wide.to(DEV).t()[:64].t()[:, ::2], 4)


@pytest.mark.parametrize("tokens,top,experts", ((1, 1, 1), (1, 7, 5), (1023, 1, 64), (1025, 1, 64), (128, 8, 16), (9000, 8, 1024), (70001, 2, 3)))
def test_group_experts_and_pairs_without_one(tokens, top, experts):
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, experts + 1, (tokens, top), generator=g, dtype=torch.int32)  # (-1 and `experts`: none)
    ids[0, 0] = 2 ** 31 - 1
    r = group_experts(ids.to(DEV), torch.ones(tokens, top, device=DEV), experts)
    check_routing(r, ids, experts)


class Case:
    def __init__(self, encoding, tokens, experts, top, n, k, dtype, seed=0, per_pair=False, without=0.0, mats=1):
        g = torch.Generator().manual_seed(seed + 7 * tokens + n)
        self.encoding, self.tokens, self.top, self.n, self.k, self.dtype = encoding, tokens, top, n, k, dtype
        self.packed = [R.pack(encoding, (0.02 * torch.randn(experts, n, k, generator=g)).numpy()) for _ in range(mats)]
        self.w = [R.weights64(encoding, p) for p in self.packed]
        self.lhs = torch.randn(*((tokens, top, k) if per_pair else (tokens, k)), generator=g).to(dtype)
        x = torch.randn(tokens, experts, generator=g) + 1.5 * torch.randn(1, experts, generator=g)
        self.ids, w = R.choose(x, top, "softmax", True)
        self.ids[torch.rand(self.ids.shape, generator=g) < without] = -1
        self.weights = w.float()
        self.routing = group_experts(self.ids.to(DEV), self.weights.to(DEV), experts)
        self.g = g

    def gpu(self, i=0):
        return self.packed[i].to(DEV)

    def products(self, i=0):
        return R.products(self.encoding, self.lhs, self.w[i], self.ids)


def check(got, want, bound, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    error = (got.cpu().double() - want).abs()
    limit = R.rounded(bound, want, dtype)
    assert (error <= limit).all(), f"worst {(error / limit).max():.3g} of the bound at {torch.nonzero(error > limit)[0].tolist()}"


SHAPES = (  # tokens, experts, top, n, k
    (1, 8, 2, 64, 256), (1, 16, 8, 40, 1024), (2, 4, 4, 33, 512), (5, 8, 2, 96, 2048), (16, 8, 2, 200, 768), (33, 60, 4, 72, 512), (64, 4, 1, 136, 1024), (130, 8, 3, 264, 512),
    (300, 3, 2, 320, 256), (700, 16, 2, 48, 512))


@pytest.mark.parametrize("encoding", GGUF, ids=lambda e: e.name)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("shape", SHAPES)
def test_products_by_expert(encoding, dtype, shape):
    c = Case(encoding, *shape, dtype)
    for out in (torch.float32, torch.bfloat16):
        check(qmatmul_experts(encoding, c.lhs.to(DEV), c.gpu(), c.routing, out_dtype=out), *c.products(), out)


def silu_bound(g, gb, u, ub):
    """silu has slopes within 1.1; exp, quotient and product: 8 u"""
    s = g * torch.sigmoid(g)
    return s * u, 1.1 * gb * (u.abs() + ub) + s.abs() * ub + 8 * R.U * (s * u).abs()


@pytest.mark.parametrize("encoding", GGUF, ids=lambda e: e.name)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("shape", SHAPES)
def test_gated_pair(encoding, dtype, shape):
    c = Case(encoding, *shape, dtype, mats=2)
    (g, gb), (u, ub) = c.products(0), c.products(1)
    for out in (torch.float32, torch.bfloat16):
        check(qmatmul_experts_swiglu(encoding, c.lhs.to(DEV), c.gpu(0), c.gpu(1), c.routing, out_dtype=out), *silu_bound(g, gb, u, ub), out)


def summed(c, residual):
    y, b = c.products()
    here = ((c.ids >= 0) & (c.ids < len(c.w[0])))[..., None]
    w = torch.where(here, c.weights.double()[..., None], torch.zeros(1, dtype=torch.float64))
    terms = w * y
    size = terms.abs().sum(1)
    r = torch.zeros_like(size) if residual is None else residual.double()
    return r + terms.sum(1), (w * b).sum(1) + (c.top + 1) * R.U * (size + r.abs())


@pytest.mark.parametrize("encoding", GGUF, ids=lambda e: e.name)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("shape", SHAPES)
def test_weighted_sum(encoding, dtype, shape):
    c = Case(encoding, *shape, dtype, per_pair=True, without=0.2)
    for out, residual in ((torch.float32, None), (torch.bfloat16, torch.randn(c.tokens, c.n, generator=c.g).bfloat16()), (torch.float32, torch.randn(c.tokens, c.n, generator=c.g))):
        got = qmatmul_experts_sum(encoding, c.lhs.to(DEV), c.gpu(), c.routing, residual=None if residual is None else residual.to(DEV), out_dtype=out)
        check(got, *summed(c, residual), out)


@pytest.mark.parametrize("encoding", GGUF, ids=lambda e: e.name)
@pytest.mark.parametrize("tokens", (1, 3, 40, 200))
def test_pairs_without_an_expert_get_zeros(encoding, tokens):
    c = Case(encoding, tokens, 4, 3, 72, 512, torch.bfloat16, without=0.5)
    none = c.ids < 0
    out = qmatmul_experts(encoding, c.lhs.to(DEV), c.gpu(), c.routing)
    check(out, *c.products(), torch.float32)
    assert (out.cpu()[none] == 0).all()
    empty = group_experts(torch.full_like(c.ids, -1).to(DEV), c.weights.to(DEV), 4)
    assert (qmatmul_experts(encoding, c.lhs.to(DEV), c.gpu(), empty) == 0).all()
    assert (qmatmul_experts_swiglu(encoding, c.lhs.to(DEV), c.gpu(), c.gpu(), empty) == 0).all()
    residual = torch.randn(tokens, 72, device=DEV)
    weights = torch.full_like(c.weights, torch.nan).to(DEV)  # of pairs that do not count
    assert torch.equal(qmatmul_experts_sum(encoding, c.lhs.to(DEV), c.gpu(), group_experts(torch.full_like(c.ids, -1).to(DEV), weights, 4), residual=residual), residual)


@pytest.mark.parametrize("encoding", GGUF, ids=lambda e: e.name)
@pytest.mark.parametrize("tokens", (1, 7, 150))
def test_gate_and_up_of_one_tensor(encoding, tokens):
    c = Case(encoding, tokens, 6, 2, 160, 512, torch.bfloat16)  # 80 rows of gate, 80 of up
    both = c.gpu()
    got = qmatmul_experts_swiglu(encoding, c.lhs.to(DEV), both[:, :80], both[:, 80:], c.routing)
    y, b = c.products()
    check(got, *silu_bound(y[..., :80], b[..., :80], y[..., 80:], b[..., 80:]), torch.float32)


@pytest.mark.parametrize("encoding", GGUF, ids=lambda e: e.name)
@pytest.mark.parametrize("offset", (1, 2, 4, 8))
@pytest.mark.parametrize("tokens", (2, 90))
def test_weights_at_any_address(encoding, offset, tokens):
    c = Case(encoding, tokens, 3, 2, 56, 256, torch.bfloat16)  # (Q6_K: an odd number of blocks in all)
    room = torch.zeros(c.packed[0].numel() + 16, dtype=torch.uint8, device=DEV)
    room[offset:offset + c.packed[0].numel()] = c.gpu().reshape(-1)
    w = room[offset:offset + c.packed[0].numel()].view(c.packed[0].shape)
    check(qmatmul_experts(encoding, c.lhs.to(DEV), w, c.routing), *c.products(), torch.float32)


@pytest.mark.parametrize("k", (32, 96, 288, 2080))
@pytest.mark.parametrize("tokens", (1, 30, 140))
def test_q4_0_rows_of_any_number_of_blocks(k, tokens):
    c = Case(QE.Q4_0, tokens, 5, 2, 72, k, torch.float32, mats=2)
    check(qmatmul_experts(QE.Q4_0, c.lhs.to(DEV), c.gpu(), c.routing), *c.products(), torch.float32)
    check(qmatmul_experts_swiglu(QE.Q4_0, c.lhs.to(DEV), c.gpu(0), c.gpu(1), c.routing), *silu_bound(*c.products(0), *c.products(1)), torch.float32)


@pytest.mark.parametrize("n", (264, 280, 297, 376, 952))
def test_many_experts_with_a_few_rows_of_more_tiles_than_a_workgroup_takes(n):
    """128 experts (four different ones over and over) whose tiles do not go into the workgroups evenly."""
    c = Case(QE.Q4_K, 70, 4, 1, n, 2304, torch.bfloat16, mats=2)
    ids = R.choose(torch.randn(70, 128, generator=c.g), 4, "softmax", True)[0]
    routing = group_experts(ids.to(DEV), torch.ones(ids.shape, device=DEV), 128)
    gate, up = (c.gpu(i)[torch.arange(128, device=DEV) % 4] for i in (0, 1))
    products = [R.products(QE.Q4_K, c.lhs, w, ids % 4) for w in c.w]
    check(qmatmul_experts(QE.Q4_K, c.lhs.to(DEV), gate, routing), *products[0], torch.float32)
    check(qmatmul_experts_swiglu(QE.Q4_K, c.lhs.to(DEV), gate, up, routing), *silu_bound(*products[0], *products[1]), torch.float32)


@pytest.mark.parametrize("k", (32, 96, 256, 288, 2080))
@pytest.mark.parametrize("n, pad", ((71, 0), (71, 2), (72, 2), (33, 4)))
@pytest.mark.parametrize("tokens", (1, 30, 140, 300))
def test_q4_0_matrices_that_begin_between_multiples_of_four(k, n, pad, tokens):
    """Blocks are 18 bytes: an expert's matrix, after an odd number of blocks or at a distance of its own, begins two bytes behind a multiple of four."""
    c = Case(QE.Q4_0, tokens, 5, 2, n, k, torch.bfloat16)
    size = n * k // 32 * 18
    room = torch.full((5 * (size + pad),), 255, dtype=torch.uint8, device=DEV)
    w = room[: 5 * (size + pad)].as_strided((5, n, k // 32 * 18), (size + pad, k // 32 * 18, 1))
    w.copy_(c.gpu())
    check(qmatmul_experts(QE.Q4_0, c.lhs.to(DEV), w, c.routing), *c.products(), torch.float32)


@pytest.mark.parametrize("encoding", GGUF, ids=lambda e: e.name)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("tokens", (1, 4, 80))
def test_lhs_rows_of_very_different_sizes(encoding, dtype, tokens):
    c = Case(encoding, tokens, 4, 2, 48, 768, dtype)
    far = 3 if encoding == QE.Q4_0 else 30  # (a Q8_0 scale is an fp16 number)
    c.lhs = (c.lhs.float() * torch.logspace(-far, far, tokens)[:, None] if tokens > 1 else c.lhs.float() * 10.0 ** -far).to(dtype)
    c.lhs[-1] = 0
    # relative to each row's size the bound is the same; in a row of wide range small values are held against the largest (2^-34): inside it
    check(qmatmul_experts(encoding, c.lhs.to(DEV), c.gpu(), c.routing), *c.products(), torch.float32)


@pytest.mark.parametrize("encoding", (QE.Q4_K, QE.Q6_K, QE.Q4_0), ids=lambda e: e.name)
@pytest.mark.parametrize("tokens", (2, 100))
def test_rows_do_not_touch_each_other(encoding, tokens):
    """A row with NaN or infinities spoils its own results only."""
    c = Case(encoding, tokens, 3, 2, 64, 512, torch.float32)
    clean = qmatmul_experts(encoding, c.lhs.to(DEV), c.gpu(), c.routing)
    x = c.lhs.clone()
    x[0, 5] = torch.nan
    spoilt = qmatmul_experts(encoding, x.to(DEV), c.gpu(), c.routing)
    y, b = c.products()
    check(spoilt[1:], y[1:], b[1:], torch.float32)
    if encoding != QE.Q4_0:
        assert spoilt[0].isnan().all()
    check(clean, y, b, torch.float32)


@pytest.mark.parametrize("tokens", (1, 9, 260))
def test_routing_arrays_that_hold_anything(tokens):
    """Numbers that are no pairs or offsets: nothing is read or written out of range, and what is named right comes out right."""
    c = Case(QE.Q4_K, tokens, 4, 2, 64, 512, torch.bfloat16)
    pairs = tokens * 2
    y, b = c.products()
    order = c.routing.order.clone()
    order[0] = 2 ** 31 - 1
    order[-1] = -7
    kept = [p for p in order.tolist() if 0 <= p < pairs]
    got = qmatmul_experts(QE.Q4_K, c.lhs.to(DEV), c.gpu(), ExpertRouting(c.routing.experts, c.routing.weights, c.routing.offsets, order)).reshape(pairs, -1)
    if tokens > 1:
        check(got[kept], y.reshape(pairs, -1)[kept], b.reshape(pairs, -1)[kept], torch.float32)
    for offsets in ([-5, 10 ** 9, -3, 7, 2], [2 ** 31 - 1] * 5, [-(2 ** 31)] * 5):
        r = ExpertRouting(c.routing.experts, c.routing.weights, torch.tensor(offsets, dtype=torch.int32, device=DEV), c.routing.order)
        qmatmul_experts_sum(QE.Q4_K, c.lhs.to(DEV), c.gpu(), r)
    torch.cuda.synchronize()


@pytest.mark.parametrize("tokens", (1, 12, 300))
def test_a_captured_block_replays(tokens):
    """Router, gated pair and sum in one graph, replayed with other inputs and eager work in between."""
    c = Case(QE.Q4_K, tokens, 8, 2, 96, 512, torch.bfloat16, mats=2)
    down = R.pack(QE.Q6_K, (0.02 * torch.randn(8, 512, 256, generator=c.g)).numpy()).to(DEV)
    gate, up = (torch.cat([c.gpu(i)] * 3, 1)[:, :256].contiguous() for i in (0, 1))
    router = torch.randn(512, 8, generator=c.g).to(DEV)

    def block(x):
        routing = route_experts(x.float() @ router, 2)
        h = qmatmul_experts_swiglu(QE.Q4_K, x, gate, up, routing, out_dtype=torch.bfloat16)
        return qmatmul_experts_sum(QE.Q6_K, h, down, routing, residual=x, out_dtype=torch.bfloat16)

    x = c.lhs.to(DEV)
    block(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = block(x)
    torch.cuda.synchronize()
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=c.g))
        want = block(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_calls_on_another_stream_and_side_by_side():
    c = Case(QE.Q4_K, 40, 8, 2, 96, 1024, torch.bfloat16)
    w, lhs = c.gpu(), c.lhs.to(DEV)
    torch.cuda.synchronize()
    want = qmatmul_experts_sum(QE.Q4_K, lhs, w, c.routing)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                outs.append(qmatmul_experts_sum(QE.Q4_K, lhs, w, c.routing))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_results_repeat():
    c = Case(QE.Q6_K, 257, 8, 4, 120, 1024, torch.float32)
    a, b = (qmatmul_experts_sum(QE.Q6_K, c.lhs.to(DEV), c.gpu(), c.routing) for _ in range(2))
    assert torch.equal(a, b)


def test_a_block_end_to_end():
    """Router, gated pair, sum onto the residual, as a layer has them, against 64 bits (fp32 activations: what is handed on is not rounded to fewer bits)."""
    tokens, experts, hidden, ffn = 50, 16, 512, 256
    c = Case(QE.Q4_K, tokens, experts, 4, ffn, hidden, torch.float32, mats=2)
    down = R.pack(QE.Q6_K, (0.02 * torch.randn(experts, hidden, ffn, generator=c.g)).numpy())
    x, router = c.lhs.to(DEV), torch.randn(hidden, experts, generator=c.g)
    logits = c.lhs @ router
    routing = route_experts(logits.to(DEV), 4)
    h = qmatmul_experts_swiglu(QE.Q4_K, x, c.gpu(0), c.gpu(1), routing)
    out = qmatmul_experts_sum(QE.Q6_K, h, down.to(DEV), routing, residual=x)
    c.ids, weights = R.choose(logits, 4, "softmax", True)
    (g, gb), (u, ub) = c.products(0), c.products(1)
    h64, hb = silu_bound(g, gb, u, ub)
    wd = R.weights64(QE.Q6_K, down)
    y, yb = R.products(QE.Q6_K, h64, wd, c.ids)
    size = torch.stack([hb[c.ids == e].abs().sum(-1).max() * wd[e].abs().max() if (c.ids == e).any() else torch.tensor(0.0) for e in range(experts)]).max()
    want = c.lhs.double() + (weights[..., None] * y).sum(1)
    check(out, want, (weights[..., None] * yb).sum(1) + size + 2.0 ** 6 * R.U * (weights[..., None] * y).abs().sum(1) + 5 * R.U * want.abs(), torch.float32)


def drawn_shapes(count):
    """Sizes over the whole range of the kernels' rules: few and many experts, rows of an expert from less than one to hundreds, one tile of columns to hundreds, one block of K to sixteen."""
    rng = random.Random(20)
    for _ in range(count):
        experts = rng.choice((1, 2, 3, 5, 8, 16, 33, 60, 64, 100, 128, 160))
        top = min(experts, rng.choice((1, 1, 2, 4, 6, 8)))
        tokens = max(1, min(int(experts * math.exp(rng.uniform(math.log(0.3), math.log(300))) / top), 8000 // top))
        encoding = rng.choice(GGUF)
        k = 32 * rng.randrange(1, 90) if encoding == QE.Q4_0 and rng.random() < 0.5 else 256 * rng.choice((1, 1, 2, 2, 3, 4, 5, 7, 8, 9, 10, 11, 14, 16))
        n = int(math.exp(rng.uniform(rng.choice((0.0, 3.0, 4.5)), math.log(min(6000, 6.2e6 / (min(experts, 4) * k), 2.0e9 / (tokens * top * k) + 40)))))
        yield encoding, tokens, experts, top, n, k, rng.choice((torch.float32, torch.bfloat16)), rng.choice(("each", "each", "gated", "sum")), rng.random() < 0.3


@pytest.mark.parametrize("shape", drawn_shapes(150), ids=lambda s: "-".join(str(getattr(v, "name", v)).replace("torch.", "") for v in s))
def test_drawn_shapes(shape):
    """Weights: up to four different experts over and over."""
    encoding, tokens, experts, top, n, k, dtype, op, per_pair = shape
    c = Case(encoding, tokens, min(experts, 4), 1, n, k, dtype, per_pair=False, mats=2 if op == "gated" else 1)
    lhs = torch.randn(tokens, top, k, generator=c.g).to(dtype) if per_pair else c.lhs
    ids, weights = R.choose(torch.randn(tokens, experts, generator=c.g) + torch.randn(1, experts, generator=c.g), top, "softmax", True)
    ids[torch.rand(ids.shape, generator=c.g) < 0.05] = -1
    routing = group_experts(ids.to(DEV), weights.float().to(DEV), experts)
    w = [c.gpu(i)[torch.arange(experts, device=DEV) % c.w[0].shape[0]] for i in range(len(c.w))]
    products = [R.products(encoding, lhs, x, torch.where(ids < 0, ids, ids % x.shape[0])) for x in c.w]
    x = lhs.to(DEV)
    if op == "gated":
        check(qmatmul_experts_swiglu(encoding, x, w[0], w[1], routing), *silu_bound(*products[0], *products[1]), torch.float32)
    elif op == "each":
        check(qmatmul_experts(encoding, x, w[0], routing), *products[0], torch.float32)
    else:
        share = torch.where(ids < 0, torch.zeros_like(weights), weights).float().double()[..., None]
        terms, bounds = (share * t for t in products[0])
        check(qmatmul_experts_sum(encoding, x, w[0], routing), terms.sum(1), bounds.sum(1) + (top + 1) * R.U * terms.abs().sum(1), torch.float32)


def test_the_experts_of_a_gguf_file(tmp_path):
    """The 3-D tensors as the reader hands them out."""
    c = Case(QE.Q4_K, 20, 4, 2, 64, 512, torch.bfloat16, mats=2)
    path = write_gguf(tmp_path / "experts.gguf", [], [(name, [512, 64, 4], 12, p.numpy().tobytes()) for name, p in zip(("gate", "up"), c.packed)])
    file = GGUFWeights(path)
    gate, up = (file.tensor(name, DEV) for name in ("gate", "up"))
    assert gate.shape == c.packed[0].shape and file.encoding("gate") == QE.Q4_K
    check(qmatmul_experts_swiglu(file.encoding("gate"), c.lhs.to(DEV), gate, up, c.routing), *silu_bound(*c.products(0), *c.products(1)), torch.float32)


def test_refusals():
    c = Case(QE.Q4_K, 6, 4, 2, 64, 512, torch.bfloat16)
    x, w, r = c.lhs.to(DEV), c.gpu(), c.routing
    for call, error, match in (
        (lambda: qmatmul_experts(QE.GPTQ, x, w, r), TypeError, "GGUF"),
        (lambda: qmatmul_experts(QE.Q4_K, x.half(), w, r), TypeError, "float32 or bfloat16"),
        (lambda: qmatmul_experts(QE.Q4_K, x[:4], w, r), ValueError, "rows"),
        (lambda: qmatmul_experts(QE.Q4_K, x[:, :256].contiguous(), w, r), ValueError, "rows hold"),
        (lambda: qmatmul_experts(QE.Q4_K, x, w[:3], r), ValueError, "experts"),
        (lambda: qmatmul_experts(QE.Q4_K, x, w[0], r), TypeError, "uint8"),
        (lambda: qmatmul_experts(QE.Q4_K, x, w[:, ::2], r), ValueError, "contiguous"),
        (lambda: qmatmul_experts(QE.Q4_K, x, w, None), TypeError, "ExpertRouting"),
        (lambda: qmatmul_experts(QE.Q4_K, x, w, r, out_dtype=torch.float16), TypeError, "out_dtype"),
        (lambda: qmatmul_experts_swiglu(QE.Q4_K, x, w, w[:, :32], r), ValueError, "same shape"),
        (lambda: qmatmul_experts_sum(QE.Q4_K, x, w, r, residual=x), TypeError, "residual"),
        (lambda: qmatmul_experts(QE.Q4_K, x.cpu(), w, r), ValueError, "GPU"),
        (lambda: route_experts(torch.zeros(3, 8, device=DEV), 9), ValueError, "top_k"),
        (lambda: route_experts(torch.zeros(3, 8, device=DEV), 0), ValueError, "top_k"),
        (lambda: route_experts(torch.zeros(0, 8, device=DEV), 2), ValueError, "row"),
        (lambda: route_experts(torch.zeros(3, 1025, device=DEV), 2), ValueError, "experts"),
        (lambda: route_experts(torch.zeros(3, 8, device=DEV), 2, scoring="tanh"), ValueError, "scoring"),
        (lambda: route_experts(torch.zeros(3, 8, device=DEV), 2, bias=torch.zeros(7, device=DEV)), TypeError, "bias"),
        (lambda: group_experts(torch.zeros(3, 2, device=DEV), torch.zeros(3, 2, device=DEV), 4), TypeError, "int32"),
        (lambda: group_experts(torch.zeros(3, 2, dtype=torch.int32, device=DEV), torch.zeros(3, 2, device=DEV), 0), ValueError, "experts"),
        (lambda: ExpertRouting(r.experts, r.weights, r.offsets, r.order[:-1]), ValueError, "order"),
        (lambda: ExpertRouting(r.experts.long(), r.weights, r.offsets, r.order), TypeError, "int32"),
    ):
        with pytest.raises(error, match=match):
            call()
