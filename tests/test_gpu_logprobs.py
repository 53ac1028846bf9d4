"""Log probabilities, entropy and alternatives against 64 bits."""
import pytest
import torch

import experts_reference as R
from mojo_amd import QuantizationEncoding as QE, logprobs, qmatmul, qmatmul_logprobs, quantize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def check(got, logits, tokens, top):
    """x - m is rounded by u |x - m|; exp, log and the sums of a wavefront's steps, lanes and parts (values of one sign) by some u of the logarithm and of the entropy's terms: 2^6 u of
    1 + |x - m| + log S (+ the mean of |x - m|, which the entropy is made of).  An exponential that is below 2^-126 beside the rounding of m log2 e, up to 2^-24 |m|, may come out as 0: `vocab` of
    them, times exponents up to 128 in the entropy."""
    want = R.log_probabilities(logits, tokens, top)
    z = logits.double()
    spread = (z.amax(-1) - torch.logsumexp(z, -1)).abs()
    for g, w, size in ((got.logprobs, want[0], want[0].abs()), (got.entropy, want[1], want[1].abs() + spread), *(((got.top_logprobs, want[3], want[3].abs()),) if top else ())):
        g = g.cpu().double()
        assert g.shape == w.shape
        least = 128 * z.shape[-1] * 2.0 ** (-126 + z.amax(-1).abs().clamp(max=2.0 ** 30) * 2.0 ** -24)
        limit = 2.0 ** 6 * R.U * size + least.reshape(-1, *[1] * (size.dim() - 1))
        error = torch.where(g == w, 0.0, (g - w).abs())  # (-inf has to be -inf)
        assert (error <= limit).all(), f"{(error / limit).max():.3g} of the bound"
    if top:
        assert torch.equal(got.top_ids.cpu(), want[2])


SHAPES = ((1, 1), (1, 7), (3, 64), (2, 1000), (5, 4097), (700, 33), (1, 32000), (3, 50257), (2, 128256), (130, 8200), (1, 300001), (1, 2 ** 22))


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("top", (0, 1, 5, 20, 64))
def test_logprobs(rows, vocab, top, dtype):
    top = min(top, vocab)
    g = torch.Generator().manual_seed(rows + vocab)
    x = (3.0 * torch.randn(rows, vocab, generator=g)).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    check(logprobs(x.to(DEV), tokens.to(DEV), top), x, tokens, top)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("skip", (0, 1, 2, 3, 5))
def test_rows_of_padded_logits_at_any_address(dtype, skip):
    g = torch.Generator().manual_seed(skip)
    wide = torch.randn(7, 9003, generator=g).to(dtype)
    wide[:, :skip] = 100.0  # not of the row
    wide[:, skip + 8990:] = 100.0
    x = wide[:, skip:skip + 8990]
    tokens = torch.randint(0, 8990, (7,), generator=g)
    check(logprobs(wide.to(DEV)[:, skip:skip + 8990], tokens.to(DEV, torch.int32), 20), x, tokens, 20)


@pytest.mark.parametrize("vocab", (100, 20000, 150000))
@pytest.mark.parametrize("order", ("rising", "falling", "equal", "two", "late", "steps"))
def test_alternatives_do_not_depend_on_where_they_lie(vocab, order):
    i = torch.arange(vocab, dtype=torch.float32)
    x = {"rising": i / vocab, "falling": -i / vocab, "equal": torch.full((vocab,), 2.5), "two": (i == vocab - 1).float() + (i == 3).float(), "late": torch.where(i >= vocab - 30, i / vocab, -3 - i / vocab),
         "steps": torch.floor(i / 7) % 5}[order].expand(2, -1).contiguous()
    tokens = torch.tensor([0, vocab - 1])
    for dtype in (torch.float32, torch.bfloat16):
        check(logprobs(x.to(dtype).to(DEV), tokens.to(DEV), 40), x.to(dtype), tokens, 40)


@pytest.mark.parametrize("rows, vocab", ((2, 9000), (2, 150000), (1100, 9000)))
@pytest.mark.parametrize("order", ("rising", "falling", "equal", "late", "steps", "mask", "few", "clusters"))
@pytest.mark.parametrize("top", (1, 20, 32))
def test_a_few_alternatives_do_not_depend_on_where_they_lie(rows, vocab, order, top):
    """One workgroup a row and many; values of which more than there is room for are equal, masked, or next to each other."""
    i = torch.arange(vocab, dtype=torch.float32)
    x = {"rising": i / vocab, "falling": -i / vocab, "equal": torch.full((vocab,), 2.5), "late": torch.where(i >= vocab - 30, i / vocab, -3 - i / vocab), "steps": torch.floor(i / 7) % 5,
         "mask": torch.where(i % 700 == 3, i / vocab, -torch.inf), "few": torch.where(i < 9, -i, -torch.inf), "clusters": torch.where(i % 2000 < 40, 1 + i / vocab, -i / vocab)}[order]
    x = x.expand(3, -1).contiguous()
    tokens = torch.tensor([0, vocab - 1, 3])
    for dtype in (torch.float32, torch.bfloat16):
        got = logprobs(x.to(dtype).to(DEV).repeat(rows // 2, 1)[:rows], tokens.to(DEV).repeat(rows // 2)[:rows], top)
        last = (rows - 1) // 3 * 3 if rows > 3 else 0
        n = min(3, rows - last)
        check(type(got)(*(t[last:last + n] for t in got)), x[:n].to(dtype), tokens[:n], top)
        assert rows == 2 or all(torch.equal(t[:999].reshape(333, 3, -1), t[:3].reshape(1, 3, -1).expand(333, -1, -1)) for t in got)


def test_more_rows_than_a_launch_takes():
    rows = 2 ** 22 + 5
    x = torch.randn(rows, 3, generator=torch.Generator().manual_seed(9))
    tokens = torch.arange(rows) % 3
    check(logprobs(x.to(DEV), tokens.to(DEV), 1), x, tokens, 1)


def test_nearly_certain_rows_keep_their_digits():
    x = torch.full((4, 70000), -30.0)
    for r, top in enumerate((0.0, 10.0, 60.0, 300.0)):
        x[r, 69 + 11000 * r] = top
    tokens = torch.tensor([69 + 11000 * r for r in range(4)])
    got = logprobs(x.to(DEV), tokens.to(DEV), 3)
    want = R.log_probabilities(x, tokens, 3)
    z = x.double() - x.double().amax(-1, keepdim=True)
    rest = torch.where(z < 0, z.exp(), 0.0).sum(-1)
    # -log p = log1p(rest), H = log1p(rest) + sum rest |z|: of one sign, so 2^6 u of themselves and u |z| of each exponential.  An exponential below the least normal
    # number, 2^-126, may come out as 0: 70000 of them leave out up to 70000 2^-126 = 8.2e-34, times |z| < 331 of the entropy.
    least = 70000 * 2.0 ** -126
    exact = -torch.log1p(rest)
    assert ((got.logprobs.cpu().double() - exact).abs() <= 2.0 ** 8 * R.U * exact.abs() + least).all()
    entropy = torch.log1p(rest) + (z.abs() * z.exp()).sum(-1) / (1 + rest)
    assert ((got.entropy.cpu().double() - entropy).abs() <= 2.0 ** 8 * R.U * entropy + 331 * least).all()
    assert torch.equal(got.top_ids.cpu(), want[2])


def test_masked_infinite_and_nan_rows():
    vocab = 5000
    x = torch.randn(7, vocab)
    x[0, 100:] = -torch.inf
    x[1] = -torch.inf
    x[2, 17] = torch.inf
    x[3, 4000] = torch.nan
    x[4] = torch.finfo(torch.float32).min
    x[5] = torch.nan
    tokens = torch.tensor([50, 3, 5, 7, 9, 11, 13])
    got = logprobs(x.to(DEV), tokens.to(DEV), 5)
    lp, h, ids, values = (t.cpu() for t in got)
    rows = [0, 4, 6]
    want = R.log_probabilities(x[rows], tokens[rows], 5)
    assert (lp[rows].double() - want[0]).abs().max() < 1e-5 and (h[rows].double() - want[1]).abs().max() < 1e-5 and torch.equal(ids[rows], want[2])
    masked = logprobs(x[:1].to(DEV), torch.tensor([200], device=DEV))
    assert masked.logprobs.item() == -torch.inf
    assert lp[1] == -torch.inf and h[1] == 0 and ids[1].tolist() == [0, 1, 2, 3, 4] and (values[1] == -torch.inf).all()
    assert lp[2].isnan() and h[2].isnan() and ids[2, 0] == 17
    assert lp[3].isnan() and h[3].isnan() and 4000 not in ids[3]
    assert lp[5].isnan() and h[5].isnan() and ids[5].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_a_nan_that_signals_hides_nobody(dtype):
    bits = {torch.float32: (torch.int32, 0x7f800001), torch.bfloat16: (torch.int16, 0x7f81)}[dtype]
    x = torch.randn(2, 9000, generator=torch.Generator().manual_seed(4)).to(dtype)
    want = torch.sort(x[1].float(), descending=True, stable=True).indices[:20]
    raw = x.view(bits[0])
    for i in want[:8].tolist():  # beside the largest
        raw[1, i ^ 1] = bits[1]
    keep = [i for i in torch.sort(torch.where(x[1].isnan(), -torch.inf, x[1].float()), descending=True, stable=True).indices[:20].tolist()]
    got = logprobs(x.to(DEV), torch.tensor([0, 0], device=DEV), 20)
    assert got.logprobs[1].isnan() and not got.logprobs[0].isnan() and got.top_ids[1].tolist() == keep


@pytest.mark.parametrize("low,high", ((-1.7e38, 1.7e38), (-3.4e38, 5.0), (-2.0, 3.0e38), (-3.4e38, -3.3e38), (1.0e37, 2.0e37), (2.0 ** 30 - 64, 2.0 ** 30), (2.0 ** 24 - 3, 2.0 ** 24 + 2), (-(2.0 ** 27) - 16, -(2.0 ** 27)), (1000.0, 1002.5)))
def test_values_at_the_ends_of_the_range(low, high):
    x = torch.full((3, 20000), low)
    x[0, 7] = x[1, 19999] = x[2, 0] = x[2, 9999] = high
    tokens = torch.tensor([7, 19999, 9999])
    check(logprobs(x.to(DEV), tokens.to(DEV), 2), x, tokens, 2)


def test_masked_everywhere_but_one_and_alternatives_beyond_the_mask():
    x = torch.full((2, 40000), -torch.inf)
    x[0, 39999] = -3.0
    x[1, 5] = x[1, 6] = 1.0
    got = logprobs(x.to(DEV), torch.tensor([39999, 6], device=DEV), 4)
    assert got.logprobs.tolist() == pytest.approx([0.0, -0.6931472], abs=1e-6) and got.entropy.tolist() == pytest.approx([0.0, 0.6931472], abs=1e-6)
    assert got.top_ids.tolist() == [[39999, 0, 1, 2], [5, 6, 0, 1]]
    assert got.top_logprobs[0, 1:].tolist() == [-torch.inf] * 3


def test_several_tokens_a_row_padding_and_unknown_tokens():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 6, 999, generator=g)
    tokens = torch.randint(0, 999, (4, 6, 5), generator=g)
    got = logprobs(x.to(DEV), tokens.to(DEV), 2)
    assert got.logprobs.shape == (4, 6, 5) and got.entropy.shape == (4, 6) and got.top_ids.shape == (4, 6, 2)
    want = R.log_probabilities(x.reshape(24, 999), tokens.reshape(24, 5), 2)
    assert (got.logprobs.cpu().reshape(24, 5).double() - want[0]).abs().max() < 2.0 ** 6 * R.U * want[0].abs().max()
    odd = torch.tensor([-1, -100, 999, 2 ** 31])
    got = logprobs(x[0, :4].contiguous().to(DEV), odd.to(DEV)).logprobs.cpu()
    assert got[:2].tolist() == [0.0, 0.0] and got[2:].isnan().all()


@pytest.mark.parametrize("rows", (1, 3, 40))
@pytest.mark.parametrize("encoding", (QE.Q6_K, QE.Q4_K, QE.Q4_0), ids=lambda e: e.name)
def test_through_the_packed_vocabulary(rows, encoding):
    g = torch.Generator().manual_seed(rows)
    w = quantize(encoding, (0.02 * torch.randn(5000, 512, generator=g)).to(DEV))
    x = torch.randn(rows, 512, generator=g).to(DEV)
    tokens = torch.randint(0, 5000, (rows,), generator=g).to(DEV)
    got, want = qmatmul_logprobs(encoding, None, x, w, tokens=tokens, top_k=7), logprobs(qmatmul(encoding, None, x, w), tokens, 7)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_more_rows_than_the_workspace_holds_at_once():
    """2^28 logits at a time: 4300 rows of 65536 are more."""
    g = torch.Generator().manual_seed(1)
    w = quantize(QE.Q4_K, (0.02 * torch.randn(65536, 256, generator=g)).to(DEV))
    x = torch.randn(4300, 256, generator=g).to(DEV, torch.bfloat16)
    tokens = torch.randint(0, 65536, (4300,), generator=g).to(DEV)
    got = qmatmul_logprobs(QE.Q4_K, None, x, w, tokens=tokens, top_k=3)
    rows = torch.tensor([0, 1, 4095, 4096, 4097, 4299], device=DEV)
    want = logprobs(qmatmul(QE.Q4_K, None, x[rows].contiguous(), w), tokens[rows], 3)
    # (another number of rows goes through another kernel: both are within 2^-18 of the logits' size)
    assert (got.logprobs[rows] - want.logprobs).abs().max() < 1e-4 and (got.entropy[rows] - want.entropy).abs().max() < 1e-4
    assert (got.top_logprobs[rows] - want.top_logprobs).abs().max() < 1e-4


def test_capture_and_replay():
    x = torch.randn(3, 40000, device=DEV)
    tokens = torch.tensor([1, 2, 3], device=DEV)
    logprobs(x, tokens, 5)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        logprobs(x, tokens, 5)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = logprobs(x, tokens, 5)
    torch.cuda.synchronize()
    for i in range(4):
        x.normal_()
        want = logprobs(x, tokens, 5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_logprobs_refusals():
    x, t = torch.randn(3, 50, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for call, error in (
        (lambda: logprobs(x.half(), t), TypeError), (lambda: logprobs(x, t.float()), TypeError), (lambda: logprobs(x, t[:2]), ValueError), (lambda: logprobs(x, t, 51), ValueError),
        (lambda: logprobs(x, t, -1), ValueError), (lambda: logprobs(x.cpu(), t), ValueError), (lambda: logprobs(x, t.cpu()), ValueError), (lambda: logprobs(x[:0], t[:0]), ValueError),
        (lambda: logprobs(x.t().contiguous().t(), t), ValueError), (lambda: logprobs(torch.zeros(2, 200, device=DEV), t[:2], 65), ValueError),
        (lambda: qmatmul_logprobs(QE.Q8_0, None, x, x, tokens=t), ValueError),
    ):
        with pytest.raises(error):
            call()
