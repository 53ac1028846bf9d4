"""Plain 64-bit restatement of the experts' products and of log probabilities (CPU), and what fp32 sums may be off by."""
import numpy as np
import torch

import np_formats as F
import oracle as O
from mojo_amd import QuantizationEncoding as QE

DEQUANT = {QE.Q4_0: F.dequant_q4_0, QE.Q4_K: F.dequant_q4_k, QE.Q5_K: F.dequant_q5_k, QE.Q6_K: F.dequant_q6_k}
ORACLE = {QE.Q4_0: O.Q4_0, QE.Q4_K: O.Q4_K, QE.Q5_K: O.Q5_K, QE.Q6_K: O.Q6_K}
U = 2.0 ** -24           # half a step of fp32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def pack(encoding, w):
    """fp32 [experts, n, k] -> packed uint8 [experts, n, bytes] (torch, CPU)"""
    e, n, k = w.shape
    return torch.from_numpy(O.quantize(ORACLE[encoding], np.ascontiguousarray(w.reshape(e * n, k)))).reshape(e, n, -1)


def weights64(encoding, packed):
    e, n, row = packed.shape
    bp = encoding.block_parameters
    k = row // bp.block_size * bp.elements_per_block
    return torch.from_numpy(DEQUANT[encoding](packed.reshape(e * n, row).contiguous().numpy(), k).astype(np.float64)).reshape(e, n, k)


def lhs64(encoding, x):
    """The lhs as the products take it: Q4_0 rounds it to Q8_0 (scale = largest times 1 / 127 in fp32, kept as fp16, codes with halves away from zero)."""
    x = x.float()
    if encoding != QE.Q4_0:
        return x.double()
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = b.abs().amax(-1, keepdim=True) * torch.tensor(np.float32(1) / np.float32(127))
    t = (b * torch.where(d != 0, 1.0 / d, torch.zeros_like(d))).double()
    codes = torch.sign(t) * torch.floor(t.abs() + 0.5)
    return (codes * d.half().double()).reshape(x.shape)


def products(encoding, lhs, w, ids):
    """(y [tokens, top, n], bound of its error) for ids [tokens, top]; zeros where there is no expert.

    Products are exact and their sums fp32: a sum of K terms is made of partial sums of at most A = sum |x| |w|, each rounded by u A at most, over chains of K / 16 steps and fewer whose roundings have
    either sign: 16 u A up to K = 4096.  A code and its minimum may each be twice as large as what they leave: A counts 2 max |w| of the row.  fp32 rows are held to 22 bits: 4 u A more.
    """
    x = lhs64(encoding, lhs)
    if x.dim() == 2:
        x = x[:, None].expand(-1, ids.shape[1], -1)
    y = torch.zeros((*ids.shape, w.shape[1]), dtype=torch.float64)
    bound = torch.zeros_like(y)
    for e in range(w.shape[0]):
        at = ids == e
        if at.any():
            y[at] = x[at] @ w[e].T
            bound[at] = 20 * U * x[at].abs().sum(-1, keepdim=True) * (2 * w[e].abs().amax(-1))
    return y, bound


def rounded(bound, value, dtype):
    """the error that rounding `value` once to `dtype` adds"""
    return bound + HALF[dtype] * (value.abs() + bound) + 1e-30


def sorted_pairs(ids, experts):
    flat = ids.reshape(-1).long()
    run = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    order = torch.sort(run, stable=True).indices
    offsets = torch.searchsorted(run.sort().values, torch.arange(experts + 1))
    return offsets.int(), order.int()


def choose(logits, top, scoring, renormalize, bias=None, scale=1.0):
    """(ids, weights) in 64 bits"""
    z = logits.double()
    score = torch.softmax(z, -1) if scoring == "softmax" else 1.0 / (1.0 + (-z).exp())
    by = z if bias is None else score + bias.double()
    ids = torch.sort(by, dim=-1, descending=True, stable=True).indices[:, :top]
    w = score.gather(1, ids)
    if renormalize:
        w = w / w.sum(-1, keepdim=True)
    return ids.int(), w * scale


def log_probabilities(logits, tokens, top):
    z = logits.double()
    z = z - z.amax(-1, keepdim=True)  # (beside 3e38 the logarithm of the sum has no digit left)
    logs = z - torch.logsumexp(z, -1, keepdim=True)
    p = logs.exp()
    entropy = -torch.where(p > 0, p * logs, torch.zeros_like(p)).sum(-1)
    ids = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :top]
    return logs.gather(1, tokens.reshape(len(z), -1).long()).reshape(tokens.shape), entropy, ids.int(), logs.gather(1, ids)
