"""The experts of a mixture-of-experts block on packed weights, and the log probabilities of what a model answers: one dict per case.

A case names an operator (``op``): the router (``route``), the experts' gated pair (``gate_up``), one product by expert (``expert``), the weighted
sum of the experts' results (``down``), log probabilities from logits (``score``) and from the hidden state through the packed vocabulary
(``head``).  ``run`` computes it from elementary torch operations in 32 bits, or, with ``own`` set, through the package's entry points.
"""
import math

import torch

own = False

BLOCK = {"Q4_0": (32, 18), "Q4_K": (256, 144), "Q5_K": (256, 176), "Q6_K": (256, 210)}  # weights and bytes of a block
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
MOST_FLOPS = 2 * 2000 * 8 * 2 * 1024 * 2048  # of the largest expert product listed
MOST_HEAD = 2 * 200 * 128256 * 4096
MOST_LOGITS = 1021 * 128256


def listed():
    return [
        # one token of a decode step chooses eight of 64 experts: latency
        {"name": "route_1", "op": "route", "tokens": 1, "experts": 64, "top": 8, "in": "f32", "scoring": "softmax", "renormalize": True},
        # a prompt, with scores of their own for each expert and a correction that balances the choice
        {"name": "route_4099", "op": "route", "tokens": 4099, "experts": 128, "top": 8, "in": "bf16", "scoring": "sigmoid", "renormalize": True},
        # gate and up of one token: the weights of eight experts
        {"name": "gate_up_q4k_1", "op": "gate_up", "enc": "Q4_K", "tokens": 1, "experts": 64, "top": 8, "n": 1024, "k": 2048, "in": "bf16", "out": "bf16"},
        # gate and up of a prompt: about 250 rows an expert, some with few
        {"name": "gate_up_q4k_2000", "op": "gate_up", "enc": "Q4_K", "tokens": 2000, "experts": 64, "top": 8, "n": 1024, "k": 2048, "in": "bf16", "out": "bf16"},
        # one projection of sixteen sequences decoded together, few large experts: most of the weights, few rows each
        {"name": "expert_q5k_16", "op": "expert", "enc": "Q5_K", "tokens": 16, "experts": 8, "top": 2, "n": 14336, "k": 4096, "in": "f32", "out": "f32"},
        # a batch that is no multiple of anything, four bits without minima, odd sizes
        {"name": "expert_q40_301", "op": "expert", "enc": "Q4_0", "tokens": 301, "experts": 16, "top": 4, "n": 1408, "k": 2080, "in": "bf16", "out": "f32"},
        # down and the weighted sum onto the residual, one token; mixed checkpoints store down in six bits
        {"name": "down_q6k_1", "op": "down", "enc": "Q6_K", "tokens": 1, "experts": 64, "top": 8, "n": 2048, "k": 1024, "in": "bf16", "out": "bf16", "residual": True},
        # the same of a chunk of a prompt, fp32 activations
        {"name": "down_q6k_500", "op": "down", "enc": "Q6_K", "tokens": 500, "experts": 64, "top": 8, "n": 2048, "k": 1024, "in": "f32", "out": "f32", "residual": True},
        # the answer's token, with twenty alternatives, from the logits of one sequence
        {"name": "score_1", "op": "score", "rows": 1, "vocab": 128256, "in": "f32", "top": 20},
        # a batch of bf16 logits in a padded buffer
        {"name": "score_1021", "op": "score", "rows": 1021, "vocab": 128256, "in": "bf16", "top": 5, "pad": 64},
        # the log probability of one token from its hidden state: the vocabulary's weights are read once
        {"name": "head_q6k_1", "op": "head", "enc": "Q6_K", "rows": 1, "vocab": 128256, "k": 4096, "in": "bf16"},
        # a text scored token by token
        {"name": "head_q6k_200", "op": "head", "enc": "Q6_K", "rows": 200, "vocab": 128256, "k": 4096, "in": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    op = rng.choices(("route", "gate_up", "expert", "down", "score", "head"), (12, 26, 20, 20, 14, 8))[0]
    c = {"op": op, "in": rng.choice(("f32", "bf16"))}
    if op == "score":
        c["vocab"] = _log(rng, 1000, 160000)
        c["rows"] = _log(rng, 1, min(4096, MOST_LOGITS // c["vocab"]))
        c["top"] = rng.choice((0, 1, 5, 20))
        c["pad"] = rng.choice((0, 0, 1, 64))
        return c
    if op == "head":
        c["enc"] = rng.choice(("Q4_K", "Q5_K", "Q6_K", "Q6_K"))
        c["vocab"], c["k"] = rng.choice(((32000, 4096), (128256, 4096), (151936, 2048), (50257, 1024)))
        c["rows"] = _log(rng, 1, min(512, MOST_HEAD // (2 * c["vocab"] * c["k"]) // (2 if c["in"] == "f32" else 1)))
        return c
    c["experts"] = rng.choice((8, 8, 16, 32, 60, 64, 64, 128, 256))
    c["top"] = rng.randint(1, min(8, c["experts"])) if c["experts"] > 8 else rng.randint(1, 2)
    if op == "route":
        c["tokens"] = _log(rng, 1, 8192)
        c["scoring"] = rng.choice(("softmax", "softmax", "sigmoid"))
        c["renormalize"] = rng.random() < 0.7
        return c
    c["enc"] = rng.choice(("Q4_K", "Q4_K", "Q4_0", "Q5_K", "Q6_K"))
    c["out"] = rng.choice(("f32", "bf16"))
    block = BLOCK[c["enc"]][0]
    c["k"] = block * max(1, _log(rng, 512, 7168) // block)
    mats = 2 if op == "gate_up" else 1
    most = (1 << 29) // (c["experts"] * c["k"] * mats)  # up to 512 Mi weights
    c["n"] = 8 * max(1, _log(rng, 512, max(512, min(14336, most))) // 8)
    flops = 2 * c["top"] * mats * c["n"] * c["k"] * (2 if c["in"] == "f32" else 1) * (2 if c["enc"] == "Q6_K" else 1)
    c["tokens"] = _log(rng, 1, max(1, min(2000, MOST_FLOPS // flops)))
    if op == "down":
        c["residual"] = rng.random() < 0.5
    return c


# ---------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------
def _half_bytes(x):
    """float16 bit patterns as bytes: [...] -> uint8 [..., 2]"""
    return x.to(torch.float16).contiguous().view(torch.uint8).reshape(*x.shape, 2)


def _scale_bytes(sc, mn):
    """6-bit scales and minima [..., 8] -> the 12 bytes that hold them"""
    a = sc[..., :4] | (sc[..., 4:] >> 4) << 6
    b = mn[..., :4] | (mn[..., 4:] >> 4) << 6
    c = (sc[..., 4:] & 15) | (mn[..., 4:] & 15) << 4
    return torch.cat((a, b, c), -1).to(torch.uint8)


def _pack(enc, w):
    """fp32 [rows, k] -> uint8 [rows, bytes]: each block fitted to its range"""
    rows, k = w.shape
    if enc == "Q4_0":
        b = w.view(rows, k // 32, 32)
        top = b.gather(-1, b.abs().argmax(-1, keepdim=True))
        d = (top / -8).to(torch.float16).float()
        q = torch.where(d == 0, 8.0, (b / d + 8.5).floor()).clamp(0, 15).to(torch.uint8)
        return torch.cat((_half_bytes(d[..., 0]), q[..., :16] | q[..., 16:] << 4), -1).view(rows, -1)
    if enc == "Q6_K":
        b = w.view(rows, k // 256, 16, 16)
        s = b.abs().amax(-1) / 31
        d = (s.amax(-1) / 127).to(torch.float16).float()
        sc = (s / d[..., None]).round().clamp(1, 127)
        q = (b / (d[..., None, None] * sc[..., None])).round().clamp(-32, 31).to(torch.int32) + 32
        q = q.view(rows, -1, 2, 4, 32)
        ql = torch.cat(((q[..., 0, :] & 15) | (q[..., 2, :] & 15) << 4, (q[..., 1, :] & 15) | (q[..., 3, :] & 15) << 4), -1)
        qh = (q[..., 0, :] >> 4) | (q[..., 1, :] >> 4) << 2 | (q[..., 2, :] >> 4) << 4 | (q[..., 3, :] >> 4) << 6
        parts = (ql.to(torch.uint8).flatten(2), qh.to(torch.uint8).flatten(2), sc.to(torch.int8).view(torch.uint8), _half_bytes(d))
        return torch.cat(parts, -1).view(rows, -1)
    most = 15 if enc == "Q4_K" else 31
    b = w.view(rows, k // 256, 8, 32)
    low = (-b.amin(-1)).clamp(min=0)
    s = (b.amax(-1) + low) / most
    d, dmin = (s.amax(-1) / 63).to(torch.float16).float(), (low.amax(-1) / 63).to(torch.float16).float()
    sc, mn = (s / d[..., None]).round().clamp(1, 63), (low / dmin[..., None]).round().clamp(0, 63)
    q = ((b + (dmin[..., None] * mn)[..., None]) / (d[..., None] * sc)[..., None]).round().clamp(0, most).to(torch.uint8)
    head = torch.cat((_half_bytes(d), _half_bytes(dmin), _scale_bytes(sc.to(torch.int32), mn.to(torch.int32))), -1)
    codes = ((q[..., 0::2, :] & 15) | (q[..., 1::2, :] & 15) << 4).flatten(2)
    if enc == "Q4_K":
        return torch.cat((head, codes), -1).view(rows, -1)
    fifth = torch.zeros_like(q[..., 0, :])
    for j in range(8):
        fifth |= (q[..., j, :] >> 4) << j
    return torch.cat((head, fifth, codes), -1).view(rows, -1)


def _weights(gen, enc, mats, n, k):
    """N(0, 0.02) weights packed matrix by matrix: uint8 [mats, n, bytes]"""
    per, size = BLOCK[enc]
    out = torch.empty((mats, n, k // per * size), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (n * k))
    rows = min(n, (1 << 27) // k)
    for i in range(0, mats, step):
        e = min(mats, i + step)
        for r in range(0, n, rows):
            t = min(n, r + rows)
            w = torch.empty(((e - i) * (t - r), k), device="cuda").normal_(0.0, 0.02, generator=gen)
            out[i:e, r:t] = _pack(enc, w).view(e - i, t - r, -1)
    return out


def _normal(gen, *shape):
    return torch.empty(shape, device="cuda").normal_(0.0, 1.0, generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], TYPES[case["in"]]
    s = {"case": case}
    if op == "score":
        width = case["vocab"] + case.get("pad", 0)
        s["logits"] = (3.0 * _normal(gen, case["rows"], width)).to(dtype)[:, :case["vocab"]]
        s["tokens"] = torch.randint(0, case["vocab"], (case["rows"],), device="cuda", generator=gen)
        return s
    if op == "head":
        s["weight"] = _weights(gen, case["enc"], 1, case["vocab"], case["k"])[0]
        s["lhs"] = _normal(gen, case["rows"], case["k"]).to(dtype)
        s["tokens"] = torch.randint(0, case["vocab"], (case["rows"],), device="cuda", generator=gen)
        return s
    tokens, experts, top = case["tokens"], case["experts"], case["top"]
    # what a router sees: some experts are asked for more than others
    logits = (1.5 * _normal(gen, tokens, experts) + 0.7 * _normal(gen, 1, experts)).to(dtype)
    if op == "route":
        s["logits"] = logits
        s["bias"] = 0.2 * _normal(gen, experts) if case["scoring"] == "sigmoid" else None
        return s
    # the router's answer: experts and weights of each token, and the pairs sorted by expert
    x = logits.float()
    s["experts"] = _order(x)[:, :top].to(torch.int32).contiguous()
    s["weights"] = torch.softmax(x.gather(1, s["experts"].long()), -1)
    s["offsets"], s["order"] = _sorted_pairs(s["experts"], experts)
    if op == "gate_up":
        s["gate"] = _weights(gen, case["enc"], experts, case["n"], case["k"])
        s["up"] = _weights(gen, case["enc"], experts, case["n"], case["k"])
    else:
        s["rhs"] = _weights(gen, case["enc"], experts, case["n"], case["k"])
    if op == "down":  # what a gated pair hands on, one row for each token and expert
        s["lhs"] = (torch.sigmoid(g := _normal(gen, tokens, top, case["k"])) * g * _normal(gen, tokens, top, case["k"])).to(dtype)
        s["residual"] = _normal(gen, tokens, case["n"]).to(TYPES[case["out"]]) if case["residual"] else None
    else:
        s["lhs"] = _normal(gen, tokens, case["k"]).to(dtype)
    return s


# ---------------------------------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------------------------------
def _order(x):
    """indices of the last axis by falling value, equal ones by rising index"""
    return torch.sort(x, dim=-1, descending=True, stable=True).indices


def _sorted_pairs(ids, experts):
    flat = ids.reshape(-1).long()
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = torch.bincount(flat, minlength=experts).cumsum(0)
    return offsets, torch.sort(flat, stable=True).indices.to(torch.int32)


def _halves(b):
    return b.contiguous().view(torch.float16).float()


def _six_bits(s):
    s = s.int()
    sc = torch.cat((s[..., 0:4] & 63, (s[..., 8:12] & 15) | s[..., 0:4] >> 6 << 4), -1)
    mn = torch.cat((s[..., 4:8] & 63, s[..., 8:12] >> 4 | s[..., 4:8] >> 6 << 4), -1)
    return sc.float(), mn.float()


def _unpack(enc, packed):
    """uint8 [n, bytes] -> fp32 [n, k]"""
    n = packed.shape[0]
    b = packed.view(n, -1, BLOCK[enc][1])
    if enc == "Q4_0":
        q = torch.cat((b[..., 2:] & 15, b[..., 2:] >> 4), -1).float() - 8.0
        return (q * _halves(b[..., :2])).reshape(n, -1)
    if enc == "Q6_K":
        ql, qh = b[..., :128].reshape(n, -1, 2, 64).int(), b[..., 128:192].reshape(n, -1, 2, 32).int()
        low = torch.stack((ql[..., :32] & 15, ql[..., 32:] & 15, ql[..., :32] >> 4, ql[..., 32:] >> 4), -2)
        high = torch.stack((qh & 3, qh >> 2 & 3, qh >> 4 & 3, qh >> 6), -2)
        q = ((low | high << 4) - 32).reshape(n, -1, 16, 16).float()
        sc = b[..., 192:208].contiguous().view(torch.int8).float() * _halves(b[..., 208:210])
        return (q * sc[..., None]).reshape(n, -1)
    d, dmin = _halves(b[..., 0:2]), _halves(b[..., 2:4])
    sc, mn = _six_bits(b[..., 4:16])
    codes = b[..., -128:].reshape(n, -1, 4, 1, 32)
    q = torch.cat((codes & 15, codes >> 4), -2).reshape(n, -1, 8, 32)
    if enc == "Q5_K":
        q = q | torch.stack([(b[..., 16:48] >> j & 1) << 4 for j in range(8)], -2)
    return (q.float() * (d * sc)[..., None] - (dmin * mn)[..., None]).reshape(n, -1)


def _activations(enc, x):
    """the lhs as the product takes it: Q4_0 rounds it to Q8_0 blocks (fp16 scale, codes with halves away from zero), the others keep it"""
    x = x.float()
    if enc != "Q4_0":
        return x
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = b.abs().amax(-1, keepdim=True) / 127.0
    t = (b * torch.where(d != 0, 1.0 / d, 0.0)).double()
    q = torch.sign(t) * (t.abs() + 0.5).floor()
    return (q.float() * d.to(torch.float16).float()).reshape(x.shape)


def _by_expert(s, rhs, lhs):
    """fp32 [tokens, top, n]: the rows of each expert times its weights"""
    case = s["case"]
    tokens, top = case["tokens"], case["top"]
    x = _activations(case["enc"], lhs)
    out = torch.zeros((tokens * top, case["n"]), device=x.device)
    ends = s["offsets"].tolist()
    for e in range(case["experts"]):
        pairs = s["order"][ends[e]:ends[e + 1]].long()
        if len(pairs):
            rows = x[pairs // top] if x.dim() == 2 else x.reshape(tokens * top, -1)[pairs]
            out[pairs] = rows @ _unpack(case["enc"], rhs[e]).t()
    return out.view(tokens, top, -1)


def _log_probabilities(x, tokens, top):
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1)
    log_total = total.log()
    chosen = (x.gather(1, tokens[:, None]) - m)[:, 0] - log_total
    entropy = log_total - (e * (x - m)).sum(-1) / total
    if top == 0:
        return [chosen, entropy]
    ids = _order(x)[:, :top] if x.shape[0] == 1 else torch.cat([_order(part)[:, :top] for part in x.split(64)])
    return [chosen, entropy, ids.to(torch.int32), x.gather(1, ids) - m - log_total[:, None]]


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "route":
        x = s["logits"].float()
        score = torch.softmax(x, -1) if case["scoring"] == "softmax" else torch.sigmoid(x)
        # (the order is that of the logits; with a correction that of the corrected scores, near each other, in 64 bits)
        ids = _order(x if s["bias"] is None else torch.sigmoid(x.double()) + s["bias"].double())[:, :case["top"]]
        weights = score.gather(1, ids)
        if case["renormalize"]:
            weights = weights / weights.sum(-1, keepdim=True)
        ids = ids.to(torch.int32)
        return [ids, weights, *_sorted_pairs(ids, case["experts"])]
    if op == "score":
        return _log_probabilities(s["logits"].float(), s["tokens"], case["top"])
    if op == "head":
        return _log_probabilities(s["lhs"].float() @ _unpack(case["enc"], s["weight"]).t(), s["tokens"], 0)
    out = TYPES[case["out"]]
    if op == "gate_up":
        g = _by_expert(s, s["gate"], s["lhs"])
        return (g * torch.sigmoid(g) * _by_expert(s, s["up"], s["lhs"])).to(out)
    y = _by_expert(s, s["rhs"], s["lhs"])
    if op == "expert":
        return y.to(out)
    y = (y * s["weights"][..., None]).sum(1)
    return (y if s["residual"] is None else y + s["residual"].float()).to(out)


def run(state):
    if not own:
        return _plain(state)
    import mojo_amd as M

    case, s = state["case"], state
    op = case["op"]
    if op == "route":
        r = M.route_experts(s["logits"], case["top"], scoring=case["scoring"], bias=s["bias"], renormalize=case["renormalize"])
        return [r.experts, r.weights, r.offsets, r.order]
    if op in ("score", "head"):
        if op == "score":
            p = M.logprobs(s["logits"], s["tokens"], top_k=case["top"])
        else:
            p = M.qmatmul_logprobs(M.QuantizationEncoding[case["enc"]], None, s["lhs"], s["weight"], tokens=s["tokens"])
        return [p.logprobs, p.entropy] + ([p.top_ids, p.top_logprobs] if case.get("top") else [])
    enc, out = M.QuantizationEncoding[case["enc"]], TYPES[case["out"]]
    routing = M.ExpertRouting(s["experts"], s["weights"], s["offsets"], s["order"])
    if op == "gate_up":
        return M.qmatmul_experts_swiglu(enc, s["lhs"], s["gate"], s["up"], routing, out_dtype=out)
    if op == "expert":
        return M.qmatmul_experts(enc, s["lhs"], s["rhs"], routing, out_dtype=out)
    return M.qmatmul_experts_sum(enc, s["lhs"], s["rhs"], routing, residual=s["residual"], out_dtype=out)


# ---------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------------
def work(case):
    op, el = case["op"], SIZE[case["in"]]
    if op == "score":
        return {"bytes": case["rows"] * (el * case["vocab"] + 16 + 8 * case["top"]), "flops": 4 * case["rows"] * case["vocab"]}
    if op == "head":
        per, size = BLOCK[case["enc"]]
        return {"bytes": case["vocab"] * case["k"] // per * size + case["rows"] * (el * case["k"] + 16), "flops": 2 * case["rows"] * case["vocab"] * case["k"]}
    tokens, experts, top = case["tokens"], case["experts"], case["top"]
    pairs = tokens * top
    if op == "route":
        return {"bytes": tokens * experts * el + 12 * pairs + 4 * experts, "flops": 4 * tokens * experts}
    per, size = BLOCK[case["enc"]]
    mats = 2 if op == "gate_up" else 1
    asked = experts * (1.0 - (1.0 - top / experts) ** tokens)  # experts that get a row, if none is preferred
    rows_in = pairs if op == "down" else tokens
    rows_out = tokens if op == "down" else pairs
    moved = asked * mats * case["n"] * case["k"] / per * size + el * rows_in * case["k"] + SIZE[case["out"]] * rows_out * case["n"] * (2 if case.get("residual") else 1)
    return {"bytes": int(moved + 12 * pairs), "flops": 2 * pairs * mats * case["n"] * case["k"]}


# ---------------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------
def _weight64(enc, packed):
    """float64 [n, k], value by value from the block layouts"""
    per, size = BLOCK[enc]
    n, k = packed.shape[0], packed.shape[1] // size * per
    blocks = packed.view(n, k // per, size)
    i = torch.arange(per, device=packed.device)

    def byte(at):
        return blocks[:, :, at].to(torch.int64)

    def half(at):
        return blocks[:, :, at:at + 2].contiguous().view(torch.float16).double()

    if enc == "Q4_0":
        code = byte(2 + i % 16) >> 4 * (i // 16) & 15
        return (half(0) * (code - 8).double()).reshape(n, k)
    if enc == "Q6_K":
        h, quarter, at = i // 128, i % 128 // 32, i % 32
        low = byte(64 * h + 32 * (quarter % 2) + at) >> 4 * (quarter // 2) & 15
        high = byte(128 + 32 * h + at) >> 2 * quarter & 3
        scale = byte(192 + i // 16)
        scale = scale - 256 * (scale > 127)
        return (half(208) * (scale * (low + 16 * high - 32)).double()).reshape(n, k)
    j = i // 32
    late = j >= 4
    sc = torch.where(late, byte(8 + j % 4 + 4) & 15 | byte(4 + j % 4) >> 6 << 4, byte(4 + j % 4) & 63)
    mn = torch.where(late, byte(8 + j % 4 + 4) >> 4 | byte(8 + j % 4) >> 6 << 4, byte(8 + j % 4) & 63)
    code = byte(size - 128 + 32 * (i // 64) + i % 32) >> 4 * (j % 2) & 15
    if enc == "Q5_K":
        code = code + 16 * (byte(16 + i % 32) >> j & 1)
    return (half(0) * (sc * code).double() - half(2) * mn.double()).reshape(n, k)


def _rows64(enc, x):
    if enc != "Q4_0":
        return x.double()
    # Q8_0 is defined by roundings to 32 and 16 bits: scale = largest / 127, code = value times its reciprocal, halves away from zero
    blocks = x.float().unflatten(-1, (-1, 32))
    scale = blocks.abs().max(-1, keepdim=True).values / 127.0
    inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    value = (blocks * inverse).double()
    code = torch.where(value < 0, (value - 0.5).ceil(), (value + 0.5).floor())
    return (code * scale.to(torch.float16).double()).flatten(-2)


def _experts64(s, rhs):
    case = s["case"]
    x = _rows64(case["enc"], s["lhs"])
    if x.dim() == 2:
        x = x[:, None].expand(-1, case["top"], -1)
    out = torch.zeros((case["tokens"], case["top"], case["n"]), dtype=torch.float64, device=x.device)
    for e in s["experts"].unique().tolist():
        chosen = s["experts"] == e
        w = _weight64(case["enc"], rhs[e])
        out[chosen] = x[chosen] @ w.t()
    return out


def _log64(z, tokens, top):
    total = torch.logsumexp(z, -1, keepdim=True)
    logs = z - total
    p = logs.exp()
    result = [logs.gather(1, tokens[:, None])[:, 0], -(p * logs).sum(-1)]
    if top:
        ids = torch.stack([torch.argsort(row, descending=True, stable=True)[:top] for row in z])
        result += [ids.to(torch.int32), logs.gather(1, ids)]
    return result


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "score":
        parts = [_log64(z.double(), t, case["top"]) for z, t in zip(s["logits"].split(64), s["tokens"].split(64))]
        return [torch.cat(p) for p in zip(*parts)]
    if op == "head":
        # (the vocabulary in parts: 64-bit weights are eight times the packed ones)
        logits = torch.cat([s["lhs"].double() @ _weight64(case["enc"], w).t() for w in s["weight"].split(8192)], 1)
        return _log64(logits, s["tokens"], 0)
    if op == "route":
        z = s["logits"].double()
        score = torch.softmax(z, -1) if case["scoring"] == "softmax" else 1.0 / (1.0 + (-z).exp())
        by = z if s["bias"] is None else score + s["bias"].double()
        ids = torch.argsort(by, dim=-1, descending=True, stable=True)[:, :case["top"]]
        weights = score.gather(1, ids)
        if case["renormalize"]:
            weights = weights / weights.sum(-1, keepdim=True)
        flat = ids.reshape(-1)
        offsets = torch.searchsorted(flat.sort().values, torch.arange(case["experts"] + 1, device=flat.device))
        return [ids.to(torch.int32), weights, offsets.to(torch.int32), torch.argsort(flat, stable=True).to(torch.int32)]
    if op == "gate_up":
        g = _experts64(s, s["gate"])
        return g / (1.0 + (-g).exp()) * _experts64(s, s["up"])
    y = _experts64(s, s["rhs"])
    if op == "expert":
        return y
    y = (s["weights"].double()[..., None] * y).sum(1)
    return y if s["residual"] is None else y + s["residual"].double()
