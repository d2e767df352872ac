"""The timed cases of further operators beside the search: 4-bit rows, norms that end in 8 bits, log probabilities.

Four operators.  "quantize4" makes 4-bit rows (e2m1 codes, a power of two for each block of 32 coordinates) and reads
them back; "matmul4" scores 4-bit queries against all 4-bit rows; "norm" adds a residual, takes the root-mean-square norm
and makes the result 8-bit; "log_probs" gives the log probabilities of given slots under a softmax of scores, its
entropy and the best alternatives, and in training the gradient.

Sizes are those of this repository's benchmark and tests (100K, 400K, 1M and 10M rows, 1536 dimensions, batches of 1024) or
generic; `draw` spreads over the same ranges.
"""
import math

import torch

own = False

_BLOCK4 = 32                                  # coordinates that share a scale in 4-bit rows
_BLOCK8 = 128                                 # and in 8-bit ones
_TOP8 = 448.0                                 # the largest e4m3 value
_EPS = 1e-6
_MOST_ELEMENTS = 400_000 * 1536               # of rows to make 4-bit
_MOST_PRODUCTS = 1024 * 100_000 * 1536        # of a product
_MOST_OUTPUTS = 1024 * 100_000
_MOST_STORED = 1_000_000 * 1536
_MOST_NORMED = 16_384 * 4096
_MOST_SCORES = 2048 * 100_000
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # A middle-sized batch of queries made 4-bit before each product: all latency.
        dict(name="quantize4_64", op="quantize4", rows=64, dim=1536, dtype="f32"),
        # Rows of a shard as a model produced them, made 4-bit as they are added.
        dict(name="quantize4_400k", op="quantize4", rows=400_000, dim=1536, dtype="f32"),
        # One query against every row of a large collection: one pass over the rows.
        dict(name="score4_one_1m", op="matmul4", m=1, n=1_000_000, dim=1536, out="f32"),
        # Odd everything: a batch off every tile edge, rows that end inside a block.
        dict(name="score4_ragged", op="matmul4", m=37, n=77_777, dim=1000, out="f32"),
        # A batch against a collection, every score wanted.
        dict(name="score4_batch_100k", op="matmul4", m=1024, n=100_000, dim=1536, out="f32"),
        # A projection of many rows in front of the index.
        dict(name="project4_4096", op="matmul4", m=4096, n=4096, dim=4096, out="bf16"),
        # One token's hidden state at the end of a layer, made 8-bit for the product behind: all latency.
        dict(name="norm_one", op="norm", rows=1, dim=4096, dtype="bf16", scale="e8m0", residual=True),
        # The same for the tokens of a long prompt, or of a batch of documents to embed.
        dict(name="norm_16k", op="norm", rows=16_384, dim=4096, dtype="bf16", scale="e8m0", residual=True),
        # Embeddings normed without a residual, rows that end inside a block, scales in 32 bits.
        dict(name="norm_ragged", op="norm", rows=4001, dim=1000, dtype="f32", scale="f32", residual=False),
        # The log probability of one drawn slot, with the twenty best: all latency.
        dict(name="log_probs_one", op="log_probs", rows=1, n=100_000, dtype="f32", given=1, top=20, temperature=1.0, allowed=1.0, grad=False),
        # A batch of draws over two-byte scores with many equal values, some slots filtered out.
        dict(name="log_probs_256", op="log_probs", rows=256, n=100_000, dtype="bf16", given=1, top=20, temperature=0.8, allowed=0.5, grad=False),
        # A training step: log probabilities and entropy of a batch of positions, and the gradient of both.
        dict(name="log_probs_train", op="log_probs", rows=2048, n=100_000, dtype="bf16", given=1, top=0, temperature=1.0, allowed=1.0, grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    dim = rng.choice([128, 256, 384, 512, 768, 1024, 1536, 2048]) if rng.random() < 0.5 else _log_int(rng, 8, 4096)
    op = rng.choice(["quantize4", "matmul4", "matmul4", "norm", "log_probs", "log_probs"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "quantize4":
        return dict(op=op, rows=_log_int(rng, 1, min(1_000_000, _MOST_ELEMENTS // dim)), dim=dim, dtype=dtype)
    if op == "matmul4":
        n = _log_int(rng, 100, min(1_000_000, _MOST_STORED // dim))
        most = min(4096, _MOST_PRODUCTS // (n * dim), _MOST_OUTPUTS // n)
        m = 1 if rng.random() < 0.25 else _log_int(rng, 1, most)
        return dict(op=op, m=m, n=n, dim=dim, out=dtype)
    if op == "norm":
        dim = dim if rng.random() < 0.75 else _log_int(rng, 4096, 16_384)
        return dict(op=op, rows=_log_int(rng, 1, min(100_000, _MOST_NORMED // dim)), dim=dim, dtype=dtype, scale=rng.choice(["e8m0", "f32"]), residual=rng.random() < 0.6)
    grad = rng.random() < 0.4
    rows = 1 if rng.random() < 0.2 else _log_int(rng, 2, 4096)
    n = _log_int(rng, 2, min(10_000_000, _MOST_SCORES // (rows * (1 if grad else 4))))
    return dict(op=op, rows=rows, n=n, dtype=dtype, given=rng.choice([1, 1, 1, min(8, n)]), top=0 if grad else rng.choice([0, 1, 5, 20, 64]),
                temperature=rng.choice([0.3, 0.8, 1.0, 1.0, 1.5]), allowed=rng.choice([1.0, 1.0, 0.5]), grad=grad)


# ---- inputs -------------------------------------------------------------------------------------

def _unit_rows(g, rows, dim):
    """Embeddings as models give them: unit vectors whose coordinates differ in spread."""
    x = torch.randn(rows, dim, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(dim, generator=g, device="cuda"))
    return x.div_(x.norm(dim=1, keepdim=True))


def _stored4(g, rows, dim):
    """(codes, scales): 4-bit rows as a program keeps them, two codes a byte, the first in the low half; each row at a multiple of 16 bytes."""
    x = _unit_rows(g, rows, dim)
    stored = torch.empty(rows, -(-dim // _BLOCK4), dtype=torch.uint8, device="cuda")
    codes = torch.zeros(rows, -(-dim // 32) * 16, dtype=torch.uint8, device="cuda")[:, :(dim + 1) // 2]
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0], device="cuda")
    for at in range(0, rows, 200_000):
        part = x[at:at + 200_000]
        q, s = _plain_round4(part)
        c = torch.bucketize(q.abs(), grid, out_int32=True).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
        c = torch.nn.functional.pad(c.view(len(part), -1)[:, :dim], (0, dim % 2))
        codes[at:at + 200_000] = c[:, 0::2] | (c[:, 1::2] << 4)
        stored[at:at + 200_000] = s
    return codes, stored.view(torch.float8_e8m0fnu)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1_000_003 + 31)
    op, state = case["op"], dict(case=case)
    if op == "quantize4":
        state["x"] = _unit_rows(g, case["rows"], case["dim"]).to(_DTYPES[case["dtype"]])
    elif op == "matmul4":
        state["a"] = _stored4(g, case["m"], case["dim"])
        state["b"] = _stored4(g, case["n"], case["dim"])
    elif op == "norm":
        rows, dim, dtype = case["rows"], case["dim"], _DTYPES[case["dtype"]]
        spread = torch.exp(0.5 * torch.randn(dim, generator=g, device="cuda"))       # (hidden states have coordinates of their own size)
        state["x"] = (torch.randn(rows, dim, generator=g, device="cuda") * spread).to(dtype)
        state["residual"] = (4 * torch.randn(rows, dim, generator=g, device="cuda") * spread).to(dtype) if case["residual"] else None
        state["weight"] = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).to(dtype)
    else:
        rows, n = case["rows"], case["n"]
        state["scores"] = (3 * torch.randn(rows, n, generator=g, device="cuda")).to(_DTYPES[case["dtype"]]).requires_grad_(case["grad"])
        state["slots"] = torch.randint(0, n, (rows, case["given"]), generator=g, device="cuda")
        state["temperature"] = case["temperature"] * (0.75 + 0.5 * torch.rand(rows, generator=g, device="cuda"))
        state["grads"] = [torch.randn(rows, case["given"], generator=g, device="cuda") / rows, -0.01 * torch.rand(rows, generator=g, device="cuda") / rows] if case["grad"] else None
        state["mask"] = None
        if case["allowed"] < 1:
            bits = torch.rand(-(-n // 64), 64, generator=g, device="cuda") < case["allowed"]
            bits[0, 0] = True                  # (something is allowed; empty masks are a matter of tests)
            state["mask"] = (bits.long() << torch.arange(64, device="cuda")).sum(1)
            there = bits.view(-1)[:n].nonzero()[:, 0]                # (what was drawn is allowed)
            state["slots"] = there[torch.randint(0, len(there), (rows, case["given"]), generator=g, device="cuda")]
    return state


# ---- the operators in plain form ------------------------------------------------------------------

def _blocks(x, size):
    """x padded with zeros and seen as [rows, blocks, size]."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % size)).view(len(x), -1, size)


def _plain_round4(x):
    """(codes as the numbers they are [rows, blocks, 32], scale bytes)."""
    x = _blocks(x.float(), _BLOCK4)
    most = x.abs().amax(2)
    m, e = torch.frexp(most)                   # most = m * 2^e; 7 = 0.875 * 2^3
    e = torch.where(most > 0, e - 3 + (m >= 0.875).int(), -126).clamp(-126, 127)
    stored = torch.where(torch.isfinite(x).all(2), e + 127, 255).to(torch.uint8)
    q = x * torch.ldexp(torch.ones_like(most), -e)[:, :, None]
    step = torch.where(q.abs() < 2, 0.5, torch.where(q.abs() < 4, 1.0, 2.0))
    return (torch.round(q / step) * step).clamp(-6.0, 6.0), stored


def _plain_quantize4(x):
    """The values of the 4-bit rows, in bfloat16 (which holds them exactly), and their scales."""
    q, stored = _plain_round4(x)
    scales = stored.view(torch.float8_e8m0fnu)
    return (q * scales.float()[:, :, None]).view(len(x), -1)[:, :x.shape[1]].to(torch.bfloat16), scales


def _plain_values4(codes, scales, dim):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device="cuda")
    both = torch.stack((codes & 15, codes >> 4), 2).view(len(codes), -1)[:, :dim]
    return grid[both.int()] * scales.float().repeat_interleave(_BLOCK4, 1)[:, :dim]


def _plain_matmul4(a, b, dim, dtype):
    return (_plain_values4(*a, dim) @ _plain_values4(*b, dim).t()).to(dtype)


def _plain_quantize8(y, scale):
    x = _blocks(y, _BLOCK8)
    most = x.abs().amax(2)
    if scale == "f32":
        s = stored = torch.clamp(most / _TOP8, min=2.0 ** -126)
    else:
        m, e = torch.frexp(most)               # most = m * 2^e, 448 = 0.875 * 2^9
        e = torch.where(most > 0, e - 9 + (m > 0.875).int(), -126).clamp(-126, 127)
        s = torch.ldexp(torch.ones_like(most), e)
        stored = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    return (x / s[:, :, None]).to(torch.float8_e4m3fn).view(len(y), -1)[:, :y.shape[1]], stored


def _plain_norm(x, residual, weight, scale):
    h = x.float() if residual is None else x.float() + residual.float()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + _EPS) * weight.float()
    made = _plain_quantize8(y, scale)
    return made if residual is None else (*made, h.to(x.dtype))


def _allowed(mask, n):
    return ((mask[:, None] >> torch.arange(64, device=mask.device)) & 1).reshape(-1)[:n].bool()


def _plain_log_probs(scores, slots, temperature, mask, top, grads):
    n = scores.shape[1]
    s = scores.float()
    if mask is not None:
        s = torch.where(_allowed(mask, n), s, -math.inf)
    d = (s - s.amax(1, keepdim=True)) / temperature[:, None]
    e = torch.exp(d)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    log_p = (d - total.log()).float()
    p = (e / total).float()
    entropy = (total.log()[:, 0] - (p * d.clamp(min=-1e30)).sum(1, dtype=torch.float64)).float()
    found = [log_p.gather(1, slots), entropy]
    if top:
        k = min(top, n)
        order = torch.sort(s, dim=1, descending=True, stable=True).indices[:, :k]
        best = log_p.gather(1, order)
        order = torch.where(best > -math.inf, order, -1)
        found += [torch.nn.functional.pad(order, (0, top - k), value=-1), torch.nn.functional.pad(best, (0, top - k), value=-math.inf)]
    if grads is not None:
        g_slots, g_entropy = grads
        g = -p * (g_slots.sum(1, keepdim=True) + g_entropy[:, None] * (log_p.clamp(min=-1e30) + entropy[:, None]))
        found.append((g.scatter_add(1, slots, g_slots) / temperature[:, None]).to(scores.dtype))
    return found


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from turbovec_amd import fp4, norm, sampling
        if op == "quantize4":
            rows = fp4.quantize(state["x"])
            return rows.values(torch.bfloat16), rows.scales
        if op == "matmul4":
            return fp4.matmul(fp4.Fp4Rows(*state["a"], case["dim"]), fp4.Fp4Rows(*state["b"], case["dim"]), dtype=_DTYPES[case["out"]])
        if op == "norm":
            if state["residual"] is None:
                rows = norm.rms_norm(state["x"], state["weight"], eps=_EPS, scale=case["scale"])
                return rows.codes, rows.scales
            rows, summed = norm.add_rms_norm(state["x"], state["residual"], state["weight"], eps=_EPS, scale=case["scale"])
            return rows.codes, rows.scales, summed
        found = sampling.log_probs(state["scores"], state["slots"], temperature=state["temperature"], mask=state["mask"], top=case["top"])
        outputs = [found.log_probs, found.entropy]
        if case["top"]:
            outputs += [found.top_slots, found.top_log_probs]
        if state["grads"] is not None:
            outputs += torch.autograd.grad((found.log_probs, found.entropy), state["scores"], state["grads"])
        return outputs
    if op == "quantize4":
        return _plain_quantize4(state["x"])
    if op == "matmul4":
        return _plain_matmul4(state["a"], state["b"], case["dim"], _DTYPES[case["out"]])
    if op == "norm":
        return _plain_norm(state["x"], state["residual"], state["weight"], case["scale"])
    with torch.no_grad():
        return _plain_log_probs(state["scores"], state["slots"], state["temperature"], state["mask"], case["top"], state["grads"])


def work(case):
    """Each input read once and each output written once; one multiply-add a coordinate of every pair.  A norm takes some ten
    operations a value, a log probability some ten a score, its gradient as many."""
    op = case["op"]
    if op == "log_probs":
        cells, size = case["rows"] * case["n"], _DTYPES[case["dtype"]].itemsize
        return {"bytes": cells * size * (2 if case["grad"] else 1) + (case["allowed"] < 1) * case["n"] / 8 + case["rows"] * (8 + 12 * case["given"] + 12 * case["top"]),
                "flops": 10.0 * cells * (2 if case["grad"] else 1)}
    dim = case["dim"]
    row4 = -(-dim // 2) + -(-dim // _BLOCK4)                  # bytes of a 4-bit row
    if op == "matmul4":
        m, n = case["m"], case["n"]
        return {"bytes": (m + n) * row4 + m * n * _DTYPES[case["out"]].itemsize, "flops": 2.0 * m * n * dim}
    cells, size = case["rows"] * dim, _DTYPES[case["dtype"]].itemsize
    if op == "quantize4":                                     # (what the rows are read back as)
        return {"bytes": cells * (size + 2) + case["rows"] * -(-dim // _BLOCK4), "flops": 3.0 * cells}
    made = cells + case["rows"] * -(-dim // _BLOCK8) * (1 if case["scale"] == "e8m0" else 4)
    return {"bytes": cells * size * (3 if case["residual"] else 1) + dim * size + made, "flops": 10.0 * cells}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def _exact_scales(y, size, border, floor=2.0 ** -126):
    """The smallest power of two, of each block, that its largest magnitude divided by is below `border` (or at it, where the border is a code)."""
    most = torch.stack([part.abs().amax(1) for part in y.split(size, 1)], 1)
    s = torch.exp2(torch.floor(torch.log2(most.clamp(min=1e-60) / border)))
    fits = (lambda s: most < border * s) if border == 7.0 else (lambda s: most <= border * s)
    s = torch.where(fits(s), s, 2 * s)
    return s.clamp(min=floor)


def _exact_matmul4(a, b, dim):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    grid = torch.cat((grid, -grid))

    def row_values(codes, scales):
        x = torch.empty(len(codes), dim, dtype=torch.float64, device="cuda")
        x[:, 0::2] = grid[(codes % 16).long()]
        x[:, 1::2] = grid[(codes // 16).long()][:, :dim // 2]
        return x * torch.exp2(scales.view(torch.uint8).double() - 127).repeat_interleave(_BLOCK4, 1)[:, :dim]

    x = row_values(*a)
    return torch.cat([x @ row_values(codes, scales).t() for codes, scales in zip(b[0].split(100_000), b[1].split(100_000))], 1)


def _exact_quantize4(x):
    """Values of the nearest codes, which a place among the middles between two codes tells; those in the middle go to the even one."""
    scales, values = _exact_scales(x, _BLOCK4, 7.0), []
    for part, s in zip(x.split(50_000), scales.split(50_000)):
        s = s.repeat_interleave(_BLOCK4, 1)[:, :x.shape[1]]
        q = part.abs() / s
        up = 0.5 * sum((q > t).double() for t in (0.25, 1.25)) + 0.5 * sum((q >= t).double() for t in (0.75, 1.75))
        up += (q > 2.5).double() + (q >= 3.5).double() + 2 * (q > 5).double()
        values.append(torch.copysign(up, part) * s)
    return torch.cat(values), scales


def _exact_norm(state, scale):
    h = state["x"].double()
    if state["residual"] is not None:
        h = h + state["residual"].double()
    y = h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + _EPS) * state["weight"].double()
    s = torch.stack([part.abs().amax(1) for part in y.split(_BLOCK8, 1)], 1) / _TOP8 if scale == "f32" else _exact_scales(y, _BLOCK8, _TOP8)
    made = (y / s.repeat_interleave(_BLOCK8, 1)[:, :y.shape[1]], s)
    return made if state["residual"] is None else (*made, h)


def _exact_log_probs(state, top):
    z = state["scores"].detach().double()
    z = z / state["temperature"].double()[:, None]
    if state["mask"] is not None:
        z = z.masked_fill(~_allowed(state["mask"], z.shape[1]), -math.inf)
    lse = torch.logsumexp(z, 1)
    q = z - lse[:, None]
    p = torch.exp(q)
    entropy = -torch.where(p > 0, p * q, 0.0).sum(1)
    found = [q.gather(1, state["slots"]), entropy]
    if top:
        best = torch.topk(q, min(top, q.shape[1]), 1).values
        found += [None, torch.nn.functional.pad(best, (0, top - best.shape[1]), value=-math.inf)]
    if state["grads"] is not None:
        g_slots, g_entropy = (g.double() for g in state["grads"])
        picked = torch.zeros_like(p)
        for i in range(g_slots.shape[1]):
            picked.scatter_add_(1, state["slots"][:, i:i + 1], g_slots[:, i:i + 1])
        towards = torch.where(p > 0, p * (q + entropy[:, None]), 0.0)
        found.append((picked - p * g_slots.sum(1, keepdim=True) - towards * g_entropy[:, None]) / state["temperature"].double()[:, None])
    return found


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize4":
        return _exact_quantize4(state["x"].double())
    if case["op"] == "matmul4":
        return _exact_matmul4(state["a"], state["b"], case["dim"])
    if case["op"] == "norm":
        return _exact_norm(state, case["scale"])
    return _exact_log_probs(state, case["top"])
