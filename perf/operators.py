"""The timed cases of the operators beside the search: 8-bit rows, their products, and drawing from scores.

Four operators.  "quantize" makes 8-bit rows (e4m3 codes, a scale for each block of 128 coordinates);
"matmul" scores 8-bit queries against all 8-bit rows; "rescore" scores the slots that a search returned
against the rows' 8-bit form and puts them in order again; "sample" draws a slot from rows of scores.

Sizes are those of this repository's benchmark and tests (100K, 1M and 10M rows, 1536 dimensions, batches
of 1024, 100 candidates) or generic; `draw` spreads over the same ranges.
"""
import math

import torch

own = False

_BLOCK = 128
_TOP = 448.0                                  # the largest e4m3 value
_MOST_ELEMENTS = 400_000 * 1536               # of rows to quantise
_MOST_PRODUCTS = 1024 * 100_000 * 1536        # of a product
_MOST_OUTPUTS = 1024 * 100_000
_MOST_STORED = 1_000_000 * 1536
_MOST_GATHERED = 1024 * 100 * 1536
_MOST_SCORES = 256 * 100_000
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # A middle-sized batch of queries made 8-bit before each product: all latency.
        dict(name="quantize_64", op="quantize", rows=64, dim=1536, dtype="f32", scale="e8m0", group=1),
        # Rows of a shard as a model produced them, made 8-bit as they are added.
        dict(name="quantize_400k", op="quantize", rows=400_000, dim=1536, dtype="f32", scale="e8m0", group=1),
        # One query through a projection in front of the index, scales of 128 x 128 tiles: all latency.
        dict(name="project_one", op="matmul", m=1, n=1536, dim=1536, out="bf16", scale="f32", group=128),
        # One query against every row of a large collection: one pass over the rows.
        dict(name="score_one_1m", op="matmul", m=1, n=1_000_000, dim=1536, out="f32", scale="e8m0", group=1),
        # Odd everything: a batch off every tile edge, rows that end inside a block, scales in 32 bits a row.
        dict(name="score_ragged", op="matmul", m=37, n=77_777, dim=1000, out="f32", scale="f32", group=1),
        # A batch against a collection, every score wanted (ground truth of a recall measurement).
        dict(name="score_batch_100k", op="matmul", m=1024, n=100_000, dim=1536, out="f32", scale="e8m0", group=1),
        # A projection of many rows with weights laid out elsewhere, scales of 128 x 128 tiles.
        dict(name="project_4096", op="matmul", m=4096, n=4096, dim=4096, out="bf16", scale="f32", group=128),
        # One user's hundred candidates scored again: all latency.
        dict(name="rescore_one", op="rescore", nq=1, m=100, n=100_000, dim=1536, k=10, dtype="f32", scale="e8m0", group=1),
        # The same for an offline batch.
        dict(name="rescore_batch", op="rescore", nq=1024, m=100, n=1_000_000, dim=1536, k=10, dtype="f32", scale="e8m0", group=1),
        # One draw from the scores of a collection, the usual filters on.
        dict(name="sample_one_100k", op="sample", rows=1, n=100_000, dtype="f32", spread=3.0, temperature=0.8, top_k=50, top_p=0.9, min_p=0.0, allowed=1.0),
        # A batch of draws over two-byte scores with many equal values, no limit on how many rows stay.
        dict(name="sample_256", op="sample", rows=256, n=100_000, dtype="bf16", spread=3.0, temperature=0.8, top_k=0, top_p=0.95, min_p=0.001, allowed=1.0),
        # A hard negative from the inner products with ten million rows, half of them filtered out.
        dict(name="sample_one_10m", op="sample", rows=1, n=10_000_000, dtype="f32", spread=0.026, temperature=0.02, top_k=0, top_p=0.5, min_p=0.0, allowed=0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    dim = rng.choice([128, 256, 384, 512, 768, 1024, 1536, 2048]) if rng.random() < 0.5 else _log_int(rng, 8, 4096)
    scale = rng.choice(["e8m0", "f32"])
    op = rng.choice(["quantize", "matmul", "matmul", "rescore", "sample", "sample"])
    if op == "quantize":
        return dict(op=op, rows=_log_int(rng, 1, min(1_000_000, _MOST_ELEMENTS // dim)), dim=dim, dtype=rng.choice(["f32", "f16", "bf16"]),
                    scale=scale, group=rng.choice([1, 1, 128]))
    if op == "matmul":
        n = _log_int(rng, 100, min(1_000_000, _MOST_STORED // dim))
        most = min(4096, _MOST_PRODUCTS // (n * dim), _MOST_OUTPUTS // n)
        m = 1 if rng.random() < 0.25 else _log_int(rng, 1, most)
        return dict(op=op, m=m, n=n, dim=dim, out=rng.choice(["f32", "f16", "bf16"]), scale=scale, group=rng.choice([1, 128]))
    if op == "rescore":
        m = _log_int(rng, 1, 1000)
        nq = _log_int(rng, 1, min(1024, _MOST_GATHERED // (m * dim)))
        return dict(op=op, nq=nq, m=m, n=_log_int(rng, 1000, min(1_000_000, _MOST_STORED // dim)), dim=dim, k=_log_int(rng, 1, min(m, 100)),
                    dtype=rng.choice(["f32", "f16", "bf16"]), scale=scale, group=rng.choice([1, 1, 128]))
    rows = 1 if rng.random() < 0.3 else _log_int(rng, 2, 1024)
    return dict(op=op, rows=rows, n=_log_int(rng, 2, min(10_000_000, _MOST_SCORES // rows)), dtype=rng.choice(["f32", "f16", "bf16"]),
                spread=rng.choice([3.0, 8.0]), temperature=rng.choice([0.3, 0.8, 1.0, 1.5]), top_k=rng.choice([0, 0, _log_int(rng, 1, 2000)]),
                top_p=rng.choice([1.0, 0.5, 0.9, 0.99]), min_p=rng.choice([0.0, 0.0, 0.02]), allowed=rng.choice([1.0, 1.0, 0.5, 0.01]))


# ---- inputs -------------------------------------------------------------------------------------

def _unit_rows(g, rows, dim):
    """Embeddings as models give them: unit vectors whose coordinates differ in spread."""
    x = torch.randn(rows, dim, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(dim, generator=g, device="cuda"))
    return x.div_(x.norm(dim=1, keepdim=True))


def _stored(g, rows, dim, scale, group):
    """(codes, scales): 8-bit rows as a program keeps them, each row at a multiple of 16 bytes."""
    at = -(-dim // 16) * 16
    codes = torch.zeros(rows, at, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :dim]
    c, s = _plain_quantize(_unit_rows(g, rows, dim), scale, group)
    codes.view(torch.uint8).copy_(c.view(torch.uint8))
    return codes, s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1_000_003 + 29)
    op, state = case["op"], dict(case=case)
    if op == "quantize":
        state["x"] = _unit_rows(g, case["rows"], case["dim"]).to(_DTYPES[case["dtype"]])
    elif op == "matmul":
        state["a"] = _stored(g, case["m"], case["dim"], case["scale"], 1)
        state["b"] = _stored(g, case["n"], case["dim"], case["scale"], case["group"])
    elif op == "rescore":
        state["rows"] = _stored(g, case["n"], case["dim"], case["scale"], case["group"])
        state["queries"] = _unit_rows(g, case["nq"], case["dim"]).to(_DTYPES[case["dtype"]])
        state["slots"] = torch.randint(0, case["n"], (case["nq"], case["m"]), generator=g, device="cuda")
    else:
        rows, n = case["rows"], case["n"]
        state["scores"] = (case["spread"] * torch.randn(rows, n, generator=g, device="cuda")).to(_DTYPES[case["dtype"]])
        state["u"] = torch.rand(rows, generator=g, device="cuda")
        state["temperature"] = case["temperature"] * (0.75 + 0.5 * torch.rand(rows, generator=g, device="cuda"))
        state["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
        state["top_p"] = torch.full((rows,), case["top_p"], device="cuda")
        state["min_p"] = torch.full((rows,), case["min_p"], device="cuda")
        state["mask"] = None
        if case["allowed"] < 1:
            bits = torch.rand(-(-n // 64), 64, generator=g, device="cuda") < case["allowed"]
            bits[0, 0] = True                  # (something is allowed; empty masks are a matter of tests)
            state["mask"] = (bits.long() << torch.arange(64, device="cuda")).sum(1)
    return state


# ---- the operators in plain form ------------------------------------------------------------------

def _blocks(x, group):
    """x padded with zeros and seen as [groups, group, blocks, 128]."""
    rows, dim = x.shape
    x = torch.nn.functional.pad(x, (0, -dim % _BLOCK, 0, -rows % group))
    return x.view(-1, group, x.shape[1] // _BLOCK, _BLOCK)


def _spread_scales(scales, group, rows, dim):
    """A scale for each code."""
    return scales.repeat_interleave(group, 0)[:rows].repeat_interleave(_BLOCK, 1)[:, :dim]


def _plain_quantize(x, scale, group):
    rows, dim = x.shape
    x = x.float()
    x4 = _blocks(x, group)
    finite = torch.isfinite(x4)
    most = torch.where(finite, x4.abs(), 0.0).amax((1, 3))
    if scale == "f32":
        s = stored = torch.clamp(most / _TOP, min=2.0 ** -126)
    else:
        m, e = torch.frexp(most)               # most = m * 2^e, 448 = 0.875 * 2^9
        e = torch.where(most > 0, e - 9 + (m > 0.875).int(), -126).clamp(-126, 127)
        s = torch.ldexp(torch.ones_like(most), e)
        stored = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    codes = torch.where(finite, x4 / s[:, None, :, None], math.nan).to(torch.float8_e4m3fn)
    return codes.view(codes.shape[0] * group, -1)[:rows, :dim], stored


def _plain_matmul(a, b, group, dtype):
    (ac, a_scales), (bc, b_scales) = a, b
    x = ac.float() * _spread_scales(a_scales.float(), 1, *ac.shape)
    y = bc.float() * _spread_scales(b_scales.float(), group, *bc.shape)
    return (x @ y.t()).to(dtype)


def _plain_rescore(queries, rows, group, slots, k):
    codes, scales = rows
    at = slots.clamp(0, len(codes) - 1)
    r = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).double()
    r *= scales.double()[at // group].repeat_interleave(_BLOCK, 2)[:, :, :codes.shape[1]]
    s = (r * queries.double()[:, None, :]).sum(2).float()
    there = (slots >= 0) & (slots < len(codes))
    s, at = torch.where(there, s, -math.inf), torch.where(there, slots, -1)
    by_slot = torch.sort(at, dim=1, stable=True)
    best = torch.sort(s.gather(1, by_slot.indices), dim=1, descending=True, stable=True)
    return best.values[:, :k].contiguous(), by_slot.values.gather(1, best.indices)[:, :k].contiguous()


def _allowed(mask, n):
    return ((mask[:, None] >> torch.arange(64, device=mask.device)) & 1).reshape(-1)[:n].bool()


def _plain_sample(scores, u, temperature, top_k, top_p, min_p, mask):
    rows, n = scores.shape
    s = scores.double()
    if mask is not None:
        s = torch.where(_allowed(mask, n), s, -math.inf)
    w = torch.exp((s - s.amax(1, keepdim=True)) / temperature.double()[:, None])
    order = torch.sort(s, dim=1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    place = torch.arange(n, device=s.device)
    ranked = torch.where((top_k[:, None] <= 0) | (place < top_k[:, None]), ranked, 0.0)
    upto = ranked.cumsum(1)
    stays = (upto - ranked < top_p.double()[:, None] * upto[:, -1:]) | (top_p[:, None] >= 1)
    stays &= ranked >= min_p.double()[:, None]
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(stays, ranked, 0.0))
    upto = kept.cumsum(1)
    slot = (upto > u.double()[:, None] * upto[:, -1:]).int().argmax(1)
    return slot, (kept.gather(1, slot[:, None]) / upto[:, -1:]).float()[:, 0]


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from turbovec_amd import fp8, sampling
        if op == "quantize":
            rows = fp8.quantize(state["x"], scale=case["scale"], group=case["group"])
            return rows.codes, rows.scales
        if op == "matmul":
            return fp8.matmul(fp8.Fp8Rows(*state["a"]), fp8.Fp8Rows(*state["b"], group=case["group"]), dtype=_DTYPES[case["out"]])
        if op == "rescore":
            return fp8.rescore(state["queries"], fp8.Fp8Rows(*state["rows"], group=case["group"]), state["slots"], case["k"])
        return sampling.sample(state["scores"], state["u"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                               min_p=state["min_p"], mask=state["mask"])
    if op == "quantize":
        return _plain_quantize(state["x"], case["scale"], case["group"])
    if op == "matmul":
        return _plain_matmul(state["a"], state["b"], case["group"], _DTYPES[case["out"]])
    if op == "rescore":
        return _plain_rescore(state["queries"], state["rows"], case["group"], state["slots"], case["k"])
    return _plain_sample(state["scores"], state["u"], state["temperature"], state["top_k"], state["top_p"], state["min_p"], state["mask"])


def work(case):
    """Each input read once and each output written once; one multiply-add a coordinate of every pair.  A draw compares,
    takes an exponential and adds: ten operations a score."""
    op = case["op"]
    if op == "sample":
        cells = case["rows"] * case["n"]
        return {"bytes": cells * _DTYPES[case["dtype"]].itemsize + (case["allowed"] < 1) * case["n"] / 8 + 32 * case["rows"], "flops": 10.0 * cells}
    dim, scale = case["dim"], 1 if case["scale"] == "e8m0" else 4
    scales = -(-dim // _BLOCK) * scale                       # bytes of a row's scales
    if op == "quantize":
        size = _DTYPES[case["dtype"]].itemsize
        return {"bytes": case["rows"] * dim * (size + 1) + -(-case["rows"] // case["group"]) * scales, "flops": 3.0 * case["rows"] * dim}
    if op == "matmul":
        m, n = case["m"], case["n"]
        return {"bytes": (m + n) * dim + (m + -(-n // case["group"])) * scales + m * n * _DTYPES[case["out"]].itemsize, "flops": 2.0 * m * n * dim}
    nq, m = case["nq"], case["m"]
    rows = min(nq * m, case["n"])
    return {"bytes": rows * dim + -(-rows // case["group"]) * scales + nq * (dim * _DTYPES[case["dtype"]].itemsize + 8 * m + 12 * case["k"]),
            "flops": 2.0 * nq * m * dim}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def _exact_quantize(x, scale, group):
    """Scales, and the unrounded quotients that the codes stand for."""
    x = x.double()
    rows, dim = x.shape
    values, scales = torch.empty_like(x), []
    for at in range(0, dim, _BLOCK):
        part = x[:, at:at + _BLOCK]
        most = part.abs().amax(1)
        most = torch.stack([p.max() for p in most.split(group)]) if group > 1 else most
        s = most / _TOP
        if scale == "e8m0":
            s = torch.where(s > 0, torch.exp2(torch.ceil(torch.log2(s))), 0.0)
        s = s.clamp(min=2.0 ** -126)
        values[:, at:at + _BLOCK] = part / s.repeat_interleave(group)[:rows, None]
        scales.append(s)
    return values, torch.stack(scales, 1)


def _exact_matmul(a, b, group):
    (ac, a_scales), (bc, b_scales) = a, b
    total = 0.0
    for k in range(a_scales.shape[1]):
        part = slice(k * _BLOCK, (k + 1) * _BLOCK)
        x = ac[:, part].double() * a_scales[:, k:k + 1].double()
        y = bc[:, part].double() * b_scales[:, k].double().repeat_interleave(group)[:len(bc), None]
        total = total + x @ y.t()
    return total


def _exact_rescore(queries, rows, group, slots, k):
    codes, scales = rows
    best = []
    for q, at in zip(queries.double(), slots):
        x = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).double()
        s = scales[at // group].double() if scales.dtype == torch.float32 else torch.exp2(scales.view(torch.uint8)[at // group].double() - 127)
        products = torch.nn.functional.pad(x * q, (0, -len(q) % _BLOCK)).view(len(at), -1, _BLOCK).sum(2)
        best.append((products * s).sum(1).sort(descending=True).values[:k])
    return torch.stack(best), None


def _exact_sample(state):
    """The probability of the slot drawn, one row after the other, from logarithms."""
    probabilities = []
    for r, row in enumerate(state["scores"]):
        z = row.double() / state["temperature"][r].double()
        there = torch.arange(len(z), device=z.device) if state["mask"] is None else _allowed(state["mask"], len(z)).nonzero()[:, 0]
        z = z[there]
        order = torch.argsort(-z, stable=True)
        if state["top_k"][r] > 0:
            order = order[:int(state["top_k"][r])]
        if state["top_p"][r] < 1:
            before = torch.softmax(z[order], 0).cumsum(0).roll(1)
            before[0] = 0
            order = order[before < state["top_p"][r].double()]
        order = order[z[order] - z.max() >= state["min_p"][r].double().log()]
        kept = order.sort().values
        p = torch.softmax(z[kept], 0)
        probabilities.append(p[torch.searchsorted(p.cumsum(0), state["u"][r].double()[None], right=True).clamp(max=len(p) - 1)[0]])
    return None, torch.stack(probabilities)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_quantize(state["x"], case["scale"], case["group"])
    if case["op"] == "matmul":
        return _exact_matmul(state["a"], state["b"], case["group"])
    if case["op"] == "rescore":
        return _exact_rescore(state["queries"], state["rows"], case["group"], state["slots"], case["k"])
    return _exact_sample(state)
