"""Drawing from scores against a plain 64-bit form of the definition: every limit alone and together, ties, masks, infinities and
NaN, rows of one score and of a million, every type and stride."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def sample():
    from turbovec_amd.sampling import sample
    return sample


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def plain_row(s, u, t, k, p, m, allowed):
    """(slot, probability) of one row; s float64.  Weights are whole multiples of 2^-(63 - ceil(log2 n)), rounded down: one below
    that is never drawn, not even by u = 0."""
    unit = 2.0 ** -(63 - max(1, int(len(s) - 1).bit_length()))
    s = np.where(allowed & ~np.isnan(s), s, -np.inf)
    if np.all(s == -np.inf):
        return -1, 0.0
    top = s.max()
    if not t > 0:
        return int(np.argmax(s)), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(s == top, 1.0, np.exp((s - top) / t))
    order = np.lexsort((np.arange(len(s)), -s))
    order = order[s[order] > -np.inf]
    if k > 0:
        order = order[:k]
    if p < 1:
        mass = np.cumsum(np.floor(w[order] / unit) * unit)
        stays = np.concatenate(([0.0], mass[:-1])) < p * mass[-1]
        stays[0] = True
        order = order[stays]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    kept = np.sort(order)
    mass = np.cumsum(np.floor(w[kept] / unit) * unit)
    want = u * mass[-1]
    at = min(int(np.searchsorted(mass, want, side="right")), len(kept) - 1)
    return int(kept[at]), w[kept[at]] / mass[-1]


def bits(mask, n):
    if mask is None:
        return np.ones(n, bool)
    words = mask.cpu().numpy().view(np.uint64)
    return ((words[:, None] >> np.arange(64, dtype=np.uint64)) & np.uint64(1)).astype(bool).ravel()[:n]


def check(sample, scores, u, mask=None, **params):
    slots, probs = sample(scores, u, mask=mask, **params)
    rows, n = scores.shape
    host = scores.double().cpu().numpy()
    value = lambda name, r, default: default if params.get(name) is None else float(params[name][r]) if isinstance(params[name], torch.Tensor) else float(np.float32(params[name]))  # noqa: E731
    for r in range(rows):
        allowed = bits(mask if mask is None or mask.dim() == 1 else mask[r], n)
        slot, prob = plain_row(host[r], float(u[r]), value("temperature", r, 1.0), int(value("top_k", r, 0)), value("top_p", r, 1.0), value("min_p", r, 0.0), allowed)
        assert int(slots[r]) == slot, (r, int(slots[r]), slot)
        # weights lose less than 2^-(63 - ceil(log2 n)) each against a sum of at least 1, and are off by their series' first term left out,
        # (ln 2 / 2)^10 / 10! = 6.9e-12 against 2^-1/2 at least; the quotient is rounded once to 32 bits
        assert abs(float(probs[r]) - prob) <= prob * (2.0 ** -24 + n * 2.0 ** -(63 - int(n - 1).bit_length()) + 1e-11) + 2.0 ** -149, (r, float(probs[r]), prob)
    return slots, probs


LIMITS = [dict(), dict(top_k=1), dict(top_k=7), dict(top_k=1000), dict(top_p=0.5), dict(top_p=0.99), dict(min_p=0.1), dict(top_k=50, top_p=0.9),
          dict(top_k=50, top_p=0.9, min_p=0.05), dict(temperature=0.1), dict(temperature=3.0, top_p=0.3), dict(temperature=0.0), dict(top_p=1e-6), dict(top_p=0.0), dict(top_p=-0.5), dict(top_p=-float("inf")),
          dict(min_p=1.0), dict(min_p=5.0), dict(top_k=-3), dict(top_p=2.0), dict(temperature=float("inf"), top_k=30)]


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 100, 1000, 1024, 1025, 5000, 20000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_limits(sample, n, dtype):
    scores = (3 * torch.randn(6, n, generator=gen(n), device="cuda")).to(dtype)
    u = torch.rand(6, generator=gen(n + 1), device="cuda")
    u[0] = 0.0
    u[1] = 1.0 - 2.0 ** -24
    for limits in LIMITS:
        check(sample, scores, u, **limits)


@pytest.mark.parametrize("n", [50_000, 131_072, 300_001, 1_000_003])
@pytest.mark.parametrize("rows", [1, 3])
def test_long_rows(sample, n, rows):
    for dtype, spread in ((torch.float32, 3.0), (torch.bfloat16, 3.0), (torch.float32, 0.03)):
        scores = (spread * torch.randn(rows, n, generator=gen(5), device="cuda")).to(dtype)
        u = torch.rand(rows, generator=gen(6), device="cuda")
        for limits in (dict(), dict(top_k=40), dict(top_k=60_000), dict(top_p=0.9), dict(top_k=5000, top_p=0.7, min_p=0.01), dict(temperature=0.2, top_p=0.95)):
            check(sample, scores, u, **limits)


@pytest.mark.parametrize("rows,n", [(2, 6144), (2, 6145), (257, 6145), (2, 16384), (2, 16385), (128, 16385), (129, 16385), (2, 40960), (2, 40961), (128, 40961), (129, 40961), (257, 16448), (257, 16449)])
def test_where_the_forms_meet(sample, rows, n):
    """Sizes on both sides of where a row gets more waves, or is cut into chunks."""
    for dtype in (torch.float32, torch.bfloat16):
        scores = (3 * torch.randn(rows, n, generator=gen(rows), device="cuda")).to(dtype)
        u = torch.rand(rows, generator=gen(n), device="cuda")
        k = torch.randint(0, 6000, (rows,), generator=gen(n + 1), device="cuda", dtype=torch.int32)
        k[::3] = 0
        t = 0.3 + torch.rand(rows, generator=gen(n + 2), device="cuda")
        check(sample, scores, u)
        check(sample, scores, u, temperature=t, top_k=k, top_p=0.9, min_p=1e-4)


@pytest.mark.parametrize("rows,n", [(1, 20_000), (1, 250_000), (3, 100_000), (140, 12_000), (140, 30_000), (600, 30_000)])
def test_thousands_stay(sample, rows, n):
    """Limits that leave more slots than are gathered: by number, by mass, by both, and by min-p."""
    scores = 2 * torch.randn(rows, n, generator=gen(rows + n), device="cuda")
    u = torch.rand(rows, generator=gen(n), device="cuda")
    some = torch.arange(0, rows, 15 if rows > 40 else 1, device="cuda")
    for limits in (dict(top_k=n // 2), dict(top_p=0.97, temperature=4.0), dict(top_k=n - 1, top_p=0.8, temperature=9.0), dict(top_k=5000, top_p=0.999, temperature=5.0, min_p=0.3),
                   dict(top_p=0.9, min_p=0.02, temperature=2.0), dict(min_p=0.01, temperature=1e4)):
        slots, probs = sample(scores, u, **limits)
        check(lambda *a, **b: (slots[some], probs[some]), scores[some], u[some], **limits)


@pytest.mark.parametrize("rows,n", [(1, 50_000), (2, 300_000), (150, 20_000)])
def test_crowded_scores(sample, rows, n):
    """Thousands of equal scores at the threshold, scores that differ in their last bits, that cross zero, that are subnormal, and one far above the others."""
    g = gen(rows)
    base = torch.randn(rows, n, generator=g, device="cuda")
    cases = [(0.5 * torch.round(2 * base), 1.0),                                   # about 20 values
             (1.0 + 2.0 ** -23 * torch.randint(0, 50, (rows, n), generator=g, device="cuda"), 1e-6),
             (1e-3 * base, 1e-3),
             (1e-41 * torch.randint(-500, 500, (rows, n), generator=g, device="cuda"), 1e-39),
             (torch.where(torch.arange(n, device="cuda") == n // 3, 1e6, base), 3e4)]
    u = torch.rand(rows, generator=g, device="cuda")
    some = torch.arange(0, rows, 50, device="cuda")
    for scores, t in cases:
        for limits in (dict(top_p=0.5), dict(top_k=n // 3), dict(top_k=6000, top_p=0.9), dict(top_k=100, top_p=0.999), dict(min_p=0.5, top_p=0.7)):
            slots, probs = sample(scores, u, temperature=t, **limits)
            check(lambda *a, **b: (slots[some], probs[some]), scores[some], u[some], temperature=t, **limits)


def test_long_rows_with_masks(sample):
    n, rows = 90_001, 5
    g = gen(50)
    scores = 3 * torch.randn(rows, n, generator=g, device="cuda")
    scores[1, 100:80_000] = float("nan")
    scores[2, 7] = scores[2, 70_000] = float("inf")
    scores[3] = -float("inf")
    words = -(-n // 64)
    half = torch.randint(-2 ** 63, 2 ** 63 - 1, (rows, words), generator=g, device="cuda", dtype=torch.int64)
    half[4] = 0
    half[4, -1] = -1 << (n % 64)                     # only bits past the row's end
    u = torch.rand(rows, generator=g, device="cuda")
    for mask in (half, half[0], half[4]):
        for limits in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95, temperature=2.0), dict(top_k=20_000, top_p=0.5), dict(temperature=0.0), dict(min_p=0.2)):
            check(sample, scores, u, mask=mask, **limits)


def test_draws_by_two_threads(sample):
    """Calls at once, each thread on a stream of its own: each gives what it gives alone."""
    import threading
    sets = []
    for i, (rows, n) in enumerate(((3, 60_000), (200, 3000))):
        scores = 3 * torch.randn(rows, n, generator=gen(60 + i), device="cuda")
        u = torch.rand(rows, generator=gen(70 + i), device="cuda")
        sets.append((scores, u, sample(scores, u, top_k=100, top_p=0.9)))
    torch.cuda.synchronize()
    same = [0, 0]

    def work(i):
        scores, u, want = sets[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = sample(scores, u, top_k=100, top_p=0.9)
                torch.cuda.current_stream().synchronize()
                same[i] += all(torch.equal(x, y) for x, y in zip(got, want))

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert same == [20, 20]


def test_more_rows_than_a_grid_has(sample):
    for n in (5, 7000):
        scores = (3 * torch.randn(66_000, n, generator=gen(81), device="cuda")).half()
        u = torch.rand(66_000, generator=gen(82), device="cuda")
        got = sample(scores, u, top_k=3, top_p=0.9)
        for lo in (0, 65_400, 65_900):
            for a, b in zip(got, sample(scores[lo:lo + 100], u[lo:lo + 100], top_k=3, top_p=0.9)):
                assert torch.equal(a[lo:lo + 100], b)
        check(sample, scores[65_530:65_545], u[65_530:65_545], top_k=3, top_p=0.9)


def test_no_rows(sample):
    slots, probs = sample(torch.empty(0, 100_000, device="cuda"), torch.empty(0, device="cuda"), top_k=5)
    assert slots.shape == probs.shape == (0,)


def test_many_rows(sample):
    scores = torch.randn(700, 1500, generator=gen(8), device="cuda")
    u = torch.rand(700, generator=gen(9), device="cuda")
    g = gen(10)
    check(sample, scores, u, temperature=2 * torch.rand(700, generator=g, device="cuda"), top_k=torch.randint(-2, 1600, (700,), generator=g, device="cuda", dtype=torch.int32),
          top_p=1.2 * torch.rand(700, generator=g, device="cuda"), min_p=0.3 * torch.rand(700, generator=g, device="cuda") - 0.05)


@pytest.mark.parametrize("n", [10, 4096, 40_000])
def test_ties(sample, n):
    """Rows of few different scores, of one, and of two far apart: what stays of equal scores is the lowest slots."""
    g = gen(11)
    few = torch.randint(0, 3, (4, n), generator=g, device="cuda").float()
    same = torch.full((4, n), -2.5, device="cuda")
    signs = torch.where(torch.rand(4, n, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    u = torch.tensor([0.0, 0.3, 0.75, 0.99999], device="cuda")
    for scores in (few, same, signs, -1e30 * few):
        for limits in (dict(), dict(top_k=5), dict(top_k=n // 2 + 1), dict(top_p=0.5), dict(top_p=0.25, top_k=n - 1), dict(min_p=1.0), dict(temperature=0.0)):
            check(sample, scores, u, **limits)


@pytest.mark.parametrize("rows,n", [(1, 1000), (1, 10_000), (200, 10_000), (2, 200_000)])
def test_min_p_above_the_slot_that_top_p_ends_at(sample, rows, n):
    """Top-p ends at a slot that is alone between its neighbours, and min-p lies closely above it: one slot is left, whatever an
    earlier call found in that place."""
    u = torch.rand(rows, generator=gen(80), device="cuda")
    for far in (-20.0, -1.3):
        scores = torch.full((rows, n), far, device="cuda")
        scores[:, n // 2] = 0.0
        scores[:, n // 3] = -1.01                      # weight 0.3642
        if far == -1.3:
            scores[:, :n // 4] = scores[:, n - n // 4:] = -30.0
            scores[:, n // 4:n // 3] = -30.0
            scores[:, n // 3 + 1:n // 3 + 3] = -1.3
            scores[:, n // 3 + 3:n // 2] = scores[:, n // 2 + 1:n - n // 4] = -30.0
        for before in (5.0, 90.0, -0.4):
            other = torch.full((rows, n), before - 60.0, device="cuda")
            other[:, 5], other[:, 9] = before, before - 0.3
            check(sample, other, u, top_p=0.8)
            slots, probs = check(sample, scores, u, top_p=0.6 if far == -1.3 else 0.9, min_p=0.36604)
            assert slots.tolist() == [n // 2] * rows and probs.tolist() == [1.0] * rows


def test_masked_and_not_numbers(sample):
    n = 3000
    g = gen(12)
    scores = 4 * torch.randn(8, n, generator=g, device="cuda")
    scores[0, ::2] = -float("inf")
    scores[1] = -float("inf")
    scores[2] = float("nan")
    scores[3, 5:2000] = float("nan")
    scores[4, 77] = float("inf")
    scores[5, 100:2000:7] = float("inf")
    scores[6] = torch.finfo(torch.float32).min
    scores[7, 1:] = -float("inf")
    u = torch.rand(8, generator=g, device="cuda")
    few = torch.rand(47, 64, generator=g, device="cuda") < 0.02
    shared = (few.long() << torch.arange(64, device="cuda")).sum(1)
    none = torch.zeros(47, dtype=torch.int64, device="cuda")
    beyond = none.clone()
    beyond[-1] = -1 << (n % 64)                     # only bits past the row's end
    own = torch.stack([shared, none, shared, shared, ~none, ~none, shared, beyond])
    for mask in (None, shared, ~none, none, beyond, own):
        for limits in (dict(), dict(top_k=9), dict(top_p=0.6), dict(top_k=500, top_p=0.9, min_p=0.02), dict(temperature=0.0), dict(temperature=1e-30), dict(temperature=1e30, top_p=0.5)):
            check(sample, scores, u, mask=mask, **limits)


def test_random_numbers_and_parameters_that_are_none(sample):
    """u outside [0, 1) or NaN, parameters that are NaN: as the ends of their ranges, or no limit."""
    scores = torch.randn(4, 500, generator=gen(13), device="cuda")
    nan = float("nan")
    slots, _ = sample(scores, torch.tensor([-1.0, nan, 1.0, 7.0], device="cuda"))
    assert slots.tolist() == [0, 0, 499, 499]
    u = torch.rand(4, generator=gen(14), device="cuda")
    want = sample(scores, u)
    for limits in (dict(top_p=nan), dict(min_p=nan), dict(min_p=-1.0), dict(top_k=0)):
        assert all(torch.equal(x, y) for x, y in zip(sample(scores, u, **limits), want))
    assert torch.equal(sample(scores, u, temperature=nan)[0], scores.argmax(1))


def test_strided_rows(sample):
    base = 3 * torch.randn(5, 2100, generator=gen(15), device="cuda")
    u = torch.rand(5, generator=gen(16), device="cuda")
    for dtype in DTYPES:
        wide = base.to(dtype)
        for off, n in ((0, 2048), (1, 2048), (3, 1999), (8, 64)):
            check(sample, wide[:, off:off + n], u, top_k=100, top_p=0.95)
            check(sample, wide[:1].expand(5, -1)[:, off:off + n], u)


def test_probabilities_are_drawn_as_often(sample):
    """Evenly spaced random numbers draw each slot as often as its probability says, to one."""
    row = 2 * torch.randn(1, 40, generator=gen(17), device="cuda")
    draws = 4096
    slots, probs = sample(row.expand(draws, -1), torch.arange(draws, device="cuda") / draws, top_p=0.9)
    count = torch.bincount(slots, minlength=40)
    p = torch.zeros(40, device="cuda").scatter(0, slots, probs)
    assert bool(((count - draws * p).abs() <= 1.01).all()) and abs(float(p.sum()) - 1) < 1e-5


def test_on_another_stream_and_in_a_graph(sample):
    scores = 3 * torch.randn(5, 70_000, generator=gen(18), device="cuda")
    u = torch.rand(5, generator=gen(19), device="cuda")
    k = torch.full((5,), 300, dtype=torch.int32, device="cuda")
    p = torch.full((5,), 0.9, device="cuda")
    run = lambda r: sample(scores[:r], u[:r], top_k=k[:r], top_p=p[:r])  # noqa: E731
    want = run(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graphs = []
    for rows in (5, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run(rows)
        graphs.append((rows, graph, held))
    for turn in range(3):
        scores.copy_(3 * torch.randn(5, 70_000, generator=gen(20 + turn), device="cuda"))
        u.copy_(torch.rand(5, generator=gen(30 + turn), device="cuda"))
        for rows, graph, held in graphs:
            graph.replay()
            torch.randn(100_000, device="cuda").sum().item()
            assert all(torch.equal(x, y) for x, y in zip(run(rows), held))


def test_scores_then_a_draw(sample):
    """Products of 8-bit rows straight into a draw, and the draw over a search's re-scored candidates."""
    from turbovec_amd import fp8
    x = torch.nn.functional.normalize(torch.randn(3000, 256, generator=gen(40), device="cuda"))
    rows, q = fp8.quantize(x), torch.nn.functional.normalize(torch.randn(9, 256, generator=gen(41), device="cuda"))
    u = torch.rand(9, generator=gen(42), device="cuda")
    check(sample, fp8.matmul(fp8.quantize(q), rows, dtype=torch.bfloat16), u, temperature=0.05, top_p=0.9)
    s, slots = fp8.rescore(q, rows, torch.randint(0, 3000, (9, 200), generator=gen(43), device="cuda"), 64)
    place, _ = check(sample, s, u, temperature=0.02, top_k=20)
    drawn = slots.gather(1, place[:, None])
    assert bool((drawn >= 0).all())


@pytest.mark.parametrize("rows,n", [(3, 1), (3, 100), (3, 5000), (3, 20_000), (3, 50_000), (300, 15_000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_temperature_that_is_not_above_zero_draws_the_best(sample, rows, n, dtype):
    """Whatever the other limits say, min-p above all: log(min_p) * T is above 0 there."""
    g = gen(100 + n)
    scores = (3 * torch.randn(rows, n, generator=g, device="cuda")).to(dtype)
    u = torch.rand(rows, generator=g, device="cuda")
    mask = torch.randint(-2 ** 63, 2 ** 63 - 1, (rows, -(-n // 64)), generator=g, device="cuda", dtype=torch.int64)
    mask[1] = 0
    allowed = ((mask[:, :, None] >> torch.arange(64, device="cuda")) & 1).reshape(rows, -1)[:, :n].bool()
    for m, best in ((None, scores.argmax(1)), (mask, torch.where(allowed.any(1), torch.where(allowed, scores, -torch.inf).argmax(1), -1))):
        for t in (-1.0, -1e-30, -1e30, -float("inf"), 0.0, -0.0, float("nan")):
            for limits in (dict(min_p=0.1), dict(min_p=0.9), dict(min_p=1e-30, top_k=7, top_p=0.5), dict(min_p=0.5, top_k=n + 1)):
                slots, probs = sample(scores, u, mask=m, temperature=t, **limits)
                assert torch.equal(slots, best), (t, limits)
                assert torch.equal(probs, (best >= 0).float()), (t, limits)


def test_temperatures_of_both_signs_in_one_call(sample):
    for rows, n in ((40, 3000), (6, 60_000)):
        g = gen(110 + rows)
        scores = 3 * torch.randn(rows, n, generator=g, device="cuda")
        u = torch.rand(rows, generator=g, device="cuda")
        t = torch.randn(rows, generator=g, device="cuda")
        check(sample, scores, u, temperature=t, min_p=0.05)
        check(sample, scores, u, temperature=t, min_p=0.3, top_p=0.9, top_k=torch.arange(rows, device="cuda", dtype=torch.int32) * 3)
